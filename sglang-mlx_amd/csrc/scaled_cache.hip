// Paged caches of E4M3 codes with a scale for each (block, KV head) of K and of V:
// the append that quantises, and the way back.
//
//   store:  a = max |x| over the finite new values of the block and head,
//           s = the least power of two with a / s <= 240, at least the block's scale
//               where it holds earlier tokens,
//           code = x / s rounded to nearest even; earlier codes c become c * (old s / s),
//           rounded the same way, where s has grown.
//   read:   x = code * s, rounded once to the output's type.
//
// 240 is the largest finite value of the format (exponent 15 stands for inf and NaN,
// which are stored as such and take no part in a).  With powers of two the quotient,
// the product and the change of scale are exact but for codes that become subnormal
// (below a / 15360): a block filled token by token holds what it would had it been
// filled at once, and no calibration is needed.  What that gives up is under one
// binade at the bottom of the range, none of the three bits of a code's significand.
//
// One wavefront per (sequence, block, head, K or V): the block's new tokens are read
// once, held in registers while their maximum is taken, and written as the layout has
// them, K as [D / 16][bs][16], V as [D][bs], so that no two wavefronts share a scale
// and nothing waits.
#include "pkv_fp8.h"
#include "pkv_launch.h"

namespace pkv {

namespace {

constexpr int kScaledWaves = 4;  // per workgroup

// A wavefront's sequence and its place in it: work items of the sequences lie end to
// end, sequence s from start_loc[s] / bs + extra * s on (a sum that grows by at least
// the blocks that n tokens touch: n / bs + 1 from a block's start on, + 2 from
// anywhere).  The last s whose items begin at or before `item`, by 64 probes at a time.
struct Found {
  int seq, start, count, nth;
};
__device__ __forceinline__ Found find_item(const int32_t* start_loc, int num_seqs, int num_tokens, int shift, int extra,
                                           int item) {
  const int lane = threadIdx.x & 63;
  auto at = [&](int s) { return s > num_seqs ? num_tokens : min(max(start_loc[s], 0), num_tokens); };
  int lo = 0, hi = num_seqs + 1;  // (the rows behind the last sequence are one more)
  while (hi - lo > 1) {
    const int step = (hi - lo + 63) / 64;
    const int s = lo + lane * step;
    const bool before = s < hi && (at(s) >> shift) + extra * s <= item;
    const int n = max(__popcll(__ballot(before)), 1);
    lo += (n - 1) * step;
    hi = min(lo + step, hi);
  }
  Found f;
  f.seq = __builtin_amdgcn_readfirstlane(lo);
  f.start = __builtin_amdgcn_readfirstlane(at(f.seq));
  f.count = max(__builtin_amdgcn_readfirstlane(at(f.seq + 1)) - f.start, 0);
  f.nth = item - ((f.start >> shift) + extra * f.seq);
  return f;
}

__device__ __forceinline__ float wave_max(float x) {
#pragma unroll
  for (int d = 1; d < 16; d <<= 1) x = fmaxf(x, __shfl_xor(x, d));
  return xchg32_max(xchg16_max(x));
}

// |x| where it is finite, else 0.
__device__ __forceinline__ float finite_size(float x) {
  const float a = __builtin_fabsf(x);
  return a < __builtin_inff() ? a : 0.f;  // (NaN compares false)
}

// The least power of two that brings a (finite, not negative) to at most 240 =
// 1.875 * 2^7; 2^-126 for what is smaller than it can serve.
__device__ __forceinline__ float scale_for(float a) {
  const uint32_t bits = __float_as_uint(a);
  const int e = (int)(bits >> 23) - 7 + ((bits & 0x7fffffu) > 0x700000u ? 1 : 0);
  return __uint_as_float((uint32_t)max(e, 1) << 23);
}

// x / scale: a product with the reciprocal where that is exact (inv != 0).
struct Divide {
  float scale, inv;
  __device__ __forceinline__ explicit Divide(float s) : scale(s) {
    const uint32_t bits = __float_as_uint(s);
    const bool two = (bits & 0x807fffffu) == 0 && bits != 0 && bits < 0x7e800000u;
    inv = two ? __uint_as_float(0x7f000000u - bits) : 0.f;
  }
  __device__ __forceinline__ float operator()(float x) const { return inv != 0.f ? x * inv : __fdiv_rn(x, scale); }
};

// Codes of four values that are at most 240 in size where they are finite.
__device__ __forceinline__ uint32_t encode4(const float* q) {
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(q[0], q[1], 0, false);
  w = __builtin_amdgcn_cvt_pk_fp8_f32(q[2], q[3], w, true);
  const float worst = fmaxf(fmaxf(__builtin_fabsf(q[0]), __builtin_fabsf(q[1])),
                            fmaxf(__builtin_fabsf(q[2]), __builtin_fabsf(q[3])));
  const bool odd = !(worst < __builtin_inff()) || q[0] != q[0] || q[1] != q[1] || q[2] != q[2] || q[3] != q[3];
  if (__builtin_expect(odd, 0)) {
    uint32_t fixed = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t b = __float_as_uint(q[i]);
      uint32_t c = ((uint32_t)w >> (8 * i)) & 0xffu;
      if ((b & 0x7fffffffu) >= 0x7f800000u) c = ((b >> 31) << 7) | 0x78u | ((b & 0x7fffffu) != 0u ? 1u : 0u);
      fixed |= c << (8 * i);
    }
    return fixed;
  }
  return (uint32_t)w;
}

// Four codes as float32; inf and NaN for exponent 15.
__device__ __forceinline__ void decode4(uint32_t w, float* x) {
  const auto a = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false);
  const auto b = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
  x[0] = a[0], x[1] = a[1], x[2] = b[0], x[3] = b[1];
  if (__builtin_expect(fp8x4_special(w) != 0u, 0)) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t c = (w >> (8 * i)) & 0xffu;
      if ((c & 0x78u) == 0x78u) x[i] = __uint_as_float((c & 7u) ? 0x7fc00000u : 0x7f800000u | ((c & 0x80u) << 24));
    }
  }
}

// Four codes in units of another scale; those of inf and NaN stay.
__device__ __forceinline__ uint32_t rescale4(uint32_t w, float old, const Divide& by) {
  float x[4];
  decode4(w, x);
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = by(x[i] * old);
  return encode4(x);
}

// Two elements of a source row as float32.
template <class S> struct Pair;
template <> struct Pair<BF16> {
  uint32_t w;
  __device__ __forceinline__ float lo() const { return __uint_as_float(w << 16); }
  __device__ __forceinline__ float hi() const { return __uint_as_float(w & 0xffff0000u); }
};
template <> struct Pair<F16> {
  uint32_t w;
  __device__ __forceinline__ float lo() const { return f16_bits_to_f32(w & 0xffffu); }
  __device__ __forceinline__ float hi() const { return f16_bits_to_f32(w >> 16); }
};
template <> struct Pair<F32> {
  float a, b;
  __device__ __forceinline__ float lo() const { return a; }
  __device__ __forceinline__ float hi() const { return b; }
};
template <class S> __device__ __forceinline__ Pair<S> no_pair() {
  Pair<S> p;
  __builtin_memset(&p, 0, sizeof p);
  return p;
}

__device__ __forceinline__ uint32_t byte_of(const uint32_t* w, int i) { return (w[i >> 2] >> (8 * (i & 3))) & 0xffu; }

}  // namespace

// BS tokens a block; NS: 128-dimension slices of a head.
//
// Bound: HBM.  A lane of K's wavefronts holds 16 dimensions of a token (two loads, one
// 16-byte store; the wavefront's stores are contiguous), one of V's two dimensions of
// all tokens (256 bytes a load, BS contiguous bytes a dimension).
template <class S, int BS, int NS>
__global__ __launch_bounds__(64 * kScaledWaves) void quantize_kernel(ScaledCacheParams p) {
  constexpr int SHIFT = BS == 8 ? 3 : BS == 16 ? 4 : 5;
  constexpr int NU = (NS * BS + 7) / 8;  // (token, 16 dimensions) units of a lane
  constexpr int W = BS / 4;              // words of a row of V
  using SS = typename Elem<S>::storage;
  const int lane = threadIdx.x & 63;
  const int64_t wave = (int64_t)blockIdx.x * kScaledWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int H = p.num_heads, D = p.head_size;
  const int is_v = (int)(wave & 1);
  const int head = (int)((wave >> 1) % H);
  const int item = (int)((wave >> 1) / H);
  const Found f = find_item(p.start_loc, p.num_seqs, p.num_tokens, SHIFT, 2, item);
  if (f.seq >= p.num_seqs || f.count == 0) return;
  const uint32_t ctx = (uint32_t)p.context_lens[f.seq];
  if (ctx == 0 || ctx > (uint64_t)p.max_blocks_per_seq * BS) return;
  // Token i of the sequence sits at position first + i; those before position 0 nowhere.
  const int64_t first = (int64_t)ctx - f.count;
  const int64_t block = (max(first, (int64_t)0) >> SHIFT) + f.nth;
  if (block * BS >= ctx) return;
  const int32_t id = p.block_tables[(int64_t)f.seq * p.max_blocks_per_seq + block];
  if (id < 0 || id >= p.num_blocks) return;
  const int o0 = (int)(max(max(first, (int64_t)0), block * BS) - block * BS);
  const int o1 = (int)(min((int64_t)ctx, (block + 1) * BS) - block * BS);
  const int64_t row0 = f.start + (block * BS + o0 - first) - o0;  // row of offset o is row0 + o
  float* scale_at = p.scales + ((int64_t)id * H + head) * 2 + is_v;
  const float before = o0 > 0 ? *scale_at : 0.f;
  uint8_t* region = static_cast<uint8_t*>(is_v ? p.v_cache : p.k_cache) + ((int64_t)id * H + head) * D * BS;

  // The block's scale from its largest new value, and the codes it holds brought to it.
  auto settle = [&](float a) { return fmaxf(scale_for(wave_max(a)), before); };
  if (!is_v) {
    const SS* src = static_cast<const SS*>(p.key) + row0 * p.key_stride + (int64_t)head * D;
    Pair<S> x[NU][8];
    float a = 0.f;
#pragma unroll
    for (int j = 0; j < NU; ++j) {
      const int u = lane + 64 * j, c = u >> SHIFT, t = u & (BS - 1);
      const bool mine = 16 * c < D && t >= o0 && t < o1;
#pragma unroll
      for (int k = 0; k < 8; ++k) x[j][k] = no_pair<S>();
      if (mine) {
        const uint4* from = reinterpret_cast<const uint4*>(src + t * p.key_stride + 16 * c);
#pragma unroll
        for (int k = 0; k < (int)sizeof(x[j]) / 16; ++k) {
          const uint4 v = from[k];
          __builtin_memcpy(reinterpret_cast<char*>(&x[j][0]) + 16 * k, &v, 16);
        }
      }
    }
#pragma unroll
    for (int j = 0; j < NU; ++j)
#pragma unroll
      for (int k = 0; k < 8; ++k) a = fmaxf(a, fmaxf(finite_size(x[j][k].lo()), finite_size(x[j][k].hi())));
    const float scale = settle(a);
    const Divide by(scale);
    const bool grown = o0 > 0 && scale != before;
#pragma unroll
    for (int j = 0; j < NU; ++j) {
      const int u = lane + 64 * j, c = u >> SHIFT, t = u & (BS - 1);
      if (16 * c >= D) continue;
      uint4* to = reinterpret_cast<uint4*>(region) + u;
      if (t >= o0 && t < o1) {
        uint32_t w[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float q[4] = {by(x[j][2 * k].lo()), by(x[j][2 * k].hi()), by(x[j][2 * k + 1].lo()),
                              by(x[j][2 * k + 1].hi())};
          w[k] = encode4(q);
        }
        *to = make_uint4(w[0], w[1], w[2], w[3]);
      } else if (grown && t < o0) {
        const uint4 was = *to;
        *to = make_uint4(rescale4(was.x, before, by), rescale4(was.y, before, by), rescale4(was.z, before, by),
                         rescale4(was.w, before, by));
      }
    }
    if (lane == 0 && (o0 == 0 || grown)) *scale_at = scale;
    return;
  }
  const SS* src = static_cast<const SS*>(p.value) + row0 * p.value_stride + (int64_t)head * D;
  Pair<S> x[NS][BS];
  float a = 0.f;
#pragma unroll
  for (int j = 0; j < NS; ++j) {
    const int d = 2 * lane + 128 * j;
#pragma unroll
    for (int t = 0; t < BS; ++t) {
      x[j][t] = no_pair<S>();
      if (d < D && t >= o0 && t < o1) x[j][t] = *reinterpret_cast<const Pair<S>*>(src + t * p.value_stride + d);
    }
  }
#pragma unroll
  for (int j = 0; j < NS; ++j)
#pragma unroll
    for (int t = 0; t < BS; ++t) a = fmaxf(a, fmaxf(finite_size(x[j][t].lo()), finite_size(x[j][t].hi())));
  const float scale = settle(a);
  const Divide by(scale);
  const bool grown = o0 > 0 && scale != before;
  const bool whole = o0 == 0 && o1 == BS;
#pragma unroll
  for (int j = 0; j < NS; ++j) {
    const int d = 2 * lane + 128 * j;
    if (d >= D) continue;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      uint32_t* row = reinterpret_cast<uint32_t*>(region + (int64_t)(d + i) * BS);
      uint32_t w[W];
#pragma unroll
      for (int k = 0; k < W; ++k) {
        float q[4];
#pragma unroll
        for (int t = 0; t < 4; ++t) q[t] = by(i == 0 ? x[j][4 * k + t].lo() : x[j][4 * k + t].hi());
        w[k] = encode4(q);
      }
      if (whole) {
        if constexpr (W == 2)
          *reinterpret_cast<uint2*>(row) = make_uint2(w[0], w[1]);
        else
#pragma unroll
          for (int k = 0; k < W; k += 4) *reinterpret_cast<uint4*>(row + k) = make_uint4(w[k], w[k + 1], w[k + 2], w[k + 3]);
        continue;
      }
#pragma unroll
      for (int k = 0; k < W; ++k) {
        // (Offsets behind the new tokens stay as they were.)
        if (grown && 4 * k < o0) {
          const uint32_t old = rescale4(row[k], before, by);
#pragma unroll
          for (int t = 0; t < 4; ++t)
            if (4 * k + t < o0) reinterpret_cast<uint8_t*>(row)[4 * k + t] = (uint8_t)(old >> (8 * t));
        }
#pragma unroll
        for (int t = 0; t < 4; ++t)
          if (4 * k + t >= o0 && 4 * k + t < o1) reinterpret_cast<uint8_t*>(row)[4 * k + t] = (uint8_t)(w[k] >> (8 * t));
      }
    }
  }
  if (lane == 0 && (o0 == 0 || grown)) *scale_at = scale;
}

// Two values in an output row.
template <class O> __device__ __forceinline__ Pair<O> make_pair_of(float a, float b) {
  Pair<O> r;
  if constexpr (std::is_same<O, F32>::value)
    r.a = a, r.b = b;
  else
    r.w = pack2(from_f32<O>(a), from_f32<O>(b));
  return r;
}

// The way back: the same wavefronts, rows of tokens out.  Rows without a block (behind
// the last sequence, past a table, a block id outside the cache) are zeros.
template <class O, int BS, int NS>
__global__ __launch_bounds__(64 * kScaledWaves) void dequantize_kernel(ScaledCacheParams p) {
  constexpr int SHIFT = BS == 8 ? 3 : BS == 16 ? 4 : 5;
  constexpr int NU = (NS * BS + 7) / 8;
  constexpr int W = BS / 4;
  using OS = typename Elem<O>::storage;
  const int lane = threadIdx.x & 63;
  const int64_t wave = (int64_t)blockIdx.x * kScaledWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int H = p.num_heads, D = p.head_size;
  const int is_v = (int)(wave & 1);
  const int head = (int)((wave >> 1) % H);
  const int item = (int)((wave >> 1) / H);
  const Found f = find_item(p.start_loc, p.num_seqs, p.num_tokens, SHIFT, 1, item);
  if ((int64_t)f.nth * BS >= f.count) return;
  const int n = min(f.count - f.nth * BS, BS);
  int32_t id = -1;
  if (f.seq < p.num_seqs && f.nth < p.max_blocks_per_seq) {
    id = p.block_tables[(int64_t)f.seq * p.max_blocks_per_seq + f.nth];
    if (id >= p.num_blocks) id = -1;
  }
  const float scale = id >= 0 ? p.scales[((int64_t)id * H + head) * 2 + is_v] : 0.f;
  const uint8_t* region =
      static_cast<const uint8_t*>(is_v ? p.v_cache : p.k_cache) + ((int64_t)max(id, 0) * H + head) * D * BS;
  OS* out = static_cast<OS*>(is_v ? p.value_out : p.key_out) + ((f.start + (int64_t)f.nth * BS) * H + head) * D;
  const int64_t stride = (int64_t)H * D;
  if (!is_v) {
#pragma unroll
    for (int j = 0; j < NU; ++j) {
      const int u = lane + 64 * j, c = u >> SHIFT, t = u & (BS - 1);
      if (16 * c >= D || t >= n) continue;
      uint32_t w[4] = {0, 0, 0, 0};
      if (id >= 0) *reinterpret_cast<uint4*>(w) = reinterpret_cast<const uint4*>(region)[u];
      Pair<O> y[8];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        float x[4];
        decode4(w[k], x);
        y[2 * k] = make_pair_of<O>(x[0] * scale, x[1] * scale);
        y[2 * k + 1] = make_pair_of<O>(x[2] * scale, x[3] * scale);
      }
      uint4* to = reinterpret_cast<uint4*>(out + t * stride + 16 * c);
#pragma unroll
      for (int k = 0; k < (int)sizeof(y) / 16; ++k) {
        uint4 v;
        __builtin_memcpy(&v, reinterpret_cast<const char*>(&y[0]) + 16 * k, 16);
        to[k] = v;
      }
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < NS; ++j) {
    const int d = 2 * lane + 128 * j;
    if (d >= D) continue;
    uint32_t w[2 * W];
#pragma unroll
    for (int k = 0; k < 2 * W; ++k) w[k] = 0;
    if (id >= 0) {
      const uint4* from = reinterpret_cast<const uint4*>(region + (int64_t)d * BS);
#pragma unroll
      for (int k = 0; k < W / 2; ++k) *reinterpret_cast<uint4*>(w + 4 * k) = from[k];
    }
#pragma unroll
    for (int k = 0; k < W; ++k) {
      float a[4], b[4];
      decode4(w[k], a);
      decode4(w[W + k], b);
#pragma unroll
      for (int t = 0; t < 4; ++t)
        if (4 * k + t < n)
          *reinterpret_cast<Pair<O>*>(out + (4 * k + t) * stride + d) = make_pair_of<O>(a[t] * scale, b[t] * scale);
    }
  }
}

namespace {

template <class T, int BS, int NS> void launch_scaled(const ScaledCacheParams& p, dim3 grid, hipStream_t stream) {
  if (p.key_out != nullptr)
    hipLaunchKernelGGL((dequantize_kernel<T, BS, NS>), grid, dim3(64 * kScaledWaves), 0, stream, p);
  else
    hipLaunchKernelGGL((quantize_kernel<T, BS, NS>), grid, dim3(64 * kScaledWaves), 0, stream, p);
}
template <class T, int BS> void launch_scaled(const ScaledCacheParams& p, dim3 grid, hipStream_t stream) {
  if (p.head_size <= 128)
    launch_scaled<T, BS, 1>(p, grid, stream);
  else
    launch_scaled<T, BS, 2>(p, grid, stream);
}
template <class T> void launch_scaled(const ScaledCacheParams& p, dim3 grid, hipStream_t stream) {
  if (p.block_shift == 3)
    launch_scaled<T, 8>(p, grid, stream);
  else if (p.block_shift == 4)
    launch_scaled<T, 16>(p, grid, stream);
  else
    launch_scaled<T, 32>(p, grid, stream);
}

}  // namespace

hipError_t launch_scaled_cache(const ScaledCacheParams& p, hipStream_t stream) {
  const dim3 grid((unsigned)scaled_cache_groups(p));
  if (p.dtype == kBF16)
    launch_scaled<BF16>(p, grid, stream);
  else if (p.dtype == kF16)
    launch_scaled<F16>(p, grid, stream);
  else
    launch_scaled<F32>(p, grid, stream);
  return hipGetLastError();
}

}  // namespace pkv
