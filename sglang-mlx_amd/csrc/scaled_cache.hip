// Paged caches of E4M3 codes with a scale for each (block, KV head) of K and of V:
// the append that quantises, and the way back.
//
//   store:  a = max |x| over the finite new values of the block and head,
//           s = the least power of two with a / s <= 240, at least the block's scale
//               where it holds earlier tokens,
//           code = x / s rounded to nearest even; earlier codes c become c * (old s / s),
//           rounded the same way, where s has grown.
//   read:   x = code * s in float32 (exact where s is a power of two), rounded to the
//           output's type.
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
// anywhere).  The last s whose items begin at or before `item`, by 64 probes at a time;
// the last round's probes hold the sequence's own numbers, its context (or null: none)
// among them.  Starts that decrease, which no call may have, can end at a sequence whose
// items begin behind `item`: nth is negative there, and the kernels leave.
struct Found {
  int seq, start, count, ctx, nth;
};
__device__ __forceinline__ Found find_item(const int32_t* start_loc, const int32_t* context_lens, int num_seqs,
                                           int num_tokens, int shift, int extra, int item) {
  const int lane = threadIdx.x & 63;
  auto at = [&](int s) { return s > num_seqs ? num_tokens : min(max(start_loc[s], 0), num_tokens); };
  auto before = [&](int s, int loc) { return (loc >> shift) + extra * s <= item; };
  int lo = 0, hi = num_seqs + 1;  // (the rows behind the last sequence are one more)
  while (hi - lo > 63) {
    const int step = (hi - lo + 63) / 64;
    const int s = lo + lane * step;
    const bool yes = s < hi && before(s, at(min(s, hi)));
    const int n = max(__popcll(__ballot(yes)), 1);
    lo += (n - 1) * step;
    hi = min(lo + step, hi);
  }
  const int s = lo + lane, loc = at(min(s, num_seqs + 1));
  const int ctx = context_lens != nullptr && s < num_seqs ? context_lens[s] : 0;
  const int n = max(__popcll(__ballot(s < hi && before(s, loc))), 1);
  Found f;
  f.seq = lo + n - 1;
  f.start = __builtin_amdgcn_readlane(loc, n - 1);
  f.count = max(__builtin_amdgcn_readlane(loc, n) - f.start, 0);  // (n < 64: hi - lo is)
  f.ctx = __builtin_amdgcn_readlane(ctx, n - 1);
  f.nth = item - ((f.start >> shift) + extra * f.seq);
  return f;
}

__device__ __forceinline__ float wave_max(float x) {  // (not NaN)
  auto turned = [&](auto by) {
    const int i = __builtin_bit_cast(int, x);
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(i, i, 0x120 + decltype(by)::value, 0xf, 0xf, true));
  };
  x = fmaxf(x, turned(std::integral_constant<int, 8>{}));
  x = fmaxf(x, turned(std::integral_constant<int, 4>{}));
  x = fmaxf(x, turned(std::integral_constant<int, 2>{}));
  x = fmaxf(x, turned(std::integral_constant<int, 1>{}));
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

// The largest size among pairs, by their bits: sizes order as integers do, those of inf
// and NaN behind the finite ones.
template <class S> struct Largest {
  typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
  static constexpr uint32_t kInf = std::is_same<S, BF16>::value ? 0x7f80u : std::is_same<S, F16>::value ? 0x7c00u
                                                                                                        : 0x7f800000u;
  uint32_t m = 0;
  __device__ __forceinline__ void add(const Pair<S>& x) {
    if constexpr (std::is_same<S, F32>::value)
      m = max(m, max(__float_as_uint(x.a) & 0x7fffffffu, __float_as_uint(x.b) & 0x7fffffffu));
    else
      m = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, m),
                                                                 __builtin_bit_cast(u16x2, x.w & 0x7fff7fffu)));
  }
  __device__ __forceinline__ uint32_t bits() const {
    return std::is_same<S, F32>::value ? m : max(m & 0xffffu, m >> 16);
  }
  __device__ __forceinline__ bool finite() const { return bits() < kInf; }
  __device__ __forceinline__ float value() const {
    if constexpr (std::is_same<S, F32>::value) return __uint_as_float(m);
    else if constexpr (std::is_same<S, BF16>::value) return __uint_as_float(bits() << 16);
    else return f16_bits_to_f32(bits());
  }
};

// The largest finite size of a wavefront's pairs; odd: whether any is inf or NaN.
template <class S, int A, int B>
__device__ __forceinline__ float largest_of(const Pair<S> (&x)[A][B], bool& odd) {
  Largest<S> most;
#pragma unroll
  for (int i = 0; i < A; ++i)
#pragma unroll
    for (int j = 0; j < B; ++j) most.add(x[i][j]);
  odd = __ballot(!most.finite()) != 0;
  float a = most.value();
  if (__builtin_expect(odd, 0)) {
    a = 0.f;
#pragma unroll
    for (int i = 0; i < A; ++i)
#pragma unroll
      for (int j = 0; j < B; ++j) a = fmaxf(a, fmaxf(finite_size(x[i][j].lo()), finite_size(x[i][j].hi())));
  }
  return wave_max(a);
}

// Codes of four values: QUICK where all are finite and the scale is a power of two.
template <bool QUICK>
__device__ __forceinline__ uint32_t codes_of(const Divide& by, float a, float b, float c, float d) {
  if constexpr (QUICK) {
    const int w = __builtin_amdgcn_cvt_pk_fp8_f32(a * by.inv, b * by.inv, 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c * by.inv, d * by.inv, w, true);
  } else {
    const float q[4] = {by(a), by(b), by(c), by(d)};
    return encode4(q);
  }
}

}  // namespace

// BS tokens a block; NS: 128-dimension slices of a head.
//
// Bound: HBM for a prompt, by these loads and stores 3.5 TB/s (16000 tokens of 8 heads of 128
// in 25 us; the append by windows moves as many at 6.0 TB/s with non-temporal ones, which are
// not used here), the chain of dependent loads (sequence, rows and block, old scale) for single
// tokens.  A lane of K's wavefronts holds 16 dimensions of a token (two
// loads, one 16-byte store; the wavefront's stores are contiguous), one of V's two
// dimensions of all tokens (256 bytes a load, BS contiguous bytes a dimension).  Four
// wavefronts a workgroup: with eight, 23 prompts of 14000 tokens in all took 29.2 us
// instead of 26.6; with two, the way back of 32000 tokens 41.4 instead of 38.5.
template <class S, int BS, int NS>
__global__ __launch_bounds__(64 * kScaledWaves) void quantize_kernel(ScaledCacheParams p) {
  constexpr int SHIFT = BS == 8 ? 3 : BS == 16 ? 4 : 5;
  constexpr int NU = (NS * BS + 7) / 8;  // (token, 16 dimensions) units of a lane
  constexpr int W = BS / 4;              // words of a row of V
  // Up to so many tokens a wavefront takes one after the other (with the code below for a
  // block's worth, most of it for tokens that are not there, 200 sequences took 12.2 us
  // instead of 4.9 for a token each, 8.8 instead of 7.8 for four, 12.3 instead of 11.4 for
  // eight; 4 heads of 128, then 8).
  constexpr int FEW = 8;
  using SS = typename Elem<S>::storage;
  const int lane = threadIdx.x & 63;
  const int64_t wave = (int64_t)blockIdx.x * kScaledWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int H = p.num_heads, D = p.head_size;
  const int is_v = (int)(wave & 1);
  const int head = (int)((wave >> 1) % H);
  const int item = (int)((wave >> 1) / H);
  const Found f = find_item(p.start_loc, p.context_lens, p.num_seqs, p.num_tokens, SHIFT, 2, item);
  if (f.seq >= p.num_seqs || f.count == 0 || f.nth < 0) return;
  const uint32_t ctx = (uint32_t)f.ctx;
  if (ctx == 0 || ctx > (uint64_t)p.max_blocks_per_seq * BS) return;
  // Token i of the sequence sits at position first + i; those before position 0 nowhere.
  const int64_t first = (int64_t)ctx - f.count;
  const int64_t block = (max(first, (int64_t)0) >> SHIFT) + f.nth;
  if (block * BS >= ctx) return;
  // (The rows are asked for before the block's id is there.)
  const int32_t id = p.block_tables[(int64_t)f.seq * p.max_blocks_per_seq + block];
  const int o0 = (int)(max(max(first, (int64_t)0), block * BS) - block * BS);
  const int o1 = (int)(min((int64_t)ctx, (block + 1) * BS) - block * BS);
  const int64_t row0 = f.start + (block * BS + o0 - first) - o0;  // row of offset o is row0 + o
  const bool in_cache = id >= 0 && id < p.num_blocks;
  const int64_t at = (int64_t)id * H + head;
  float* scale_at = p.scales + at * 2 + is_v;
  uint8_t* region = static_cast<uint8_t*>(is_v ? p.v_cache : p.k_cache) + at * D * BS;
  // Brings the earlier tokens' codes to a larger scale, a word a lane: of K four dimensions,
  // of V up to four tokens of a dimension.
  auto regrow = [&](float before, const Divide& by) __attribute__((always_inline)) {
#pragma unroll 1
    for (int i = lane; i < D * BS / 4; i += 64) {
      const int t = is_v ? 4 * i & (BS - 1) : (i >> 2) & (BS - 1);
      if (t >= o0) continue;
      uint32_t* to = reinterpret_cast<uint32_t*>(region) + i;
      const uint32_t now = rescale4(*to, before, by);
      if (!is_v || t + 4 <= o0) {
        *to = now;
        continue;
      }
#pragma unroll
      for (int k = 0; k < 3; ++k)
        if (t + k < o0) reinterpret_cast<uint8_t*>(to)[k] = (uint8_t)(now >> (8 * k));
    }
  };
  bool odd;
  if (o1 - o0 <= FEW && o1 - o0 < BS) {
    // A few tokens: two dimensions a lane.
    const int64_t stride = is_v ? p.value_stride : p.key_stride;
    const SS* src = static_cast<const SS*>(is_v ? p.value : p.key) + (row0 + o0) * stride + (int64_t)head * D;
    const int n = o1 - o0;
    Pair<S> x[FEW][NS];
#pragma unroll
    for (int t = 0; t < FEW; ++t)
#pragma unroll
      for (int j = 0; j < NS; ++j) {
        const int d = 2 * lane + 128 * j;
        x[t][j] = no_pair<S>();
        if (t < n && d < D) x[t][j] = *reinterpret_cast<const Pair<S>*>(src + t * stride + d);
      }
    if (!in_cache) return;
    const float before = o0 > 0 ? *scale_at : 0.f;
    const float scale = fmaxf(scale_for(largest_of(x, odd)), before);
    const Divide by(scale);
    const bool grown = o0 > 0 && scale != before;
    if (grown) regrow(before, by);
    auto write = [&](auto quick) __attribute__((always_inline)) {
#pragma unroll
      for (int t = 0; t < FEW; ++t)
#pragma unroll
        for (int j = 0; j < NS; ++j) {
          const int d = 2 * lane + 128 * j;
          if (t >= n || d >= D) continue;
          const uint32_t w = codes_of<decltype(quick)::value>(by, x[t][j].lo(), x[t][j].hi(), 0.f, 0.f);
          if (is_v) {
            region[d * BS + o0 + t] = (uint8_t)w;
            region[(d + 1) * BS + o0 + t] = (uint8_t)(w >> 8);
          } else {
            *reinterpret_cast<uint16_t*>(region + ((d >> 4) * BS + o0 + t) * 16 + (d & 15)) = (uint16_t)w;
          }
        }
    };
    if (!odd && by.inv != 0.f) write(std::true_type{});
    else write(std::false_type{});
    if (lane == 0 && (o0 == 0 || grown)) *scale_at = scale;
    return;
  }
  if (!is_v) {
    const SS* src = static_cast<const SS*>(p.key) + row0 * p.key_stride + (int64_t)head * D;
    Pair<S> x[NU][8];
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
    if (!in_cache) return;
    const float before = o0 > 0 ? *scale_at : 0.f;
    const float scale = fmaxf(scale_for(largest_of(x, odd)), before);
    const Divide by(scale);
    const bool grown = o0 > 0 && scale != before;
    auto write = [&](auto quick) __attribute__((always_inline)) {
#pragma unroll
      for (int j = 0; j < NU; ++j) {
        const int u = lane + 64 * j, c = u >> SHIFT, t = u & (BS - 1);
        if (16 * c >= D || t < o0 || t >= o1) continue;
        uint32_t w[4];
#pragma unroll
        for (int k = 0; k < 4; ++k)
          w[k] = codes_of<decltype(quick)::value>(by, x[j][2 * k].lo(), x[j][2 * k].hi(), x[j][2 * k + 1].lo(),
                                                  x[j][2 * k + 1].hi());
        reinterpret_cast<uint4*>(region)[u] = make_uint4(w[0], w[1], w[2], w[3]);
      }
    };
    if (!odd && by.inv != 0.f) write(std::true_type{});
    else write(std::false_type{});
    if (grown) regrow(before, by);
    if (lane == 0 && (o0 == 0 || grown)) *scale_at = scale;
    return;
  }
  const SS* src = static_cast<const SS*>(p.value) + row0 * p.value_stride + (int64_t)head * D;
  Pair<S> x[NS][BS];
#pragma unroll
  for (int j = 0; j < NS; ++j) {
    const int d = 2 * lane + 128 * j;
#pragma unroll
    for (int t = 0; t < BS; ++t) {
      x[j][t] = no_pair<S>();
      if (d < D && t >= o0 && t < o1) x[j][t] = *reinterpret_cast<const Pair<S>*>(src + t * p.value_stride + d);
    }
  }
  if (!in_cache) return;
  const float before = o0 > 0 ? *scale_at : 0.f;
  const float scale = fmaxf(scale_for(largest_of(x, odd)), before);
  const Divide by(scale);
  const bool grown = o0 > 0 && scale != before;
  const bool whole = o0 == 0 && o1 == BS;
  auto write = [&](auto quick) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < NS; ++j) {
      const int d = 2 * lane + 128 * j;
      if (d >= D) continue;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        uint32_t* row = reinterpret_cast<uint32_t*>(region + (d + i) * BS);
        auto value = [&](int t) { return i == 0 ? x[j][t].lo() : x[j][t].hi(); };
        uint32_t w[W];
#pragma unroll
        for (int k = 0; k < W; ++k)
          w[k] = codes_of<decltype(quick)::value>(by, value(4 * k), value(4 * k + 1), value(4 * k + 2), value(4 * k + 3));
        if (whole) {
          if constexpr (W == 2)
            *reinterpret_cast<uint2*>(row) = make_uint2(w[0], w[1]);
          else
#pragma unroll
            for (int k = 0; k < W; k += 4)
              *reinterpret_cast<uint4*>(row + k) = make_uint4(w[k], w[k + 1], w[k + 2], w[k + 3]);
          continue;
        }
        // (Offsets behind the new tokens stay as they were.)
#pragma unroll
        for (int t = 0; t < BS; ++t)
          if (t >= o0 && t < o1) reinterpret_cast<uint8_t*>(row)[t] = (uint8_t)(w[t / 4] >> (8 * (t % 4)));
      }
    }
  };
  if (!odd && by.inv != 0.f) write(std::true_type{});
  else write(std::false_type{});
  if (grown) regrow(before, by);
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

// The way back: the same wavefronts, rows of tokens out (HBM: 32000 tokens of 8 heads of 128
// in 37 us, 5.4 TB/s).  Rows without a block (behind the last sequence, past a table, a
// block id outside the cache) are zeros.
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
  const Found f = find_item(p.start_loc, nullptr, p.num_seqs, p.num_tokens, SHIFT, 1, item);
  if (f.nth < 0 || (int64_t)f.nth * BS >= f.count) return;
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
