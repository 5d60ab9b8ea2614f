// Norm of queries and keys for each head, the rotation by their positions, and
// the append of the rotated keys and the values to a KV cache, in one launch.
//
// A row x of D elements (one token's one head) becomes y = x * rsqrt(mean(x^2) +
// eps) * w (x itself where there is no weight), and its first rot elements turn
// in pairs (a, b) -> (a cos - b sin, b cos + a sin), pair i of the halves layout
// being (i, i + rot / 2) and of the interleaved layout (2 i, 2 i + 1).  cos and
// sin come from a float32 table, row = position.  Everything is float32 from
// the load to the one rounding at the store.
//
// A group of G lanes, the power of two that covers D / 8, holds a row: lane c
// has the 16 bytes (float32: 32) of elements 8c .. 8c+7.  The sum of squares is
// an xor reduction over the group, a pair's other half comes from the lane
// rot / 16 away, and a lane keeps its cosines and sines over the kHeads heads
// of one token that its group takes.
//
// The paged cache's regions are filled by workgroups of their own, one per
// (window of block_size batch tokens, head), as in reshape_and_cache.hip: tokens that fill a
// whole block in order go through an LDS image of the block's K and V regions
// and leave as whole lines, others leave the image token by token.  Token rows
// are written like the queries.
//
// Bound: HBM traffic (each input read once, each output written once), and for
// a few tokens the chain position -> table -> store.
#include "pkv_fp8.h"
#include "pkv_launch.h"
#include "rac_window.h"

namespace pkv {

namespace {

constexpr int kThreads = 256;
constexpr int kHeads = 4;  // heads of one token per lane group

typedef unsigned int u32x4_t __attribute__((ext_vector_type(4)));

// Eight elements of a row as loaded.
template <class T> struct Piece {
  uint4 a;
};
template <> struct Piece<F32> {
  float4 a, b;
};
__device__ __forceinline__ void unpack(const Piece<F32>& r, float (&x)[8]) {
  x[0] = r.a.x, x[1] = r.a.y, x[2] = r.a.z, x[3] = r.a.w, x[4] = r.b.x, x[5] = r.b.y, x[6] = r.b.z, x[7] = r.b.w;
}
template <class T> __device__ __forceinline__ void unpack(const Piece<T>& r, float (&x)[8]) {
  const uint32_t u[4] = {r.a.x, r.a.y, r.a.z, r.a.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = to_f32<T>((uint16_t)(u[i] & 0xffffu));
    x[2 * i + 1] = to_f32<T>((uint16_t)(u[i] >> 16));
  }
}
template <class T>
__device__ __forceinline__ Piece<T> load_piece(const typename Elem<T>::storage* src) {
  Piece<T> r;
  if constexpr (std::is_same<T, F32>::value) {
    r.a = reinterpret_cast<const float4*>(src)[0];
    r.b = reinterpret_cast<const float4*>(src)[1];
  } else {
    r.a = *reinterpret_cast<const uint4*>(src);
  }
  return r;
}
template <class T> __device__ __forceinline__ Piece<T> no_piece() {
  Piece<T> r;
  __builtin_memset(&r, 0, sizeof(r));
  return r;
}

// Eight floats as elements of type T: 32, 16 or 8 bytes.
template <class T> struct Packed {
  uint4 a;
};
template <> struct Packed<F32> {
  float4 a, b;
};
template <> struct Packed<FP8> {
  uint2 a;
};
template <class T> __device__ __forceinline__ Packed<T> pack(const float (&x)[8], const Fp8Scale& s) {
  Packed<T> r;
  if constexpr (std::is_same<T, F32>::value) {
    r.a = make_float4(x[0], x[1], x[2], x[3]);
    r.b = make_float4(x[4], x[5], x[6], x[7]);
  } else if constexpr (std::is_same<T, FP8>::value) {
    r.a = make_uint2(fp8_encode4_scaled(x, s), fp8_encode4_scaled(x + 4, s));
  } else {
    r.a = make_uint4(pack2(from_f32<T>(x[0]), from_f32<T>(x[1])), pack2(from_f32<T>(x[2]), from_f32<T>(x[3])),
                     pack2(from_f32<T>(x[4]), from_f32<T>(x[5])), pack2(from_f32<T>(x[6]), from_f32<T>(x[7])));
  }
  return r;
}
// Values are copied: the same bits where the cache has their type.
template <class S, class T> __device__ __forceinline__ Packed<T> pack_value(const Piece<S>& v, const Fp8Scale& s) {
  if constexpr (std::is_same<S, T>::value) {
    return __builtin_bit_cast(Packed<T>, v);
  } else {
    float x[8];
    unpack(v, x);
    return pack<T>(x, s);
  }
}
template <class T>
__device__ __forceinline__ void store_piece(typename Elem<T>::storage* dst, const Packed<T>& r) {
  if constexpr (std::is_same<T, F32>::value) {
    reinterpret_cast<float4*>(dst)[0] = r.a;
    reinterpret_cast<float4*>(dst)[1] = r.b;
  } else {
    *reinterpret_cast<decltype(r.a)*>(dst) = r.a;
  }
}

// How the rotation of this call goes (uniform).
struct Turn {
  int rot, half, c, partner;  // partner: the lane that holds the pairs' other half
  bool interleaved, vec;      // vec: pairs' halves and the table in whole pieces
};
__device__ __forceinline__ Turn make_turn(const NormRopeParams& p, int lane, int c, int group) {
  Turn t;
  t.rot = p.rot;
  t.half = p.rot >> 1;
  t.c = c;
  t.interleaved = p.interleaved != 0;
  t.vec = p.rot % (t.interleaved ? 8 : 16) == 0;
  const int k = p.rot >> 4;
  t.partner = (lane & ~(group - 1)) + (c < k ? c + k : c < 2 * k ? c - k : c);
  return t;
}

// This lane's cosines and sines of a token: element i's (halves) or pair i's
// (interleaved, the first four).  Elements that do not turn get (1, 0).
struct Angles {
  float cos[8], sin[8];
};
__device__ __forceinline__ Angles load_angles(const NormRopeParams& p, const Turn& t, int32_t pos) {
  Angles a;
  const int64_t at = min(max((int64_t)pos, (int64_t)0), p.num_positions - 1);
  const float* row = p.cos_sin + at * t.rot;
#pragma unroll
  for (int i = 0; i < 8; ++i) a.cos[i] = 1.f, a.sin[i] = 0.f;
  const int e0 = 8 * t.c;
  if (e0 >= t.rot) return a;
  if (t.interleaved) {
    const int i0 = e0 >> 1;
    if (t.vec) {
      const float4 c = *reinterpret_cast<const float4*>(row + i0);
      const float4 s = *reinterpret_cast<const float4*>(row + t.half + i0);
      a.cos[0] = c.x, a.cos[1] = c.y, a.cos[2] = c.z, a.cos[3] = c.w;
      a.sin[0] = s.x, a.sin[1] = s.y, a.sin[2] = s.z, a.sin[3] = s.w;
    } else {
      for (int i = 0; i < 4; ++i)
        if (e0 + 2 * i < t.rot) a.cos[i] = row[i0 + i], a.sin[i] = row[t.half + i0 + i];
    }
  } else if (t.vec) {
    const int i0 = e0 < t.half ? e0 : e0 - t.half;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const float4 c = *reinterpret_cast<const float4*>(row + i0 + 4 * j);
      const float4 s = *reinterpret_cast<const float4*>(row + t.half + i0 + 4 * j);
      a.cos[4 * j] = c.x, a.cos[4 * j + 1] = c.y, a.cos[4 * j + 2] = c.z, a.cos[4 * j + 3] = c.w;
      a.sin[4 * j] = s.x, a.sin[4 * j + 1] = s.y, a.sin[4 * j + 2] = s.z, a.sin[4 * j + 3] = s.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int e = e0 + i;
      if (e < t.rot) {
        const int k = e < t.half ? e : e - t.half;
        a.cos[i] = row[k], a.sin[i] = row[t.half + k];
      }
    }
  }
  return a;
}

// One element of a norm's weight.
template <class T> __device__ __forceinline__ float weight_at(const void* w, bool f32, int e) {
  return f32 ? static_cast<const float*>(w)[e] : to_f32<T>(static_cast<const typename Elem<T>::storage*>(w)[e]);
}
template <class T> __device__ __forceinline__ void load_weight(const void* w, bool f32, int c, float (&x)[8]) {
  if (f32)
    unpack(load_piece<F32>(static_cast<const float*>(w) + 8 * c), x);
  else
    unpack(load_piece<T>(static_cast<const typename Elem<T>::storage*>(w) + 8 * c), x);
}

// x: the lane's eight elements of a row, normed and turned in place.  Every
// lane of the wavefront takes part; lanes past the row hold zeros.  row: the
// row in memory.
template <class T>
__device__ __forceinline__ void norm_turn(const NormRopeParams& p, const Turn& t, const Angles& a, int group, bool live,
                                          const void* weight, const float (&w)[8],
                                          const typename Elem<T>::storage* row, float (&x)[8]) {
  float r = 1.f;
  if (weight != nullptr) {
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) ss += x[i] * x[i];
    for (int m = 1; m < group; m <<= 1) ss += __shfl_xor(ss, m);
    r = 1.f / __builtin_sqrtf(ss / (float)p.cache.head_size + p.eps);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = x[i] * r * w[i];
  }
  if (t.interleaved) {
    const int e0 = 8 * t.c;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float u = x[2 * i], v = x[2 * i + 1];
      if (e0 + 2 * i < t.rot) {
        x[2 * i] = u * a.cos[i] - v * a.sin[i];
        x[2 * i + 1] = v * a.cos[i] + u * a.sin[i];
      }
    }
    return;
  }
  const int e0 = 8 * t.c;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    float other;
    if (t.vec) {
      other = __shfl(x[i], t.partner);
    } else {
      other = 0.f;
      const int e = e0 + i;
      if (live && e < t.rot) {
        const int k = e < t.half ? e + t.half : e - t.half;
        other = to_f32<T>(row[k]);
        if (weight != nullptr) other = other * r * weight_at<T>(weight, p.weight_f32 != 0, k);
      }
    }
    // (Other lanes read x[i] in the same step: it is written after.)
    if (e0 + i < t.rot) x[i] = x[i] * a.cos[i] + (e0 + i < t.half ? -other : other) * a.sin[i];
  }
}

// ---- one window of a paged cache ----------------------------------------------
// Keys and values of batch tokens [s0, s0 + count) of head h -> the LDS images
// of one (block, head) region each, token s0 + t at the place of offset t.
template <class KT, class CT>
__device__ __forceinline__ void stage_window(const NormRopeParams& p, char* s_k, char* s_v, int64_t s0, int count,
                                             int h, int group, int bs) {
  using KS = typename Elem<KT>::storage;
  using CS = typename Elem<CT>::storage;
  constexpr int X = 16 / Elem<CT>::kBytes;
  const int tid = threadIdx.x, lane = tid & 63;
  const int D = p.cache.head_size, c = tid & (group - 1), groups = kThreads / group;
  const bool live_lane = 8 * c < D;
  const Turn t = make_turn(p, lane, c, group);
  const Fp8Scale ks{p.cache.k_scale, p.cache.k_inv, p.cache.fast_div != 0};
  const Fp8Scale vs{p.cache.v_scale, p.cache.v_inv, p.cache.fast_div != 0};
  float w[8];
  if (p.k_weight != nullptr && live_lane) load_weight<KT>(p.k_weight, p.weight_f32 != 0, c, w);
  // (A wavefront's trips are the same in every lane.)
  for (int j0 = 0; j0 < count; j0 += groups) {
    const int j = j0 + tid / group;
    const bool live = live_lane && j < count;
    const int64_t tok = s0 + min(j, count - 1);
    const KS* krow = static_cast<const KS*>(p.cache.key) + tok * p.cache.key_stride + (int64_t)h * D;
    const KS* vrow = static_cast<const KS*>(p.cache.value) + tok * p.cache.value_stride + (int64_t)h * D;
    const Piece<KT> kr = live ? load_piece<KT>(krow + 8 * c) : no_piece<KT>();
    const Piece<KT> vr = live ? load_piece<KT>(vrow + 8 * c) : no_piece<KT>();
    const Angles a = load_angles(p, t, p.positions[tok]);
    float x[8];
    unpack(kr, x);
    norm_turn<KT>(p, t, a, group, live, p.k_weight, w, krow, x);
    if (!live) continue;
    const Packed<CT> kp = pack<CT>(x, ks), vp = pack_value<KT, CT>(vr, vs);
    CS* kd = reinterpret_cast<CS*>(s_k);
    CS* vd = reinterpret_cast<CS*>(s_v);
    const CS* ke = reinterpret_cast<const CS*>(&kp);
    const CS* ve = reinterpret_cast<const CS*>(&vp);
    constexpr int W = X < 8 ? X : 8;  // elements of one K store: 16 bytes, or 8 codes
#pragma unroll
    for (int i = 0; i < 8; i += W) {
      const int d = 8 * c + i;
      __builtin_memcpy(__builtin_assume_aligned(kd + ((d / X) * bs + j) * X + d % X, W * sizeof(CS)), ke + i,
                       W * sizeof(CS));
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) vd[(8 * c + i) * bs + j] = ve[i];
  }
}

template <class KT, class CT>
__device__ __forceinline__ void paged_window(const NormRopeParams& p, int64_t window, int h, int group, char* s_k) {
  using CS = typename Elem<CT>::storage;
  constexpr int X = 16 / Elem<CT>::kBytes;
  const RacParams& rc = p.cache;
  const int tid = threadIdx.x, lane = tid & 63, bs = rc.block_size, D = rc.head_size;
  const int region_bytes = D * bs * (int)sizeof(CS);
  char* s_v = s_k + region_bytes;
  int64_t prev, run;
  int lane_slot;  // lanes bs .. 2 bs - 1: the window's slots
  if (bs == 8)
    rac_window_runs<8>(rc, window, lane, prev, run, lane_slot);
  else if (bs == 16)
    rac_window_runs<16>(rc, window, lane, prev, run, lane_slot);
  else
    rac_window_runs<32>(rc, window, lane, prev, run, lane_slot);
  const int64_t w0 = window * bs;
  char* kc = static_cast<char*>(rc.key_cache);
  char* vc = static_cast<char*>(rc.value_cache);
  if (run >= 0) {
    stage_window<KT, CT>(p, s_k, s_v, run, bs, h, group, bs);
    __syncthreads();
    const int64_t blk = __builtin_amdgcn_readlane(lane_slot, bs + (int)(run - w0)) / bs;
    const int64_t at = (blk * rc.num_heads + h) * region_bytes;
    // Whole lines that nothing in the launch reads back.
    for (int u = tid * 16; u < region_bytes; u += kThreads * 16) {
      __builtin_nontemporal_store(*reinterpret_cast<const u32x4_t*>(s_k + u), reinterpret_cast<u32x4_t*>(kc + at + u));
      __builtin_nontemporal_store(*reinterpret_cast<const u32x4_t*>(s_v + u), reinterpret_cast<u32x4_t*>(vc + at + u));
    }
    __syncthreads();
  }
  // The window's other tokens.
  const int64_t s0 = prev >= 0 ? prev + bs : w0;
  const int64_t s1 = run >= 0 ? run : min(w0 + bs, rc.num_tokens);
  if (s0 >= s1) return;
  const int count = (int)(s1 - s0), lane0 = (int)(s0 - w0) + bs;  // lane0 holds token s0's slot
  stage_window<KT, CT>(p, s_k, s_v, s0, count, h, group, bs);
  __syncthreads();
  const int chunks = D / X;
  // (The slots come from other lanes: a wavefront's trips are the same in every lane.)
  for (int u = tid; u - lane < count * chunks; u += kThreads) {
    const int j = u / chunks, ch = u - j * chunks;
    const int32_t slot = __shfl(lane_slot, (lane0 + j) & 63);
    if (u >= count * chunks || slot < 0 || (int64_t)slot >= rc.num_slots) continue;
    const int64_t at = ((int64_t)(slot / bs) * rc.num_heads + h) * region_bytes;
    *reinterpret_cast<uint4*>(kc + at + (ch * bs + slot % bs) * 16) =
        *reinterpret_cast<const uint4*>(s_k + (ch * bs + j) * 16);
  }
  for (int u = tid; u - lane < count * D; u += kThreads) {
    const int j = u / D, d = u - j * D;
    const int32_t slot = __shfl(lane_slot, (lane0 + j) & 63);
    if (u >= count * D || slot < 0 || (int64_t)slot >= rc.num_slots) continue;
    CS* dst = static_cast<CS*>(rc.value_cache) + ((int64_t)(slot / bs) * rc.num_heads + h) * (int64_t)D * bs;
    dst[d * bs + slot % bs] = reinterpret_cast<const CS*>(s_v)[d * bs + j];
  }
}

// Workgroups [0, window_groups): windows of a paged cache.  The others: rows, a
// lane group each taking up to kHeads heads of a token's queries, of its keys
// and of its values (keys and values: no cache, or token rows).
template <class KT, class CT>
__global__ __launch_bounds__(kThreads) void norm_rope_kernel(NormRopeParams p, int window_groups, int group) {
  using KS = typename Elem<KT>::storage;
  using CS = typename Elem<CT>::storage;
  extern __shared__ __align__(16) char s_image[];
  const RacParams& rc = p.cache;
  const int H = rc.num_heads, D = rc.head_size;
  if ((int)blockIdx.x < window_groups) {
    const int64_t window = blockIdx.x / (uint32_t)H;
    paged_window<KT, CT>(p, window, (int)(blockIdx.x - (uint32_t)window * (uint32_t)H), group, s_image);
    return;
  }
  const int tid = threadIdx.x, lane = tid & 63, c = tid & (group - 1);
  const bool rows = rc.key_cache != nullptr && rc.layout == 1;
  const int q_units = (p.num_heads + kHeads - 1) / kHeads, kv_units = (H + kHeads - 1) / kHeads;
  const int units = q_units + (rows ? 2 * kv_units : p.k_out != nullptr ? kv_units : 0);
  const int64_t id = (int64_t)(blockIdx.x - window_groups) * (kThreads / group) + tid / group;
  const int64_t tok0 = id / units;
  const bool in_batch = tok0 < rc.num_tokens;
  const int64_t tok = in_batch ? tok0 : rc.num_tokens - 1;
  int unit = (int)(id - tok0 * units);
  const int kind = unit < q_units ? 0 : unit < q_units + kv_units ? 1 : 2;  // queries, keys, values
  unit -= kind == 0 ? 0 : kind == 1 ? q_units : q_units + kv_units;
  const int heads = kind == 0 ? p.num_heads : H, h0 = unit * kHeads;
  const bool live_lane = in_batch && 8 * c < D;
  const KS* src = kind == 0   ? static_cast<const KS*>(p.query) + tok * p.q_stride
                  : kind == 1 ? static_cast<const KS*>(rc.key) + tok * rc.key_stride
                              : static_cast<const KS*>(rc.value) + tok * rc.value_stride;
  Piece<KT> raw[kHeads];
#pragma unroll
  for (int i = 0; i < kHeads; ++i)
    raw[i] = live_lane && h0 + i < heads ? load_piece<KT>(src + (int64_t)(h0 + i) * D + 8 * c) : no_piece<KT>();
  const Turn t = make_turn(p, lane, c, group);
  const Angles a = load_angles(p, t, p.positions[tok]);
  const void* weight = kind == 0 ? p.q_weight : p.k_weight;
  float w[8] = {1.f, 1.f, 1.f, 1.f, 1.f, 1.f, 1.f, 1.f};
  if (weight != nullptr && live_lane) load_weight<KT>(weight, p.weight_f32 != 0, c, w);
  const int32_t slot = rows ? rc.slot_mapping[tok] : 0;
  const bool stored = !rows || (slot >= 0 && (int64_t)slot < rc.num_slots);
  const Fp8Scale ks{rc.k_scale, rc.k_inv, rc.fast_div != 0}, vs{rc.v_scale, rc.v_inv, rc.fast_div != 0};
#pragma unroll
  for (int i = 0; i < kHeads; ++i) {
    const int h = h0 + i;
    const bool live = live_lane && h < heads;
    float x[8];
    unpack(raw[i], x);
    // (A wavefront can hold rows of several kinds: all lanes take part.)
    norm_turn<KT>(p, t, a, group, live, weight, w, src + (int64_t)min(h, heads - 1) * D, x);
    if (!live) continue;
    if (kind == 0) {
      store_piece<KT>(static_cast<KS*>(p.q_out) + (tok * p.num_heads + h) * D + 8 * c, pack<KT>(x, ks));
    } else if (!rows) {
      store_piece<KT>(static_cast<KS*>(p.k_out) + (tok * H + h) * D + 8 * c, pack<KT>(x, ks));
    } else if (stored) {
      const int64_t at = ((int64_t)slot * H + h) * D + 8 * c;
      if (kind == 1)
        store_piece<CT>(static_cast<CS*>(rc.key_cache) + at, pack<CT>(x, ks));
      else
        store_piece<CT>(static_cast<CS*>(rc.value_cache) + at, pack_value<KT, CT>(raw[i], vs));
    }
  }
}

template <class KT, class CT>
hipError_t launch_typed(const NormRopeParams& p, hipStream_t stream) {
  const RacParams& rc = p.cache;
  int group = 1;
  while (group * 8 < rc.head_size) group *= 2;
  const bool cache = rc.key_cache != nullptr, paged = cache && rc.layout == 0;
  const int64_t windows = paged ? (rc.num_tokens + rc.block_size - 1) / rc.block_size * rc.num_heads : 0;
  const int q_units = (p.num_heads + kHeads - 1) / kHeads, kv_units = (rc.num_heads + kHeads - 1) / kHeads;
  const int64_t units = rc.num_tokens * (q_units + (paged ? 0 : cache ? 2 * kv_units : kv_units));
  const int64_t blocks = windows + (units * group + kThreads - 1) / kThreads;
  if (blocks * kThreads >= ((int64_t)1 << 32)) return hipErrorInvalidConfiguration;
  const size_t lds = paged ? (size_t)2 * rc.head_size * rc.block_size * Elem<CT>::kBytes : 0;
  hipLaunchKernelGGL((norm_rope_kernel<KT, CT>), dim3((unsigned)blocks), dim3(kThreads), lds, stream, p, (int)windows,
                     group);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_norm_rope(const NormRopeParams& p, hipStream_t stream) {
  const int kt = p.cache.kv_dtype, ct = p.cache.cache_dtype;
  if (kt == kF32 && ct == kF32) return launch_typed<F32, F32>(p, stream);
  if (kt == kF16 && ct == kF16) return launch_typed<F16, F16>(p, stream);
  if (kt == kBF16 && ct == kBF16) return launch_typed<BF16, BF16>(p, stream);
  if (kt == kF32 && ct == kF16) return launch_typed<F32, F16>(p, stream);
  if (kt == kF32 && ct == kBF16) return launch_typed<F32, BF16>(p, stream);
  if (kt == kF32 && ct == kFP8) return launch_typed<F32, FP8>(p, stream);
  if (kt == kF16 && ct == kFP8) return launch_typed<F16, FP8>(p, stream);
  if (kt == kBF16 && ct == kFP8) return launch_typed<BF16, FP8>(p, stream);
  return hipErrorInvalidValue;
}

}  // namespace pkv
