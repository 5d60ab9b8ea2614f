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
// a reduction over the group, a pair's other half comes from the lane rot / 16
// away, and a lane keeps its cosines and sines over the kHeads heads of one
// token that its group takes.
//
// One launch has workgroups of three kinds:
//   values of a paged cache, as in reshape_and_cache.hip: tokens that fill a whole
//     block in order are regrouped in registers and leave as whole lines, others
//     one (token, head) per wavefront;
//   rows of keys: the groups of a workgroup take consecutive tokens of the same
//     heads, whose 16-byte chunks of a paged cache then complete its lines in one
//     L2; token rows (and their values) and plain outputs go the same way;
//   rows of queries: consecutive heads of a token.
//
// Bound: HBM traffic (each input read once, each output written once): 8192 tokens
// of 32 + 8 + 8 heads of 128, bf16, 206 MB, take 44 us on the device, 4.7 TB/s, into
// FP8 caches, 189 MB, 46 us; for a few tokens the chain position -> angles -> store:
// one token 4.0 us.
#include "pkv_fp8.h"
#include "pkv_launch.h"
#include "rac_window.h"

namespace pkv {

namespace {

constexpr int kThreads = 256;
constexpr int kHeads = 4;  // the most heads of one token per lane group

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
// (Nontemporal: lines that nothing in the launch reads back.)
template <class T>
__device__ __forceinline__ void store_piece(typename Elem<T>::storage* dst, const Packed<T>& r) {
  if constexpr (std::is_same<T, F32>::value) {
    store8<true>(dst, __builtin_bit_cast(uint4, r.a));
    store8<true>(dst + 4, __builtin_bit_cast(uint4, r.b));
  } else {
    store8<true>(dst, r.a);
  }
}

// How pairs lie: halves or interleaved, in whole pieces (rot a multiple of 16, or
// of 8), or halves that pieces straddle.
enum { kHalves = 0, kInterleaved = 1, kStraddling = 2 };
struct Turn {
  int rot, half, c, partner;  // partner: the lane that holds the pairs' other half
  bool vec;                   // the table's cosines and sines in whole vectors
};
template <int MODE, int G> __device__ __forceinline__ Turn make_turn(const NormRopeParams& p, int lane, int c) {
  Turn t;
  t.rot = p.rot;
  t.half = p.rot >> 1;
  t.c = c;
  t.vec = p.rot % 8 == 0;
  const int k = p.rot >> 4;
  t.partner = (lane & ~(G - 1)) + (c < k ? c + k : c < 2 * k ? c - k : c);
  return t;
}

// This lane's cosines and sines of a token: element i's (halves) or pair i's
// (interleaved, the first four).  Elements that do not turn get (1, 0).
struct Angles {
  float cos[8], sin[8];
};
template <int MODE> __device__ __forceinline__ Angles load_angles(const NormRopeParams& p, const Turn& t, int32_t pos) {
  Angles a;
  const int64_t at = min(max((int64_t)pos, (int64_t)0), p.num_positions - 1);
  const float* row = p.cos_sin + at * t.rot;
#pragma unroll
  for (int i = 0; i < 8; ++i) a.cos[i] = 1.f, a.sin[i] = 0.f;
  const int e0 = 8 * t.c;
  if (e0 >= t.rot) return a;
  auto four = [&](int i, int from) __attribute__((always_inline)) {
    const float4 c = *reinterpret_cast<const float4*>(row + from);
    const float4 s = *reinterpret_cast<const float4*>(row + t.half + from);
    a.cos[i] = c.x, a.cos[i + 1] = c.y, a.cos[i + 2] = c.z, a.cos[i + 3] = c.w;
    a.sin[i] = s.x, a.sin[i + 1] = s.y, a.sin[i + 2] = s.z, a.sin[i + 3] = s.w;
  };
  if constexpr (MODE == kInterleaved) {
    if (t.vec) {
      four(0, e0 >> 1);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (e0 + 2 * i < t.rot) a.cos[i] = row[(e0 >> 1) + i], a.sin[i] = row[t.half + (e0 >> 1) + i];
    }
  } else if constexpr (MODE == kHalves) {
    const int i0 = e0 < t.half ? e0 : e0 - t.half;
    four(0, i0);
    four(4, i0 + 4);
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

// Sum over a lane group of G (rows of 16 by DPP: neighbours, pairs, mirrored
// halves, mirrored row; equal values meet at each step).
template <int CTRL> __device__ __forceinline__ float dpp(float x) {
  return __uint_as_float((uint32_t)__builtin_amdgcn_mov_dpp((int)__float_as_uint(x), CTRL, 0xf, 0xf, false));
}
template <int G> __device__ __forceinline__ float group_sum(float x) {
  if constexpr (G >= 2) x += dpp<0xB1>(x);   // quad_perm [1, 0, 3, 2]
  if constexpr (G >= 4) x += dpp<0x4E>(x);   // quad_perm [2, 3, 0, 1]
  if constexpr (G >= 8) x += dpp<0x141>(x);  // row_half_mirror
  if constexpr (G >= 16) x += dpp<0x140>(x); // row_mirror
  if constexpr (G >= 32) x = xchg16_sum(x);
  return x;
}

// x: the lane's eight elements of a row, normed and turned in place.  Every
// lane of the group takes part; lanes past the row hold zeros.  row: the row in
// memory (kStraddling reads pairs' other halves from it).
template <class T, int MODE, int G>
__device__ __forceinline__ void norm_turn(const NormRopeParams& p, const Turn& t, const Angles& a, bool live,
                                          const void* weight, const float (&w)[8],
                                          const typename Elem<T>::storage* row, float (&x)[8]) {
  float r = 1.f;
  if (weight != nullptr) {
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) ss += x[i] * x[i];
    r = __builtin_amdgcn_rsqf(group_sum<G>(ss) * p.inv_head_size + p.eps);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = x[i] * r * w[i];
  }
  const int e0 = 8 * t.c;
  if constexpr (MODE == kInterleaved) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float u = x[2 * i], v = x[2 * i + 1];
      if (e0 + 2 * i < t.rot) {
        x[2 * i] = u * a.cos[i] - v * a.sin[i];
        x[2 * i + 1] = v * a.cos[i] + u * a.sin[i];
      }
    }
  } else {
    float other[8];
    if constexpr (MODE == kHalves) {
      if (G == 16 && t.rot == 128) {
#pragma unroll
        for (int i = 0; i < 8; ++i) other[i] = dpp<0x128>(x[i]);  // row_ror:8, the lane 8 away
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) other[i] = __shfl(x[i], t.partner);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        other[i] = 0.f;
        const int e = e0 + i;
        if (live && e < t.rot) {
          const int k = e < t.half ? e + t.half : e - t.half;
          other[i] = to_f32<T>(row[k]);
          if (weight != nullptr) other[i] = other[i] * r * weight_at<T>(weight, p.weight_f32 != 0, k);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (e0 + i < t.rot) x[i] = x[i] * a.cos[i] + (e0 + i < t.half ? -other[i] : other[i]) * a.sin[i];
  }
}

// ---- values of a paged cache ----------------------------------------------------

// One value as an element of the cache.
template <class S, class T>
__device__ __forceinline__ typename Elem<T>::storage value_elem(typename Elem<S>::storage v, const Fp8Scale& s) {
  if constexpr (std::is_same<T, FP8>::value)
    return (uint8_t)fp8_e4m3_encode(__fdiv_rn(to_f32<S>(v), s.scale));
  else
    return convert_elem<S, T>(v);
}

// One (token, head) by a wavefront, lanes over the dimensions, so that a store
// instruction's accesses to one line leave as one request.
template <class KT, class CT>
__device__ __forceinline__ void put_value(const RacParams& c, int64_t tok, int h, int32_t slot, int lane,
                                          const Fp8Scale& s) {
  using KS = typename Elem<KT>::storage;
  using CS = typename Elem<CT>::storage;
  const int D = c.head_size;
  const KS* src = static_cast<const KS*>(c.value) + tok * c.value_stride + (int64_t)h * D;
  KS v[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = lane + 64 * i < D ? src[lane + 64 * i] : (KS)0;
  if (slot < 0 || (int64_t)slot >= c.num_slots) return;
  const int bs = c.block_size;
  CS* dst = static_cast<CS*>(c.value_cache) + ((int64_t)(slot / bs) * c.num_heads + h) * (int64_t)D * bs + slot % bs;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (lane + 64 * i < D) dst[(int64_t)(lane + 64 * i) * bs] = value_elem<KT, CT>(v[i], s);
}

// The values of heads [h0, h0 + nh) of a window of BS batch tokens.
template <class KT, class CT, int BS>
__device__ __forceinline__ void value_window(const RacParams& c, int64_t window, int h0, int nh) {
  using KS = typename Elem<KT>::storage;
  using CS = typename Elem<CT>::storage;
  const int tid = threadIdx.x, lane = tid & 63, D = c.head_size;
  const Fp8Scale vs{c.v_scale, c.v_inv, c.fast_div != 0};
  int64_t prev, run;
  int lane_slot;  // lanes BS .. 2 BS - 1: the window's slots
  rac_window_runs<BS>(c, window, lane, prev, run, lane_slot);
  const int64_t w0 = window * BS;
  if (run >= 0) {
    const int units = D * (BS / 8);
    const int64_t blk = __builtin_amdgcn_readlane(lane_slot, BS + (int)(run - w0)) / BS;
    const KS* v0 = static_cast<const KS*>(c.value) + run * c.value_stride + (int64_t)h0 * D;
    CS* dst = static_cast<CS*>(c.value_cache) + (blk * c.num_heads + h0) * (int64_t)D * BS;
    for (int i = tid; i < nh * units; i += kThreads) {
      const int h = i / units, u = i - h * units;
      const int quad = u % (BS / 4), pair = u / (BS / 4);
      const auto v = load_v_task<KT, CT>(v0 + (int64_t)(4 * quad) * c.value_stride + h * D + 2 * pair, c.value_stride,
                                         (quad & 1) != 0, vs);
      store8<true>(dst + (int64_t)h * D * BS + (2 * pair + (quad & 1)) * BS + 8 * (quad >> 1), v);
    }
  }
  // The window's other tokens.
  const int s0 = prev >= 0 ? (int)(prev + BS - w0) : 0;
  const int s1 = run >= 0 ? (int)(run - w0) : (int)min((int64_t)BS, c.num_tokens - w0);
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  for (int i = wave; i < (s1 - s0) * nh; i += kThreads / 64) {
    const int j = s0 + i / nh;
    put_value<KT, CT>(c, w0 + j, h0 + i % nh, __builtin_amdgcn_readlane(lane_slot, BS + j), lane, vs);
  }
}

// ---- the kernel -------------------------------------------------------------------

// Workgroups of a launch: [0, value_groups) values of a paged cache (windows of
// hg heads where hg > 0, else one (token, head) per wavefront), then key_groups of
// keys (and values of token rows), then queries.
struct Groups {
  int value_groups, hg, key_groups;
  int heads;  // heads of one token per lane group, at most kHeads
};

template <class KT, class CT, int MODE, int G>
__global__ __launch_bounds__(kThreads) void norm_rope_kernel(NormRopeParams p, Groups gr) {
  using KS = typename Elem<KT>::storage;
  using CS = typename Elem<CT>::storage;
  constexpr int X = 16 / Elem<CT>::kBytes;
  constexpr int ROWS = kThreads / G;  // lane groups of a workgroup
  const RacParams& rc = p.cache;
  const int H = rc.num_heads, D = rc.head_size;
  const int tid = threadIdx.x, lane = tid & 63;
  const Fp8Scale ks{rc.k_scale, rc.k_inv, rc.fast_div != 0}, vs{rc.v_scale, rc.v_inv, rc.fast_div != 0};
  if ((int)blockIdx.x < gr.value_groups) {
    if (gr.hg == 0) {
      const uint32_t pair = blockIdx.x * (kThreads / 64) + __builtin_amdgcn_readfirstlane(tid >> 6);
      const uint32_t tok = pair / (uint32_t)H;
      if (tok < rc.num_tokens)
        put_value<KT, CT>(rc, tok, (int)(pair - tok * (uint32_t)H), rc.slot_mapping[tok], lane, vs);
      return;
    }
    if constexpr (!std::is_same<CT, F32>::value) {
      const int parts = (H + gr.hg - 1) / gr.hg;
      const uint32_t window = blockIdx.x / (uint32_t)parts;
      const int h0 = (int)(blockIdx.x - window * (uint32_t)parts) * gr.hg, nh = min(gr.hg, H - h0);
      if (rc.block_size == 8)
        value_window<KT, CT, 8>(rc, window, h0, nh);
      else if (rc.block_size == 16)
        value_window<KT, CT, 16>(rc, window, h0, nh);
      else
        value_window<KT, CT, 32>(rc, window, h0, nh);
    }
    return;
  }
  const int c = tid & (G - 1), slotless = rc.key_cache == nullptr;
  const bool rows = !slotless && rc.layout == 1;
  // The token, the kind (0: queries, 1: keys, 2: values) and the first head of
  // this lane group.
  int64_t tok;
  int kind, h0;
  const int kb = (int)blockIdx.x - gr.value_groups;
  if (kb < gr.key_groups) {
    const int units = (H + gr.heads - 1) / gr.heads, all = rows ? 2 * units : units;
    const int tile = kb / all, unit = kb - tile * all;
    tok = (int64_t)tile * ROWS + tid / G;
    kind = unit < units ? 1 : 2;
    h0 = (unit - (kind == 2 ? units : 0)) * gr.heads;
  } else {
    const int units = (p.num_heads + gr.heads - 1) / gr.heads;
    // (A launch has less than 2^32 threads: lane groups are counted in 32 bits.)
    const uint32_t id = (uint32_t)(kb - gr.key_groups) * ROWS + tid / G;
    const uint32_t q = id / (uint32_t)units;
    tok = q;
    kind = 0;
    h0 = (int)(id - q * (uint32_t)units) * gr.heads;
  }
  const bool in_batch = tok < rc.num_tokens;
  tok = in_batch ? tok : rc.num_tokens - 1;
  const int heads = min(kind == 0 ? p.num_heads : H, h0 + gr.heads);  // this group's end
  const bool live_lane = in_batch && 8 * c < D;
  const KS* src = kind == 0   ? static_cast<const KS*>(p.query) + tok * p.q_stride
                  : kind == 1 ? static_cast<const KS*>(rc.key) + tok * rc.key_stride
                              : static_cast<const KS*>(rc.value) + tok * rc.value_stride;
  Piece<KT> raw[kHeads];
#pragma unroll
  for (int i = 0; i < kHeads; ++i)
    raw[i] = live_lane && h0 + i < heads ? load_piece<KT>(src + (int64_t)(h0 + i) * D + 8 * c) : no_piece<KT>();
  const int32_t slot = kind != 0 && !slotless ? rc.slot_mapping[tok] : 0;
  const bool stored = slotless || (slot >= 0 && (int64_t)slot < rc.num_slots);
  if (kind == 2) {
    if (!live_lane || !stored) return;
#pragma unroll
    for (int i = 0; i < kHeads; ++i)
      if (h0 + i < heads)
        store_piece<CT>(static_cast<CS*>(rc.value_cache) + ((int64_t)slot * H + h0 + i) * D + 8 * c,
                        pack_value<KT, CT>(raw[i], vs));
    return;
  }
  const Turn t = make_turn<MODE, G>(p, lane, c);
  const Angles a = load_angles<MODE>(p, t, p.positions[tok]);
  const void* weight = kind == 0 ? p.q_weight : p.k_weight;
  float w[8] = {1.f, 1.f, 1.f, 1.f, 1.f, 1.f, 1.f, 1.f};
  if (weight != nullptr && live_lane) load_weight<KT>(weight, p.weight_f32 != 0, c, w);
  const int bs = rc.block_size;
  const int64_t block = (int64_t)(slot / bs) * H;
  const int at = slot % bs;
#pragma unroll
  for (int i = 0; i < kHeads; ++i) {
    if (i >= gr.heads) break;
    const int h = h0 + i;
    const bool live = live_lane && h < heads;
    float x[8];
    unpack(raw[i], x);
    norm_turn<KT, MODE, G>(p, t, a, live, weight, w, src + (int64_t)min(h, heads - 1) * D, x);
    if (!live) continue;
    if (kind == 0) {
      store_piece<KT>(static_cast<KS*>(p.q_out) + (tok * p.num_heads + h) * D + 8 * c, pack<KT>(x, ks));
    } else if (slotless) {
      store_piece<KT>(static_cast<KS*>(p.k_out) + (tok * H + h) * D + 8 * c, pack<KT>(x, ks));
    } else if (stored) {
      const Packed<CT> y = pack<CT>(x, ks);
      CS* kc = static_cast<CS*>(rc.key_cache);
      if (rows) {
        store_piece<CT>(kc + ((int64_t)slot * H + h) * D + 8 * c, y);
      } else {
        // Chunks of X elements, block_size of them apart (default stores: the L2
        // joins the tokens' chunks; nontemporal, 8192 tokens took 47.2 us
        // instead of 43.9).
        kc += (block + h) * (int64_t)D * bs;
        if constexpr (std::is_same<CT, F32>::value) {
          *reinterpret_cast<float4*>(kc + (2 * c * bs + at) * X) = y.a;
          *reinterpret_cast<float4*>(kc + ((2 * c + 1) * bs + at) * X) = y.b;
        } else {
          const int d = 8 * c;
          store8<false>(kc + ((d / X) * bs + at) * X + d % X, y.a);
        }
      }
    }
  }
}

template <class KT, class CT, int MODE, int G>
hipError_t launch_group(const NormRopeParams& p, hipStream_t stream) {
  const RacParams& rc = p.cache;
  constexpr int ROWS = kThreads / G;
  const bool cache = rc.key_cache != nullptr, paged = cache && rc.layout == 0;
  const int64_t N = rc.num_tokens, H = rc.num_heads;
  Groups gr{0, 0, 0};
  int64_t values = 0;
  if (paged) {
    // Runs are looked for where writing a run's values one by one costs more (the
    // line of reshape_and_cache.hip).
    if (!std::is_same<CT, F32>::value && N >= rc.block_size && N * H * rc.head_size > (int64_t)1 << 17) {
      const int units = rc.head_size * (rc.block_size / 8);
      gr.hg = (int)std::min<int64_t>(H, (kThreads + units - 1) / units);
      values = (N + rc.block_size - 1) / rc.block_size * ((H + gr.hg - 1) / gr.hg);
    } else {
      values = (N * H * 64 + kThreads - 1) / kThreads;
    }
  }
  // Heads per lane group: one while that gives every CU little, then as many as
  // 64 bytes a lane of loads in flight.  8192 bf16 tokens, 32 + 8 heads x 128:
  // one 62.6, two 50.4, four 43.9 us; 512 tokens 8.7, 7.9, 8.6; one 5.0, 5.5, 5.9.
  const int64_t rows = N * p.num_heads;
  gr.heads = rows <= 4096 ? 1 : rows <= 16384 || std::is_same<KT, F32>::value ? 2 : kHeads;
  const int64_t kv_units = (H + gr.heads - 1) / gr.heads, q_units = (p.num_heads + gr.heads - 1) / gr.heads;
  const int64_t keys = (N + ROWS - 1) / ROWS * (cache && !paged ? 2 * kv_units : kv_units);
  const int64_t queries = (N * q_units + ROWS - 1) / ROWS;
  if ((values + keys + queries) * kThreads >= ((int64_t)1 << 32)) return hipErrorInvalidConfiguration;
  gr.value_groups = (int)values;
  gr.key_groups = (int)keys;
  hipLaunchKernelGGL((norm_rope_kernel<KT, CT, MODE, G>), dim3((unsigned)(values + keys + queries)), dim3(kThreads), 0,
                     stream, p, gr);
  return hipGetLastError();
}

template <class KT, class CT, int MODE> hipError_t launch_mode(const NormRopeParams& p, hipStream_t stream) {
  const int pieces = p.cache.head_size / 8;
  if (pieces <= 8) return launch_group<KT, CT, MODE, 8>(p, stream);
  if (pieces <= 16) return launch_group<KT, CT, MODE, 16>(p, stream);
  return launch_group<KT, CT, MODE, 32>(p, stream);
}

template <class KT, class CT> hipError_t launch_typed(const NormRopeParams& params, hipStream_t stream) {
  NormRopeParams p = params;
  p.inv_head_size = 1.f / (float)p.cache.head_size;
  if (p.interleaved) return launch_mode<KT, CT, kInterleaved>(p, stream);
  if (p.rot % 16 == 0) return launch_mode<KT, CT, kHalves>(p, stream);
  return launch_mode<KT, CT, kStraddling>(p, stream);
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
