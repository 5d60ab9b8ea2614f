// Parts of a paged append shared by the kernels that append (reshape_and_cache.hip,
// norm_rope.hip): element conversion, runs of whole blocks among the tokens, and
// the tasks that write a run's V region.
#pragma once

#include "pkv_fp8.h"
#include "pkv_launch.h"

namespace pkv {

// ---- vector helpers ----------------------------------------------------------
// Load VE elements of type S starting at src (aligned when ALIGNED) and
// convert them to VE elements of type D written to dst.
template <class S, class D, int VE, bool ALIGNED>
__device__ __forceinline__ void convert_run(const typename Elem<S>::storage* __restrict__ src,
                                            typename Elem<D>::storage* __restrict__ dst) {
  if constexpr (ALIGNED && Elem<S>::kBytes == Elem<D>::kBytes && Elem<S>::kBytes * VE == 16 &&
                std::is_same<S, D>::value) {
    *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(src);
  } else if constexpr (ALIGNED && Elem<D>::kBytes == 2 && Elem<S>::kBytes == 4 && VE == 8) {
    const float4 a = reinterpret_cast<const float4*>(src)[0];
    const float4 b = reinterpret_cast<const float4*>(src)[1];
    uint4 o;
    o.x = pack2(from_f32<D>(a.x), from_f32<D>(a.y));
    o.y = pack2(from_f32<D>(a.z), from_f32<D>(a.w));
    o.z = pack2(from_f32<D>(b.x), from_f32<D>(b.y));
    o.w = pack2(from_f32<D>(b.z), from_f32<D>(b.w));
    *reinterpret_cast<uint4*>(dst) = o;
  } else {
#pragma unroll
    for (int i = 0; i < VE; ++i) dst[i] = convert_elem<S, D>(src[i]);
  }
}

// One 16-byte cache vector (16 / sizeof(CT) elements) read from an aligned
// source run and converted.
template <class S, class D>
__device__ __forceinline__ uint4 load_vec16(const typename Elem<S>::storage* __restrict__ src) {
  constexpr int VE = 16 / Elem<D>::kBytes;
  if constexpr (std::is_same<S, D>::value) {
    return *reinterpret_cast<const uint4*>(src);
  } else {
    typename Elem<D>::storage t[VE];
    convert_run<S, D, VE, true>(src, t);
    return *reinterpret_cast<const uint4*>(t);
  }
}

typedef unsigned int u32x4_t __attribute__((ext_vector_type(4)));
typedef unsigned int u32x2_t __attribute__((ext_vector_type(2)));

// ---- FP8 caches: E4M3 codes of x / scale (pkv_fp8.h) -------------------------------
// Eight source elements -> eight codes.
template <class KT>
__device__ __forceinline__ uint2 encode8(const typename Elem<KT>::storage* __restrict__ src, const Fp8Scale& s) {
  float v[8];
  if constexpr (std::is_same<KT, F32>::value) {
    const float4 a = reinterpret_cast<const float4*>(src)[0], b = reinterpret_cast<const float4*>(src)[1];
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
  } else {
    const uint4 w = *reinterpret_cast<const uint4*>(src);
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = to_f32<KT>((uint16_t)(u[i] & 0xffffu));
      v[2 * i + 1] = to_f32<KT>((uint16_t)(u[i] >> 16));
    }
  }
  return make_uint2(fp8_encode4_scaled(v, s), fp8_encode4_scaled(v + 4, s));
}

// Batch positions of a window that each wavefront needs: the run that started
// in the previous window (prev) and the one that starts in this window (run),
// -1 if there is none; every lane gets the same values.  slot: the slot of
// token (window - 1) * BS + lane, -1 outside the batch.
template <int BS>
__device__ __forceinline__ void rac_window_runs(const RacParams& p, int64_t window, int lane, int64_t& prev,
                                                int64_t& run, int& slot) {
  const int64_t base = (window - 1) * BS;  // the lanes look at [base, base + 3 BS)
  // Bit i: token base + i's slot is followed by its successor's.
  auto links = [&](int64_t pos, int& slot) -> uint64_t {
    slot = pos >= 0 && pos < p.num_tokens ? p.slot_mapping[pos] : -1;
    const int next = pos >= 0 && pos + 1 < p.num_tokens ? p.slot_mapping[pos + 1] : -1;
    return __ballot(slot >= 0 && slot < INT32_MAX && next == slot + 1);
  };
  int unused;
  const uint64_t lo = links(base + lane, slot);
  uint64_t follow = lo >> lane;
  if constexpr (3 * BS > 64) {
    const uint64_t hi = links(base + 64 + lane, unused);
    if (lane > 0) follow |= hi << (64 - lane);
  }
  constexpr uint64_t kAll = ((uint64_t)1 << (BS - 1)) - 1;
  const bool starts = lane < 2 * BS && slot >= 0 && slot % BS == 0 && (int64_t)slot + BS <= p.num_slots &&
                      (follow & kAll) == kAll;
  const uint64_t m = __ballot(starts);
  constexpr uint64_t kWin = ((uint64_t)1 << BS) - 1;
  const uint64_t mp = m & kWin, mr = (m >> BS) & kWin;
  prev = mp ? base + __builtin_ctzll(mp) : -1;
  run = mr ? base + BS + __builtin_ctzll(mr) : -1;
}

// Eight cache elements of a source run: one 16-byte vector (16-bit caches)
// or 8 code bytes (FP8).
template <class CT> struct Vec8 { using type = uint4; };
template <> struct Vec8<FP8> { using type = uint2; };

template <class KT, class CT>
__device__ __forceinline__ typename Vec8<CT>::type load8(const typename Elem<KT>::storage* src, const Fp8Scale& s) {
  if constexpr (std::is_same<CT, FP8>::value)
    return encode8<KT>(src, s);
  else
    return load_vec16<KT, CT>(src);
}

template <bool NT> __device__ __forceinline__ void store8(void* dst, uint4 v) {
  if constexpr (NT)
    __builtin_nontemporal_store(__builtin_bit_cast(u32x4_t, v), reinterpret_cast<u32x4_t*>(dst));
  else
    *reinterpret_cast<uint4*>(dst) = v;
}
template <bool NT> __device__ __forceinline__ void store8(void* dst, uint2 v) {
  if constexpr (NT)
    __builtin_nontemporal_store(__builtin_bit_cast(u32x2_t, v), reinterpret_cast<u32x2_t*>(dst));
  else
    *reinterpret_cast<uint2*>(dst) = v;
}

// Two neighbouring source elements as floats (or raw 16-bit words when the
// cache has the source's type).
template <class KT> struct Pair { float a, b; };
template <class KT>
__device__ __forceinline__ Pair<KT> load_pair(const typename Elem<KT>::storage* src) {
  if constexpr (std::is_same<KT, F32>::value) {
    const float2 x = *reinterpret_cast<const float2*>(src);
    return {x.x, x.y};
  } else {
    const uint32_t w = *reinterpret_cast<const uint32_t*>(src);
    return {to_f32<KT>((uint16_t)(w & 0xffffu)), to_f32<KT>((uint16_t)(w >> 16))};
  }
}

// A V task's four tokens of two dimensions -> eight tokens of one: this
// lane's four of dimension d0 + (lane & 1) and its neighbour's.  (Both
// dimensions are exchanged and the lane keeps one: the exchange then reads
// registers as loaded, never a select's result.)
__device__ __forceinline__ uint32_t swap_pair(uint32_t x) {
  constexpr int kSwap1 = 1 | (0 << 2) | (3 << 4) | (2 << 6);  // quad_perm: lane ^ 1
  return (uint32_t)__builtin_amdgcn_mov_dpp((int)x, kSwap1, 0xf, 0xf, false);
}

template <class KT, class CT>
__device__ __forceinline__ typename Vec8<CT>::type load_v_task(const typename Elem<KT>::storage* src, int64_t stride,
                                                               bool odd, const Fp8Scale& s) {
  if constexpr (std::is_same<CT, FP8>::value) {
    float x[8];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const Pair<KT> w = load_pair<KT>(src + e * stride);
      x[e] = w.a;
      x[4 + e] = w.b;
    }
    const uint32_t d0 = fp8_encode4_scaled(x, s), d1 = fp8_encode4_scaled(x + 4, s);
    const uint32_t s0 = swap_pair(d0), s1 = swap_pair(d1);
    return odd ? make_uint2(s1, d1) : make_uint2(d0, s0);
  } else {
    uint32_t w[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if constexpr (std::is_same<KT, CT>::value) {
        w[e] = *reinterpret_cast<const uint32_t*>(src + e * stride);
      } else {
        const Pair<KT> x = load_pair<KT>(src + e * stride);
        w[e] = pack2(from_f32<CT>(x.a), from_f32<CT>(x.b));
      }
    }
    // Low halves: dimension d0 of tokens 0 1 | 2 3; high halves: d0 + 1.
    const uint2 d0 = make_uint2(__builtin_amdgcn_perm(w[1], w[0], 0x05040100u),
                                __builtin_amdgcn_perm(w[3], w[2], 0x05040100u));
    const uint2 d1 = make_uint2(__builtin_amdgcn_perm(w[1], w[0], 0x07060302u),
                                __builtin_amdgcn_perm(w[3], w[2], 0x07060302u));
    const uint2 s0 = make_uint2(swap_pair(d0.x), swap_pair(d0.y)), s1 = make_uint2(swap_pair(d1.x), swap_pair(d1.y));
    return odd ? make_uint4(s1.x, s1.y, d1.x, d1.y) : make_uint4(d0.x, d0.y, s0.x, s0.y);
  }
}

}  // namespace pkv
