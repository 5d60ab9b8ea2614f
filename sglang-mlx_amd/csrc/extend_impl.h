// Attention of new tokens over a paged KV cache, causal, over the whole context
// or over a sliding window and the context's first tokens.
//
// Sequence s brings n query tokens, the last n of its c tokens: query i sits at
// position p = c - n + i and sees the keys t <= p, of them only those with
// t > p - window or t < sinks where there is a window.  A query row is one
// (token, head); the rows of the heads that share a KV head are attended
// together, row r of a sequence being head r % group of token r / group.
//
// Both kernels compute S^T = K Q^T and O^T = V^T P^T, so that a query row is a
// column of every matrix: a lane holds scores, weights and outputs of one row
// only, the running maximum and sum of its softmax are one register each, and a
// tile's weights leave the score product in the lanes where the second product
// wants them.  For that the K rows of a tile are taken in an order that gives
// each lane the weights of consecutive tokens (see the kernels), which then
// meet V's paged layout, [D][block_size], in whole 16-byte loads.
//
// Weights are rounded to the queries' 16-bit type for the second product (the
// matrix units take no other), their sum is of the float32 weights.  bfloat16 has
// float32's exponents, so that a small weight keeps as many bits as a large one;
// float16's normal range ends at 2^-14, so its weights are scaled by a constant power
// of two that brings the largest to at most 2^15 (the sum has the same factor, and
// the division by it takes both out).  Without it thousands of light tokens beside
// one heavy one lost their low bits, or all, together: 8 % of the share, 0.6 %, of
// 32768 tokens 2^22.3 times lighter than one.
#pragma once

#include "pkv_fp8.h"
#include "pkv_launch.h"

namespace pkv {

typedef float f32x16 __attribute__((ext_vector_type(16)));

// D[32x32] += A[32x16] * B[16x32]: lane l supplies A[l % 32][8 (l / 32) ..+7]
// and B[8 (l / 32) ..+7][l % 32]; register r of lane l is
// D[r % 4 + 8 (r / 4) + 4 (l / 32)][l % 32].
template <class T> __device__ __forceinline__ f32x16 mma32(uint4 a, uint4 b, f32x16 c);
template <> __device__ __forceinline__ f32x16 mma32<BF16>(uint4 a, uint4 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0,
                                                 0);
}
template <> __device__ __forceinline__ f32x16 mma32<F16>(uint4 a, uint4 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0,
                                                0);
}

// Two weights (finite, not negative) as 16-bit elements, rounded to nearest even.
template <class T> __device__ __forceinline__ uint32_t pack_weights(float a, float b);
template <> __device__ __forceinline__ uint32_t pack_weights<BF16>(float a, float b) {
  typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
  bf16x2 v;
  v[0] = (__bf16)a;
  v[1] = (__bf16)b;
  return __builtin_bit_cast(uint32_t, v);
}
template <> __device__ __forceinline__ uint32_t pack_weights<F16>(float a, float b) {
  typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
  f16x2 v;
  v[0] = (_Float16)a;
  v[1] = (_Float16)b;
  return __builtin_bit_cast(uint32_t, v);
}

// The power of two by which a weight of 2^most at the most is scaled.
template <class T> constexpr float weight_shift(float most) { return std::is_same<T, F16>::value ? 15.f - most : 0.f; }

// Keeps the elements of eight 16-bit ones whose bit is set.
__device__ __forceinline__ uint4 keep8(uint4 v, uint32_t bits) {
  auto m = [&](int i) {
    return ((bits >> (2 * i)) & 1u ? 0xffffu : 0u) | ((bits >> (2 * i + 1)) & 1u ? 0xffff0000u : 0u);
  };
  return make_uint4(v.x & m(0), v.y & m(1), v.z & m(2), v.w & m(3));
}

// Eight elements of an FP8 cache as 16-bit ones.  special: the wavefront has a
// code with exponent 15 among those that it converts (the hardware conversion is
// right for all others).
template <class T> __device__ __forceinline__ uint4 decode8(uint2 codes, bool special) {
  const uint2 a = special ? fp8x4_exact_inline<T>(codes.x) : fp8x4_cvt<T>(codes.x);
  const uint2 b = special ? fp8x4_exact_inline<T>(codes.y) : fp8x4_cvt<T>(codes.y);
  return make_uint4(a.x, a.y, b.x, b.y);
}

constexpr float kNoScore = -__builtin_inff();

// States that cross workgroups inside one launch travel by agent-scope relaxed
// atomic accesses, each coherent at agent scope by itself (the L2 caches are per
// XCD and not coherent with one another for ordinary accesses); a workgroup
// counts its arrival only when its stores have completed.
__device__ __forceinline__ void store_agent(float* p, float a, float b) {
  const uint64_t v = (uint64_t)__float_as_uint(a) | ((uint64_t)__float_as_uint(b) << 32);
  __hip_atomic_store(reinterpret_cast<uint64_t*>(p), v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float2 load_agent(const float* p) {
  const uint64_t v =
      __hip_atomic_load(reinterpret_cast<const uint64_t*>(p), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  return make_float2(__uint_as_float((uint32_t)v), __uint_as_float((uint32_t)(v >> 32)));
}
__device__ __forceinline__ void wait_agent_stores() {
  __atomic_signal_fence(__ATOMIC_SEQ_CST);
  __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0); expcnt and lgkmcnt left at their maxima
  __atomic_signal_fence(__ATOMIC_SEQ_CST);
}
// Counts one arrival; true for the expected-th, which sets the counter back to
// zero (every arrival of the launch has happened by then).
__device__ __forceinline__ bool arrived_last(int32_t* counter, int expected) {
  const bool last = __hip_atomic_fetch_add(counter, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == expected - 1;
  if (last) __hip_atomic_store(counter, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  return last;
}

// What a sequence brings to this call.
struct ExtendSeq {
  int start, count;  // query rows [start, start + count) of the batch
  int ctx;           // 0: nothing to attend (every row is zero)
};
__device__ __forceinline__ ExtendSeq extend_seq(const ExtendParams& p, int s) {
  ExtendSeq q;
  if (p.query_start_loc != nullptr) {
    q.start = min(max(p.query_start_loc[s], 0), p.num_tokens);
    q.count = min(max(p.query_start_loc[s + 1], q.start), p.num_tokens) - q.start;
  } else {
    q.start = s;
    q.count = 1;
  }
  const uint32_t c = (uint32_t)p.context_lens[s];
  q.ctx = c > (uint32_t)p.max_seq_len || q.count > p.max_query_len ? 0 : (int)c;
  return q;
}

// Zeroes tokens [t0, t1) of the output, heads [h0, h0 + nh), by all threads of the
// workgroup, 16 bytes a lane.
template <class QT, int NT>
__device__ __forceinline__ void zero_tokens(const ExtendParams& p, int D, int64_t t0, int64_t t1, int h0, int nh) {
  using QS = typename Elem<QT>::storage;
  const int per = nh * (D / 8);  // pieces of a token
  const int tokens = NT / per, rest = NT - tokens * per;
  int64_t t = t0 + (int)threadIdx.x / per;
  int piece = (int)threadIdx.x % per;
  for (; t < t1; t += tokens) {
    *reinterpret_cast<uint4*>(static_cast<QS*>(p.out) + (t * p.num_heads + h0) * D + 8 * piece) = make_uint4(0, 0, 0, 0);
    piece += rest;
    if (piece >= per) piece -= per, ++t;
  }
}

// ---------------------------------------------------------------------------
// Tiles of query rows: one workgroup per (128 rows of a sequence, KV head,
// split), four wavefronts of 32 rows.
//
// A tile of 64 tokens of K and V lies in LDS as the matrix units read it: K as
// [token group of 16][D / 8][16 tokens][8], V as [token group of 8][D][8].  Both
// are gathers of 16-byte pieces of the paged layout: 16-bit caches go there by
// direct-to-LDS loads, a tile ahead of the one in use; FP8 codes pass through
// registers and become 16-bit elements.  A load takes its pieces from one block
// (K of 8-token blocks: from two), so that its address is a scalar and a lane
// offset that stays: with an address per lane and load the vector unit spent
// 110 of 243 instructions a tile on them.
//
// Row rho of a 32-token score product is token 16 (rho / 4 % 2) + 4 (rho / 8) +
// rho % 4, so that register r of half h is token 16 h + r.  Reads of both images
// meet no bank twice: counted conflicts are 0, where K's groups 64 or 128 bytes
// further apart than they are long took half as many LDS cycles again.
//
// Tiles that every row of a wavefront sees in full take no mask; a wavefront
// skips tiles that none of its rows sees.
//
// Bound: neither unit, but their order: a wavefront's products wait for its softmax,
// and all for the tile's barrier.  8192 new tokens on 8192, 32 heads of 128, bf16,
// take 1.70 - 1.76 ms, 940 - 970 TFLOP/s of the 1381 that a large matrix product
// reaches, the matrix units busy 43 % and the vector units 42 % of the time; 32-token
// tiles in four stages with the softmax of one beside the products of the next came
// to 952 TFLOP/s.  128 rows let two workgroups share a CU (three at head sizes up to
// 64, none above 128), so that one computes while another waits.  At head size 64 the
// third costs spills, 40 bytes a lane (FP8 caches 56), and still pays (launch_extend_d).
// ---------------------------------------------------------------------------
constexpr int kExtendTile = 64;
constexpr int kExtendThreads = 256;
// A row's reference point moves only when its maximum passes it by this much
// (log2), so that most tiles leave the outputs unscaled.  Weights then stay below
// 2^8, which changes no rounding of bfloat16; float16 leaves less of its range to it
// (8192 new tokens on 8192, float16: 1.82 ms, with 8 and unscaled weights 1.79).
template <class T> constexpr float kExtendSlack = std::is_same<T, F16>::value ? 4.f : 8.f;

// Bit r of 16: a query at position pos sees token a + r.
__device__ __forceinline__ uint32_t seen16(int pos, int a, int window, int sinks) {
  auto below = [](int n) { return n <= 0 ? 0u : n >= 16 ? 0xffffu : (1u << n) - 1u; };  // the first n
  return below(pos + 1 - a) & (~below(pos - window + 1 - a) | below(sinks - a));
}

// What lanes without a token load in its place.
static __device__ const uint4 kNothing = {0, 0, 0, 0};

// 16 bytes per lane, memory -> LDS at dst + 16 lane.
__device__ __forceinline__ void load_to_lds(const void* src, uint4* dst) {
  __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)src,
                                   (__attribute__((address_space(3))) void*)dst, 16, 0, 0);
}

template <class QT, class CT, int D>
__global__ __launch_bounds__(kExtendThreads, D <= 64 ? 3 : D <= 128 ? 2 : 1) void extend_kernel(ExtendParams p) {
  using QS = typename Elem<QT>::storage;
  using CS = typename Elem<CT>::storage;
  constexpr bool F8 = std::is_same<CT, FP8>::value;
  constexpr int KSTEPS = (D + 15) / 16;  // score products per 32 tokens
  constexpr int DT = (D + 31) / 32;      // 32-dimension tiles of the output
  constexpr int DK = KSTEPS * 2;         // 8-dimension chunks staged
  constexpr int DV = DT * 32;            // dimensions of V staged
  constexpr int KG = DK * 16;            // 16-byte pieces from one token group of K's image to the next
  constexpr int VU = DV / 8;             // 64-lane loads of a tile of V
  // Two stages, arrays of their own: the compiler then knows that the loads in
  // flight do not touch what is read.
  __shared__ uint4 s_k0[4 * KG], s_k1[4 * KG];
  __shared__ uint4 s_v0[8 * DV], s_v1[8 * DV];
  __shared__ int s_seq[3], s_again;
  using I0 = std::integral_constant<int, 0>;
  using I1 = std::integral_constant<int, 1>;
  auto k_image = [&](auto k) __attribute__((always_inline)) -> uint4* {
    if constexpr (decltype(k)::value == 0) return s_k0;
    else return s_k1;
  };
  auto v_image = [&](auto k) __attribute__((always_inline)) -> uint4* {
    if constexpr (decltype(k)::value == 0) return s_v0;
    else return s_v1;
  };

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 31, half = lane >> 5;
  const int kvh = blockIdx.x % p.num_kv_heads;
  const int item = blockIdx.x / p.num_kv_heads;
  const int items = gridDim.x / p.num_kv_heads;
  const int split = blockIdx.y;
  const int group = p.group, h0 = kvh * group;

  // The workgroup's sequence and row tile: tiles of the sequences lie end to
  // end, a sequence's last tile (the longest) first.
  if (wave == 0) {
    int base = 0, found = -1, z = 0;
    for (int s0 = 0; s0 < p.num_seqs; s0 += 64) {
      const int s = s0 + lane;
      int tiles = 0;
      if (s < p.num_seqs) tiles = (extend_seq(p, s).count * group + kExtendRows - 1) / kExtendRows;
      int sum = tiles;
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) {
        const int a = __shfl_up(sum, d);
        if (lane >= d) sum += a;
      }
      const uint64_t past = __ballot(base + sum > item);
      if (past) {
        const int w = __builtin_ctzll(past);
        found = s0 + w;
        z = base + __shfl(sum, w) - 1 - item;  // counted from the sequence's first tile
        break;
      }
      base += __shfl(sum, 63);
    }
    if (lane == 0) s_seq[0] = found, s_seq[1] = z, s_seq[2] = base, s_again = 0;
  }
  __syncthreads();
  const int seq = __builtin_amdgcn_readfirstlane(s_seq[0]);
  if (seq < 0) {
    // Past the last tile: rows behind the last sequence become zeros.
    const int tiles = s_seq[2];
    if (split != 0) return;
    const int last = p.query_start_loc ? min(max(p.query_start_loc[p.num_seqs], 0), p.num_tokens) : p.num_seqs;
    const int share = (p.num_tokens - last + items - tiles - 1) / (items - tiles);
    const int64_t t0 = last + (int64_t)(item - tiles) * share;
    zero_tokens<QT, kExtendThreads>(p, D, t0, min(t0 + share, (int64_t)p.num_tokens), h0, group);
    return;
  }
  const int z = __builtin_amdgcn_readfirstlane(s_seq[1]);
  const ExtendSeq q = extend_seq(p, seq);
  const int first_pos = q.ctx - q.count;  // position of the sequence's first query token
  const int rows = q.count * group;
  const int row0 = z * kExtendRows;
  const int row_end = min(row0 + kExtendRows, rows);
  // Positions of the workgroup's rows; tokens before position 0 see nothing.
  const int pmin = first_pos + row0 / group, pmax = first_pos + (row_end - 1) / group;

  // This lane's row.
  const int wr0 = row0 + wave * 32, wr1 = min(wr0 + 32, rows);
  const int row = wr0 + col;
  const bool live = row < rows;
  const int tok = live ? row / group : 0;
  const int head = h0 + (live ? row - tok * group : 0);
  const int64_t qrow = q.start + tok;
  const int pos = live && q.ctx > 0 ? first_pos + tok : -1;
  // Positions of the wavefront's rows (uniform): none where w_min > w_max.
  const bool w_any = wr0 < wr1 && q.ctx > 0;
  const int w_min = w_any ? first_pos + wr0 / group : 0, w_max = w_any ? first_pos + (wr1 - 1) / group : -1;

  // The tiles to visit: those of the sinks, then those of the window.
  const int window = p.window > 0 ? p.window : p.max_seq_len;
  const int sinks = p.window > 0 ? p.sinks : 0;
  int lead = 0, base_tile = 0, ntiles = 0;
  if (q.ctx > 0 && pmax >= 0) {
    const int lo = max(0, max(pmin, 0) - window + 1);
    lead = (min(sinks, lo) + kExtendTile - 1) / kExtendTile;
    base_tile = max(lo / kExtendTile, lead);
    ntiles = lead + max(0, pmax / kExtendTile + 1 - base_tile);
  }
  const int per = (ntiles + p.splits - 1) / p.splits;
  const int v0 = min(split * per, ntiles), v1 = min(v0 + per, ntiles);
  auto tile_start = [&](int v) { return (v < lead ? v : base_tile + v - lead) * kExtendTile; };

  uint4 qf[KSTEPS];
  const uint32_t sign = p.scale_log2 < 0.f ? 0x80008000u : 0u;  // (a negative scale goes into the queries)
  const float scale = fmaxf(__builtin_fabsf(p.scale_log2), 0x1p-120f);
  {
    const QS* src = static_cast<const QS*>(p.q) + qrow * p.q_stride + (int64_t)head * D;
#pragma unroll
    for (int j = 0; j < KSTEPS; ++j) {
      const int d = 16 * j + 8 * half;
      const uint4 x = live && d < D ? *reinterpret_cast<const uint4*>(src + d) : make_uint4(0, 0, 0, 0);
      qf[j] = make_uint4(x.x ^ sign, x.y ^ sign, x.z ^ sign, x.w ^ sign);
    }
  }
  f32x16 o[DT];
  float m, l;
  auto reset = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int r = 0; r < 16; ++r) o[dt][r] = 0.f;
    m = kNoScore;
    l = 0.f;
  };
  reset();

  const int shift = p.block_shift, bs = 1 << shift;
  const int32_t* table = p.block_tables + (int64_t)seq * p.max_blocks_per_seq;
  const CS* kc = static_cast<const CS*>(p.k_cache) + (int64_t)kvh * p.k_head_stride;
  const CS* vc = static_cast<const CS*>(p.v_cache) + (int64_t)kvh * p.v_head_stride;

  // The block of 8-token group lane % 8 of tile v, -1 past the context, outside
  // the pool or past the last tile.
  auto load_bid = [&](int v) __attribute__((always_inline)) {
    int32_t bid = -1;
    if (v < v1) {
      const int t = tile_start(v) + 8 * (lane & 7);
      if (t < q.ctx) bid = table[t >> shift];
    }
    return bid >= 0 && (int64_t)bid < p.num_blocks ? bid : -1;
  };
  // Wavefront w stages token group w of K: a load is four chunks (FP8: four of
  // 16) of 16 tokens.  A missing block's tokens are masked: any block will do.
  constexpr int KL = F8 ? (D / 16 + 3) / 4 : (DK + 3) / 4;
  constexpr int X = 16 / Elem<CT>::kBytes;
  const int k_chunk = lane >> 4, k_tok = lane & 15;
  // FP8: a tile's codes on their way to LDS.
  constexpr int FK = F8 ? KL : 1, FV = F8 ? (VU + 3) / 4 : 1;
  uint4 fk[FK] = {};
  uint2 fv[FV] = {};
  // Issues the loads of the tile at t0, whose groups' blocks are bid.
  auto stage = [&](auto k, int t0, int32_t bid) __attribute__((always_inline)) {
    auto load_k = [&](const CS* base, int at) __attribute__((always_inline)) {  // at: this lane's token in the block
#pragma unroll
      for (int j = 0; j < KL; ++j) {
        const CS* src = base + 4 * j * X * bs + (k_chunk * bs + at) * X;
        if constexpr (F8) {
          fk[j] = make_uint4(0, 0, 0, 0);
          if ((D / 16) % 4 == 0 || 4 * j + k_chunk < D / 16) fk[j] = *reinterpret_cast<const uint4*>(src);
        } else {
          // (The image of a head size that 16 does not divide ends in a chunk of
          // zeros, that of one that 32 does not in half a load.)
          const bool have = D % 32 == 0 || (4 * j + k_chunk) * 8 < D;
          if (D % 32 == 0 || 4 * j + k_chunk < DK)
            load_to_lds(have ? (const void*)src : (const void*)&kNothing, k_image(k) + wave * KG + 64 * j);
        }
      }
    };
    const int kt = (t0 + 16 * wave) & (bs - 1);
    if (bs >= 16) {
      const int b = max(__builtin_amdgcn_readlane(bid, 2 * wave), 0);
      load_k(kc + (int64_t)b * p.k_block_stride + kt * X, k_tok);
    } else {
      const int b = max(__shfl(bid, 2 * wave + (k_tok >> 3)), 0);
      load_k(kc + (int64_t)b * p.k_block_stride, k_tok & 7);
    }
#pragma unroll
    for (int j = 0; j < (VU + 3) / 4; ++j) {
      const int u0 = (4 * j + wave) * 64;
      if (VU % 4 != 0 && u0 >= 8 * DV) continue;
      auto load_v = [&](const CS* src, bool have) __attribute__((always_inline)) {
        if constexpr (!F8) {
          load_to_lds(have ? (const void*)src : (const void*)&kNothing, v_image(k) + u0);
        } else {
          fv[j] = make_uint2(0, 0);
          if (have) fv[j] = *reinterpret_cast<const uint2*>(src);
        }
      };
      if constexpr (DV % 64 == 0) {
        const int tg = u0 / DV, d = u0 % DV + lane;
        const int b = __builtin_amdgcn_readlane(bid, tg);
        const CS* base = vc + (int64_t)b * p.v_block_stride + ((t0 + 8 * tg) & (bs - 1));
        if (b >= 0)
          load_v(base + d * bs, D % 64 == 0 || d < D);
        else
          load_v(nullptr, false);
      } else {
        const int u = u0 + lane, tg = u / DV, d = u - tg * DV;
        const int b = __shfl(bid, tg);
        load_v(vc + (int64_t)max(b, 0) * p.v_block_stride + (d * bs + ((t0 + 8 * tg) & (bs - 1))), b >= 0 && d < D);
      }
    }
  };
  auto finish_stage = [&](auto k) __attribute__((always_inline)) {
    if constexpr (F8) {
      uint32_t probe = 0;
#pragma unroll
      for (int j = 0; j < FK; ++j)
        probe |= fp8x4_special(fk[j].x) | fp8x4_special(fk[j].y) | fp8x4_special(fk[j].z) | fp8x4_special(fk[j].w);
#pragma unroll
      for (int j = 0; j < FV; ++j) probe |= fp8x4_special(fv[j].x) | fp8x4_special(fv[j].y);
      auto write = [&](bool special) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < FK; ++j) {
          const int c = 4 * j + k_chunk;
          if ((D / 16) % 4 == 0 || c < D / 16) {
            uint4* dst = k_image(k) + wave * KG + 2 * c * 16 + k_tok;
            dst[0] = decode8<QT>(make_uint2(fk[j].x, fk[j].y), special);
            dst[16] = decode8<QT>(make_uint2(fk[j].z, fk[j].w), special);
          }
        }
#pragma unroll
        for (int j = 0; j < FV; ++j) {
          const int u0 = (4 * j + wave) * 64;
          if (VU % 4 == 0 || u0 < 8 * DV) v_image(k)[u0 + lane] = decode8<QT>(fv[j], special);
        }
      };
      if (__any(probe != 0u))
        write(true);
      else
        write(false);
    }
  };
  // The workgroup meets at a bare s_barrier, each wavefront's own loads and LDS
  // accesses awaited before (a __syncthreads would do the same).
  auto meet = [] __attribute__((always_inline)) {
    __builtin_amdgcn_s_waitcnt(0x0070);  // vmcnt(0) lgkmcnt(0)
    asm volatile("s_barrier" ::: "memory");
  };

  // Bit r: the block of token 32 sub + 16 half + r of the tile is in the pool.
  auto held = [&](uint32_t ok, int sub) {
    const uint32_t g = ok >> (4 * sub + 2 * half);
    return (g & 1u ? 0xffu : 0u) | (g & 2u ? 0xff00u : 0u);
  };
  // The tile at t0, in image k.  whole: every row of the wavefront sees all of it.
  // CAREFUL: what a row does not see is kept out of its products.
  auto attend = [&](auto k, auto careful, bool whole, int t0, uint32_t ok) __attribute__((always_inline)) {
    constexpr bool CAREFUL = decltype(careful)::value;
    // (K: group (col / 4) % 2 of a pair, its token 4 (col / 8) + col % 4.)
    const uint4* ki = k_image(k) + ((col >> 2) & 1) * KG + half * 16 + 4 * (col >> 3) + (col & 3);
    const uint4* vi = v_image(k) + 2 * half * DV + col;
    f32x16 s[2];
#pragma unroll
    for (int sub = 0; sub < 2; ++sub) {
#pragma unroll
      for (int r = 0; r < 16; ++r) s[sub][r] = 0.f;
#pragma unroll
      for (int j = 0; j < KSTEPS; ++j) s[sub] = mma32<QT>(ki[2 * sub * KG + 32 * j], qf[j], s[sub]);
    }
    if (!whole) {
#pragma unroll
      for (int sub = 0; sub < 2; ++sub) {
        const uint32_t sees = seen16(pos, t0 + 32 * sub + 16 * half, window, sinks) & held(ok, sub);
#pragma unroll
        for (int r = 0; r < 16; ++r) s[sub][r] = sees >> r & 1u ? s[sub][r] : kNoScore;
      }
    }
    float mt = kNoScore;
#pragma unroll
    for (int sub = 0; sub < 2; ++sub)
#pragma unroll
      for (int r = 0; r < 16; ++r) mt = fmaxf(mt, s[sub][r]);
    mt = fmaxf(xchg32_max(mt), m);
    if (__any(mt * scale > m * scale + kExtendSlack<QT> || (m == kNoScore && mt != kNoScore))) {
      const float alpha = mt == kNoScore ? 1.f : __builtin_amdgcn_exp2f((m - mt) * scale);
      m = mt;
      l *= alpha;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[dt][r] *= alpha;
    }
    // (A row that has seen nothing keeps a finite reference point: no inf - inf.)
    const float ref = (m == kNoScore ? 0.f : m * scale) - weight_shift<QT>(kExtendSlack<QT>);
    uint32_t w[2][8];
    auto exponentials = [&](int sub) __attribute__((always_inline)) {
#pragma unroll
      for (int r = 0; r < 16; r += 2) {
        const float a = __builtin_amdgcn_exp2f(__builtin_fmaf(s[sub][r], scale, -ref));
        const float b = __builtin_amdgcn_exp2f(__builtin_fmaf(s[sub][r + 1], scale, -ref));
        l += a + b;
        w[sub][r / 2] = pack_weights<QT>(a, b);
      }
    };
    auto v_piece = [&](int dt, int sub, int k8) {  // tokens 32 sub + 16 half + 8 k8 ..+7 of dimension 32 dt + col
      return vi[(4 * sub + k8) * DV + 32 * dt];
    };
    auto weights = [&](int sub, int k8) {
      return make_uint4(w[sub][4 * k8], w[sub][4 * k8 + 1], w[sub][4 * k8 + 2], w[sub][4 * k8 + 3]);
    };
    auto products = [&](int sub) __attribute__((always_inline)) {
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int k8 = 0; k8 < 2; ++k8) o[dt] = mma32<QT>(v_piece(dt, sub, k8), weights(sub, k8), o[dt]);
    };
    exponentials(0);
    if constexpr (!CAREFUL) {
      products(0);
      exponentials(1);
      products(1);
    } else {
      exponentials(1);
      // One query position at a time, with the tokens that it does not see taken
      // out of V; the other positions' rows keep their sums.
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll 1
        for (int at = w_min; at <= w_max; ++at)
#pragma unroll
          for (int sub = 0; sub < 2; ++sub) {
            const uint32_t keep = seen16(at, t0 + 32 * sub + 16 * half, window, sinks);
            const uint4 va = keep8(v_piece(dt, sub, 0), keep), vb = keep8(v_piece(dt, sub, 1), keep >> 8);
            f32x16 n = mma32<QT>(va, weights(sub, 0), o[dt]);
            n = mma32<QT>(vb, weights(sub, 1), n);
#pragma unroll
            for (int r = 0; r < 16; ++r) o[dt][r] = pos == at ? n[r] : o[dt][r];
          }
    }
    if (!CAREFUL && !whole) {
      // A token that some rows do not see must not reach them, whatever its
      // value, but a weight of 0 times inf or NaN is NaN.  The product with zeros
      // tells whether the tile has such a value: the rows are then done again.
      f32x16 zero;
#pragma unroll
      for (int r = 0; r < 16; ++r) zero[r] = 0.f;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int j = 0; j < 4; ++j) zero = mma32<QT>(v_piece(dt, j >> 1, j & 1), make_uint4(0, 0, 0, 0), zero);
      float sum = 0.f;
#pragma unroll
      for (int r = 0; r < 16; ++r) sum += zero[r];
      if (__any(sum != 0.f)) s_again = 1;
    }
  };
  auto consume = [&](auto k, auto careful, int t0, uint32_t ok) __attribute__((always_inline)) {
    // Whether any of the wavefront's rows sees a token of the tile, and whether all see all.
    if (w_max < t0 || !(t0 < sinks || t0 + kExtendTile > w_min - window + 1)) return;
    // (Lanes without a row compute on zero queries and store nothing.)
    const bool whole =
        t0 + kExtendTile - 1 <= w_min && (t0 > w_max - window || t0 + kExtendTile <= sinks) && ok == 0xffu;
    attend(k, careful, whole, t0, ok);
  };

  // Takes the tokens past the context out of the last tile's image of V (K's are
  // masked out): the 8-token group in which the context ends was loaded whole.
  auto trim = [&](auto k, int t0) __attribute__((always_inline)) {
    if (t0 + kExtendTile <= q.ctx || q.ctx % 8 == 0) return;
    uint4* group8 = v_image(k) + (q.ctx - t0) / 8 * DV;
    for (int d = tid; d < DV; d += kExtendThreads) group8[d] = keep8(group8[d], (1u << q.ctx % 8) - 1u);
    meet();
  };
  // Tile v is consumed while tile v + 1 loads and the blocks of tile v + 2 are
  // looked up.
  if (v0 < v1) {
    int32_t bid = load_bid(v0), next = load_bid(v0 + 1);
    uint32_t ok = (uint32_t)__ballot(bid >= 0) & 0xffu;
    stage(I0{}, tile_start(v0), bid);
    finish_stage(I0{});
    auto step = [&](auto k, int v) __attribute__((always_inline)) {
      using KN = std::integral_constant<int, decltype(k)::value ^ 1>;
      const int t0 = tile_start(v);
      meet();  // tile v has landed, tile v - 1 has been read
      trim(k, t0);
      const uint32_t ok_next = (uint32_t)__ballot(next >= 0) & 0xffu;
      if (v + 1 < v1) stage(KN{}, tile_start(v + 1), next);
      next = load_bid(v + 2);
      consume(k, std::false_type{}, t0, ok);
      if (v + 1 < v1) finish_stage(KN{});
      ok = ok_next;
    };
    for (int v = v0; v < v1; v += 2) {
      step(I0{}, v);
      if (v + 1 >= v1) break;
      step(I1{}, v + 1);
    }
    meet();
    if (__builtin_expect(s_again, 0)) {
      reset();
#pragma unroll 1
      for (int v = v0; v < v1; ++v) {
        const int t0 = tile_start(v);
        bid = load_bid(v);
        ok = (uint32_t)__ballot(bid >= 0) & 0xffu;
        meet();
        stage(I0{}, t0, bid);
        finish_stage(I0{});
        meet();
        trim(I0{}, t0);
        consume(I0{}, std::true_type{}, t0, ok);
      }
    }
  }

  l = xchg32_sum(l);
  if (!live) return;
  if (p.splits == 1) {
    const float inv = l > 0.f ? p.v_scale / l : l == 0.f ? 0.f : l;  // (NaN stays NaN)
    QS* out = static_cast<QS*>(p.out) + (qrow * p.num_heads + head) * D;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int r = 0; r < 16; r += 4) {
        const int d = 32 * dt + 2 * r + 4 * half;
        if (D % 32 != 0 && d >= D) continue;
        uint2 x;
        x.x = pack2(from_f32<QT>(o[dt][r] * inv), from_f32<QT>(o[dt][r + 1] * inv));
        x.y = pack2(from_f32<QT>(o[dt][r + 2] * inv), from_f32<QT>(o[dt][r + 3] * inv));
        *reinterpret_cast<uint2*>(out + d) = x;
      }
    return;
  }
  const int64_t at = (qrow * p.num_heads + head) * p.splits + split;
  float* wo = p.ws_o + at * D;
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int r = 0; r < 16; r += 4) {
      const int d = 32 * dt + 2 * r + 4 * half;
      if (D % 32 != 0 && d >= D) continue;
      *reinterpret_cast<float4*>(wo + d) = make_float4(o[dt][r], o[dt][r + 1], o[dt][r + 2], o[dt][r + 3]);
    }
  if (half == 0) *reinterpret_cast<float2*>(p.ws_ml + at * 2) = make_float2(m * scale, l);
}

// The outputs of a call whose row tiles are split: one wavefront per query row.
template <class QT, int D>
__global__ __launch_bounds__(256) void extend_merge_kernel(ExtendParams p) {
  using QS = typename Elem<QT>::storage;
  const int lane = threadIdx.x & 63;
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);  // token * heads + head
  if (row >= (int64_t)p.num_tokens * p.num_heads) return;
  if (p.query_start_loc != nullptr && row / p.num_heads >= max(p.query_start_loc[p.num_seqs], 0))
    return;  // a row behind the last sequence: the tiles' kernel zeroed it
  const float* ml = p.ws_ml + row * p.splits * 2;
  const float* wo = p.ws_o + row * p.splits * D;
  float m = kNoScore;
  for (int i = 0; i < p.splits; ++i) m = fmaxf(m, ml[2 * i]);
  const float ref = m == kNoScore ? 0.f : m;
  float l = 0.f, o[(D + 63) / 64];
#pragma unroll
  for (int k = 0; k < (D + 63) / 64; ++k) o[k] = 0.f;
  for (int i = 0; i < p.splits; ++i) {
    const float f = __builtin_amdgcn_exp2f(ml[2 * i] - ref);
    l += f * ml[2 * i + 1];
#pragma unroll
    for (int k = 0; k < (D + 63) / 64; ++k)
      if (lane + 64 * k < D) o[k] += f * wo[(int64_t)i * D + lane + 64 * k];
  }
  const float inv = l > 0.f ? p.v_scale / l : l == 0.f ? 0.f : l;
  QS* out = static_cast<QS*>(p.out) + row * D;
#pragma unroll
  for (int k = 0; k < (D + 63) / 64; ++k)
    if (lane + 64 * k < D) out[lane + 64 * k] = from_f32<QT>(o[k] * inv);
}

// ---------------------------------------------------------------------------
// Few query rows per sequence (decodes, drafted tokens): one workgroup per
// (sequence, 16 rows of a KV head, part of the length), four wavefronts that take
// tiles of 32 tokens in turn, K and V from the cache straight into the matrix
// units' registers.
//
// Row i of score product u (of two) is token 8 (i / 4) + 4 u + i % 4, so that
// the registers of both products in lane group g are tokens 8 g ..+7.
//
// ONE: a sequence has one token, whose heads all see the same keys.
//
// Bound: HBM reads of K and V.  128 sequences, window 4000, fp16: 141 us, 5.3 TB/s;
// 64 sequences, window 1024, FP8: 32 us, 4.2 TB/s; one sequence, window 4096:
// 11 us, of which the reads take 4 and the launch, the chain context length ->
// block -> tile, and the merge of the parts the rest.
// ---------------------------------------------------------------------------
constexpr int kWindowTile = 32;

template <class QT, class CT, int D, bool ONE>
__global__ __launch_bounds__(256, D <= 128 ? 2 : 1) void extend_few_kernel(ExtendParams p) {
  using QS = typename Elem<QT>::storage;
  using CS = typename Elem<CT>::storage;
  constexpr bool F8 = std::is_same<CT, FP8>::value;
  constexpr int X = F8 ? 16 : 8;  // elements of a 16-byte K chunk
  constexpr int KSTEPS = F8 ? (D + 63) / 64 * 2 : (D + 31) / 32;
  constexpr int DT = (D + 15) / 16;
  __shared__ float s_o[4][DT * 4][64];
  __shared__ float s_m[4][16], s_l[4][16];
  __shared__ int s_last;

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g = lane >> 4, col = lane & 15;
  const int unit = blockIdx.x % p.units;
  const int seq = blockIdx.x / p.units;
  const int split = blockIdx.y;
  const int kvh = unit / p.slices, slice = unit - kvh * p.slices;
  const int group = p.group, h0 = kvh * group;
  if (seq >= p.num_seqs) {
    // Rows behind the last sequence become zeros.
    const int last = min(max(p.query_start_loc[p.num_seqs], 0), p.num_tokens);
    const int groups = (gridDim.x - p.num_seqs * p.units) * gridDim.y;
    const int share = (p.num_tokens - last + groups - 1) / groups;
    const int64_t t0 = last + (int64_t)((blockIdx.x - p.num_seqs * p.units) * gridDim.y + split) * share;
    zero_tokens<QT, 256>(p, D, t0, min(t0 + share, (int64_t)p.num_tokens), 0, p.num_heads);
    return;
  }
  const ExtendSeq q = extend_seq(p, seq);
  if (q.count == 0) return;
  if (q.ctx == 0) {
    if (split == 0 && slice == 0) zero_tokens<QT, 256>(p, D, q.start, q.start + q.count, h0, group);
    return;
  }
  // Row row0 + c, c < nr, is head (row0 + c) % group of token (row0 + c) / group;
  // this lane's is c = col.
  const int row0 = 16 * slice, nr = min(16, q.count * group - row0);
  if (nr <= 0) return;
  const int first_pos = q.ctx - q.count;
  const int pmin = first_pos + row0 / group, pmax = first_pos + (row0 + nr - 1) / group;  // (uniform)
  const bool live = col < nr;
  const int mine = row0 + min(col, nr - 1), token = mine / group;
  const int pos = first_pos + token;
  auto row_of = [&](int c) {  // of the output and of the states
    const int tok = (row0 + c) / group;
    return ((int64_t)q.start + tok) * p.num_heads + h0 + (row0 + c - tok * group);
  };
  if (pmax < 0) {
    if (split == 0)
      for (int i = tid; i < nr * D; i += 256) static_cast<QS*>(p.out)[row_of(i / D) * D + i % D] = 0;
    return;
  }
  const int window = p.window > 0 ? p.window : p.max_seq_len;
  const int sinks = p.window > 0 ? p.sinks : 0;
  const int lo = max(0, max(pmin, 0) - window + 1);
  const int lead = (min(sinks, lo) + kWindowTile - 1) / kWindowTile;
  const int base_tile = max(lo / kWindowTile, lead);
  const int ntiles = lead + max(0, pmax / kWindowTile + 1 - base_tile);
  // Parts of one length for all sequences, that of the longest cut in p.splits.
  const int per = p.part_tiles;
  const int parts = max((ntiles + per - 1) / per, 1);
  const int v0 = split * per, v1 = min(v0 + per, ntiles);
  if (split >= parts) return;

  uint4 qf[KSTEPS];
  {
    const QS* src =
        static_cast<const QS*>(p.q) + (q.start + token) * p.q_stride + (int64_t)(h0 + (mine - token * group)) * D;
#pragma unroll
    for (int j = 0; j < KSTEPS; ++j) {
      const int d = F8 ? 64 * (j / 2) + 16 * g + 8 * (j & 1) : 32 * j + 8 * g;
      qf[j] = live && d < D ? *reinterpret_cast<const uint4*>(src + d) : make_uint4(0, 0, 0, 0);
    }
  }
  const int shift = p.block_shift, bs = 1 << shift;
  const int32_t* table = p.block_tables + (int64_t)seq * p.max_blocks_per_seq;
  const CS* kc = static_cast<const CS*>(p.k_cache) + (int64_t)kvh * p.k_head_stride;
  const CS* vc = static_cast<const CS*>(p.v_cache) + (int64_t)kvh * p.v_head_stride;

  f32x4 o[DT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) o[dt] = {0.f, 0.f, 0.f, 0.f};
  float m = kNoScore, l = 0.f;

  // A tile's blocks (of this lane's K row and of its V pieces), and its K and V.
  struct Blocks {
    int k, v;
  };
  auto tile_start = [&](int v) { return (v < lead ? v : base_tile + v - lead) * kWindowTile; };
  auto load_blocks = [&](int v) __attribute__((always_inline)) {
    Blocks b{-1, -1};
    if (v < v1) {
      const int t0 = tile_start(v), tk = t0 + 8 * (col >> 2), tv = t0 + 8 * g;
      if (tk < q.ctx) b.k = table[tk >> shift];
      if (tv < q.ctx) b.v = table[tv >> shift];
    }
    auto valid = [&](int id) { return id >= 0 && (int64_t)id < p.num_blocks ? id : -1; };
    return Blocks{valid(b.k), valid(b.v)};
  };
  using VR = typename std::conditional<F8, uint2, uint4>::type;
  constexpr int KL = F8 ? KSTEPS / 2 : KSTEPS;  // 16-byte loads of K per product
  struct Tile {
    uint4 k[2][KL];
    VR v[DT];
  };
  // (A missing block's loads go to block 0; its tokens are masked.)
  auto load_tile = [&](Tile& x, int v, const Blocks& b) __attribute__((always_inline)) {
    const int t0 = tile_start(v), tk = t0 + 8 * (col >> 2), tv = t0 + 8 * g;
    const CS* kp = kc + (int64_t)max(b.k, 0) * p.k_block_stride + ((tk & (bs - 1)) + (col & 3)) * X;
    const CS* vp = vc + (int64_t)max(b.v, 0) * p.v_block_stride + (tv & (bs - 1));
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int j = 0; j < KL; ++j) {
        const int c = 4 * j + g;
        x.k[u][j] = c * X < D ? *reinterpret_cast<const uint4*>(kp + (c * bs + 4 * u) * X) : make_uint4(0, 0, 0, 0);
      }
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
      x.v[dt] = *reinterpret_cast<const VR*>(vp + (D % 16 == 0 ? 16 * dt + col : min(16 * dt + col, D - 1)) * bs);
  };
  auto attend = [&](const Tile& x, int v, const Blocks& b) __attribute__((always_inline)) {
    const int tv = tile_start(v) + 8 * g;
    bool special = false;
    if constexpr (F8) {
      uint32_t probe = 0;
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int j = 0; j < KL; ++j)
          probe |= fp8x4_special(x.k[u][j].x) | fp8x4_special(x.k[u][j].y) | fp8x4_special(x.k[u][j].z) |
                   fp8x4_special(x.k[u][j].w);
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) probe |= fp8x4_special(x.v[dt].x) | fp8x4_special(x.v[dt].y);
      special = __any(probe != 0u);
    }
    f32x4 s[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      s[u] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < KL; ++j) {
        if constexpr (F8) {
          s[u] = Mma<QT>::k32(decode8<QT>(make_uint2(x.k[u][j].x, x.k[u][j].y), special), qf[2 * j], s[u]);
          s[u] = Mma<QT>::k32(decode8<QT>(make_uint2(x.k[u][j].z, x.k[u][j].w), special), qf[2 * j + 1], s[u]);
        } else {
          s[u] = Mma<QT>::k32(x.k[u][j], qf[j], s[u]);
        }
      }
    }
    // Bit r: this lane's row sees token tv + r.
    const uint32_t sees = b.v >= 0 ? seen16(pos, tv, window, sinks) & 0xffu : 0u;
    float mt = m;
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        s[u][r] = sees >> (4 * u + r) & 1u ? s[u][r] * p.scale_log2 : kNoScore;
        mt = fmaxf(mt, s[u][r]);
      }
    mt = column_max(mt);
    const float ref = mt == kNoScore ? 0.f : mt;
    const float alpha = __builtin_amdgcn_exp2f(m - ref);
    m = mt;
    l *= alpha;
    const float from = ref - weight_shift<QT>(0.f);
    uint32_t w[4];
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int r = 0; r < 4; r += 2) {
        const float a = __builtin_amdgcn_exp2f(s[u][r] - from), c = __builtin_amdgcn_exp2f(s[u][r + 1] - from);
        l += a + c;
        w[2 * u + r / 2] = pack_weights<QT>(a, c);
      }
    const uint4 wf = make_uint4(w[0], w[1], w[2], w[3]);
    // What a token that a row does not see holds must not matter (a weight of 0
    // times inf or NaN is NaN): it is taken out of V, and where the rows see
    // different tokens, at the few tiles where a row's keys begin or end, one query
    // position at a time; the others' rows keep their sums.
    const int t0 = tile_start(v);
    const bool one = ONE || (t0 + kWindowTile - 1 <= pmin && (t0 > pmax - window || t0 + kWindowTile <= sinks));
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
      uint4 y;
      if constexpr (F8)
        y = decode8<QT>(x.v[dt], special);
      else
        y = x.v[dt];
#pragma unroll
      for (int r = 0; r < 4; ++r) o[dt][r] *= alpha;
      if (one) {
        o[dt] = Mma<QT>::k32(keep8(y, sees), wf, o[dt]);
        continue;
      }
      for (int at = pmin; at <= pmax; ++at) {
        const f32x4 n = Mma<QT>::k32(keep8(y, b.v >= 0 ? seen16(at, tv, window, sinks) : 0u), wf, o[dt]);
#pragma unroll
        for (int r = 0; r < 4; ++r) o[dt][r] = pos == at ? n[r] : o[dt][r];
      }
    }
  };
  // Each wavefront takes every fourth tile.  While one is attended, the next one
  // loads (where the registers hold two, which stops at head size 128) and the
  // blocks of the one after are looked up.
  constexpr int NW = 4;
  Blocks b0 = load_blocks(v0 + wave);
  if constexpr (D <= 128) {
    Blocks b1 = load_blocks(v0 + wave + NW);
    Tile x0, x1;
    if (v0 + wave < v1) load_tile(x0, v0 + wave, b0);
    for (int v = v0 + wave; v < v1; v += 2 * NW) {
      Blocks b2 = load_blocks(v + 2 * NW);
      if (v + NW < v1) load_tile(x1, v + NW, b1);
      attend(x0, v, b0);
      if (v + NW >= v1) break;
      b0 = b2;
      b2 = load_blocks(v + 3 * NW);
      if (v + 2 * NW < v1) load_tile(x0, v + 2 * NW, b0);
      attend(x1, v + NW, b1);
      b1 = b2;
    }
  } else {
    for (int v = v0 + wave; v < v1; v += NW) {
      const Blocks b1 = load_blocks(v + NW);
      Tile x;
      load_tile(x, v, b0);
      attend(x, v, b0);
      b0 = b1;
    }
  }

  // The wavefronts' states: column col is row row0 + col.
  l = column_sum(l);
  if (g == 0) s_m[wave][col] = m, s_l[wave][col] = l;
  __syncthreads();
  float M = kNoScore, L = 0.f;
#pragma unroll
  for (int w = 0; w < 4; ++w) M = fmaxf(M, s_m[w][col]);
  {
    const float ref = M == kNoScore ? 0.f : M;
#pragma unroll
    for (int w = 0; w < 4; ++w) L += s_l[w][col] * __builtin_amdgcn_exp2f(s_m[w][col] - ref);
    const float f = __builtin_amdgcn_exp2f(m - ref);
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int r = 0; r < 4; ++r) s_o[wave][dt * 4 + r][lane] = o[dt][r] * f;
  }
  __syncthreads();
  // Wavefront w sums the 16-dimension tiles w, w + 4, ...
  const float inv = L > 0.f ? p.v_scale / L : L == 0.f ? 0.f : L;
  const int64_t row = row_of(min(col, nr - 1));
#pragma unroll
  for (int k = 0; k < (DT + 3) / 4; ++k) {
    const int dt = 4 * k + wave;
    const int d = 16 * dt + 4 * g;
    if (dt >= DT || !live || d >= D) continue;
    float x[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int at = dt * 4 + r;
      x[r] = s_o[0][at][lane] + s_o[1][at][lane] + s_o[2][at][lane] + s_o[3][at][lane];
    }
    if (parts == 1) {
      uint2 y;
      y.x = pack2(from_f32<QT>(x[0] * inv), from_f32<QT>(x[1] * inv));
      y.y = pack2(from_f32<QT>(x[2] * inv), from_f32<QT>(x[3] * inv));
      *reinterpret_cast<uint2*>(static_cast<QS*>(p.out) + row * D + d) = y;
    } else {
      float* to = p.ws_o + (row * p.splits + split) * D + d;
      store_agent(to, x[0], x[1]);
      store_agent(to + 2, x[2], x[3]);
    }
  }
  if (parts > 1 && wave == 0 && g == 0 && live) store_agent(p.ws_ml + (row * p.splits + split) * 2, M, L);
  if (parts == 1) return;
  // The workgroup whose part is the last to arrive merges all, in their order.
  wait_agent_stores();
  __syncthreads();
  if (tid == 0) s_last = arrived_last(p.counters + (int64_t)seq * p.units + unit, parts);
  __syncthreads();
  if (!s_last) return;
  // (The states lie in what was the wavefronts' outputs.)
  static_assert(sizeof(s_o) >= 16 * kFewMaxSplits * sizeof(float2), "room for every state");
  float2* s_ml = reinterpret_cast<float2*>(&s_o[0][0][0]);
  for (int i = tid; i < nr * parts; i += 256) {
    const int c = i / parts;
    s_ml[i] = load_agent(p.ws_ml + (row_of(c) * p.splits + (i - c * parts)) * 2);
  }
  __syncthreads();
  for (int i = tid; i < nr * (D / 2); i += 256) {
    const int c = i / (D / 2), d = 2 * (i - c * (D / 2));
    const int64_t r = row_of(c);
    const float2* state = s_ml + c * parts;
    const float* from = p.ws_o + r * p.splits * D + d;
    float mm = kNoScore;
    for (int s = 0; s < parts; ++s) mm = fmaxf(mm, state[s].x);
    const float rf = mm == kNoScore ? 0.f : mm;
    float ll = 0.f, x = 0.f, y = 0.f;
    constexpr int U = 8;  // loads in flight
    for (int s = 0; s < parts; s += U) {
      float2 v[U];
#pragma unroll
      for (int k = 0; k < U; ++k) v[k] = load_agent(from + (int64_t)min(s + k, parts - 1) * D);
#pragma unroll
      for (int k = 0; k < U; ++k) {
        if (s + k >= parts) continue;
        const float e = __builtin_amdgcn_exp2f(state[s + k].x - rf);
        ll += e * state[s + k].y;
        x += e * v[k].x;
        y += e * v[k].y;
      }
    }
    const float iv = ll > 0.f ? p.v_scale / ll : ll == 0.f ? 0.f : ll;
    *reinterpret_cast<uint32_t*>(static_cast<QS*>(p.out) + r * D + d) =
        pack2(from_f32<QT>(x * iv), from_f32<QT>(y * iv));
  }
}

template <class QT, class CT, int D>
hipError_t launch_extend_d(const ExtendParams& p, hipStream_t stream) {
  if (p.part_tiles > 0) {
    const int64_t tail = p.query_start_loc != nullptr ? extend_tail_groups(p.num_tokens, p.num_heads, D, p.splits) : 0;
    const dim3 grid((unsigned)((int64_t)p.num_seqs * p.units + tail), (unsigned)p.splits);
    if (p.max_query_len == 1)
      hipLaunchKernelGGL((extend_few_kernel<QT, CT, D, true>), grid, dim3(256), 0, stream, p);
    else
      hipLaunchKernelGGL((extend_few_kernel<QT, CT, D, false>), grid, dim3(256), 0, stream, p);
    return hipGetLastError();
  }
  const int64_t items = extend_items(p.num_tokens, p.num_seqs, p.group);
  // Head sizes up to 64 let three workgroups share a CU, which hides more of a tile's
  // softmax (13 prompts of up to 1700 tokens, window 1024, FP8: 178 us, with two 206).
  // A launch of no more than two per CU asks for shared memory that a third would
  // not have, so that it spreads over the chip (4 sequences, 100 tokens on 7900: 61
  // us, else 75).
  const int64_t tiles = std::max(((int64_t)p.num_tokens * p.group + kExtendRows - 1) / kExtendRows,
                                 (int64_t)std::min(p.num_seqs, p.num_tokens));
  const int64_t full = tiles * p.num_kv_heads * p.splits;
  const unsigned lds = D <= 64 && full <= 512 ? 40960 : 0;
  hipLaunchKernelGGL((extend_kernel<QT, CT, D>), dim3((unsigned)(items * p.num_kv_heads), (unsigned)p.splits),
                     dim3(kExtendThreads), lds, stream, p);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || p.splits == 1) return e;
  const int64_t rows = (int64_t)p.num_tokens * p.num_heads;
  hipLaunchKernelGGL((extend_merge_kernel<QT, D>), dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, stream, p);
  return hipGetLastError();
}

template <class QT, class CT>
hipError_t launch_extend_typed(const ExtendParams& p, int head_size, hipStream_t stream) {
  switch (head_size) {
    case 32: return launch_extend_d<QT, CT, 32>(p, stream);
    case 64: return launch_extend_d<QT, CT, 64>(p, stream);
    case 80: return launch_extend_d<QT, CT, 80>(p, stream);
    case 96: return launch_extend_d<QT, CT, 96>(p, stream);
    case 112: return launch_extend_d<QT, CT, 112>(p, stream);
    case 120:
      if constexpr (std::is_same<CT, FP8>::value) return hipErrorInvalidValue;  // (16 does not divide it)
      else return launch_extend_d<QT, CT, 120>(p, stream);
    case 128: return launch_extend_d<QT, CT, 128>(p, stream);
    case 192: return launch_extend_d<QT, CT, 192>(p, stream);
    case 256: return launch_extend_d<QT, CT, 256>(p, stream);
  }
  return hipErrorInvalidValue;
}

}  // namespace pkv
