// Causal attention of packed prompts over their keys and values as rows, [tokens, heads,
// head_size], the whole of a sequence or a sliding window and its first tokens.
//
// Sequence s brings n query tokens, the last n of its c key tokens: query i sits at
// position p = c - n + i and sees the keys t <= p, of them only those with t > p - window
// or t < sinks where there is a window.  A query row is one (token, head); the rows of the
// heads that share a KV head are attended together, row r of a sequence being head
// r % group of token r / group, so that they share the tiles of K and V.
//
// S^T = K Q^T and O^T = V^T P^T, as in extend_impl.h: a query row is a column of every
// matrix, its maximum and sum are one register a lane, and the weights leave the first
// product in the lanes where the second takes them.  K and V rows lie in LDS as they lie in
// memory; the second product wants 8 tokens of a dimension in a lane, which the transposing
// LDS read gives: of 16 lanes, lanes 4 k ..+3 name 16 elements of row k, and lane i
// receives element i of the rows 0 .. 3.
//
// Bound: the matrix units (64 % of the time) and the exponentials and sums beside them
// (vector units 61 %).  8192 tokens, 32 heads over 8 of 128: 495 .. 540 us, 1020 .. 1110
// TFLOP/s; the products alone took 297 us, with the weights 434, with all but the reads of
// LDS 506.  128 rows a workgroup, up to three workgroups a CU, one tile ahead: 256 rows by eight
// wavefronts took 555 us and left short prompts waiting (177 tokens 15 us instead of 11).
#pragma once

#include "extend_impl.h"

namespace pkv {

constexpr int kPromptTile = 64;
constexpr int kPromptThreads = 256;
// Wavefronts a SIMD.  Three at head size 64, with pieces of LDS two products ahead, take 119
// us for 54 prompts of 365 .. 485 tokens and 347 for 8192 tokens (32 heads over 8); two, with
// four ahead, 134 and 359.
constexpr int prompt_waves(int D) { return D <= 64 ? 3 : D <= 128 ? 2 : 1; }

// 16-byte chunk c of row r of an image with ROW chunks a row sits at chunk
// c ^ prompt_swizzle(r).  Reads meet no bank twice: 16 rows at one chunk (K) and 4 rows of
// 4 chunks (V) both take the 256 bytes of all banks once.
template <int ROW> __device__ __forceinline__ constexpr int prompt_swizzle(int r) {
  return ROW >= 16 ? ((r & 3) << 2) | ((r >> 2) & 3) : ROW == 8 ? (((r >> 1) & 1) << 2) | ((r >> 2) & 3) : (r >> 2) & 3;
}

// Over all 64 lanes, in every lane: within 16 by rotations, between them by exchanges.
template <class OP> __device__ __forceinline__ int wave_all(int x, OP op) {
  x = op(x, __builtin_amdgcn_update_dpp(0, x, 0x128, 0xf, 0xf, true));  // row_ror:8
  x = op(x, __builtin_amdgcn_update_dpp(0, x, 0x124, 0xf, 0xf, true));
  x = op(x, __builtin_amdgcn_update_dpp(0, x, 0x122, 0xf, 0xf, true));
  x = op(x, __builtin_amdgcn_update_dpp(0, x, 0x121, 0xf, 0xf, true));
  const auto a = __builtin_amdgcn_permlane16_swap((uint32_t)x, (uint32_t)x, false, false);
  x = op((int)a[0], (int)a[1]);
  const auto b = __builtin_amdgcn_permlane32_swap((uint32_t)x, (uint32_t)x, false, false);
  return __builtin_amdgcn_readfirstlane(op((int)b[0], (int)b[1]));
}
__device__ __forceinline__ int wave_sum(int x) {
  return wave_all(x, [](int a, int b) { return a + b; });
}
__device__ __forceinline__ int wave_max(int x) {
  return wave_all(x, [](int a, int b) { return max(a, b); });
}

struct PromptSeq {
  int start, count;  // query rows
  int key, ctx;      // key rows
};
__device__ __forceinline__ PromptSeq prompt_seq(const PromptParams& p, int s) {
  PromptSeq q;
  q.start = min(max(p.query_start_loc[s], 0), p.num_tokens);
  q.count = min(max(p.query_start_loc[s + 1], q.start), p.num_tokens) - q.start;
  q.key = min(max(p.key_start_loc[s], 0), p.num_keys);
  q.ctx = min(max(p.key_start_loc[s + 1], q.key), p.num_keys) - q.key;
  return q;
}

// Bit i of 32: a query at position pos sees token a + i.
__device__ __forceinline__ uint32_t seen32(int pos, int a, int window, int sinks) {
  auto below = [](int n) { return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1u; };
  return below(pos + 1 - a) & (~below(pos - window + 1 - a) | below(sinks - a));
}

template <class QT, int D>
__global__ __launch_bounds__(kPromptThreads, prompt_waves(D)) void prompt_kernel(PromptParams p) {
  using QS = typename Elem<QT>::storage;
  constexpr int KSTEPS = (D + 15) / 16;  // score products per 32 tokens
  constexpr int DT = (D + 31) / 32;      // 32-dimension tiles of the output
  constexpr int ROW = D <= 32 ? 4 : D <= 64 ? 8 : D <= 128 ? 16 : 32;
  constexpr int IMG = kPromptTile * ROW;
  constexpr int SR = kPromptTile / 4;   // rows of a tile that a wavefront stages
  constexpr int LOADS = SR * ROW / 64;  // and their 64-lane loads
  // Arrays of their own: the compiler then knows that the loads in flight do not touch
  // what is read.
  __shared__ uint4 s_k0[IMG], s_k1[IMG], s_v0[IMG], s_v1[IMG];
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
  const int item = p.by_kv_heads.of(blockIdx.x), kvh = blockIdx.x - item * p.num_kv_heads;
  const int split = blockIdx.y;
  const int group = p.group, h0 = kvh * group;

  // The workgroup's sequence and row tile: of 64 sequences at a time, the tiles that lie
  // furthest back in their sequences first (the longest, where all begin at position 0).
  // (Sequence by sequence, each from its end, nine prompts of 155 .. 1665 tokens with 14
  // heads of 64 took 50 us instead of 41: the last one's longest tiles ran alone.)
  if (wave == 0) {
    int base = 0, found = -1, z = 0;
    for (int s0 = 0; s0 < p.num_seqs; s0 += 64) {
      const int s = s0 + lane;
      int tiles = 0;
      if (s < p.num_seqs) tiles = (prompt_seq(p, s).count * group + kExtendRows - 1) / kExtendRows;
      const int all = wave_sum(tiles);
      if (item < base + all) {
        // The last tile index of which more than `rank` tiles lie at it or behind it.
        const int rank = item - base;
        int lo = 0, hi = wave_max(tiles);  // (behind(lo) > rank >= behind(hi) = 0)
        if (all == hi) lo = hi - 1 - rank, hi = lo + 1;  // (a single sequence's: 0.2 us sooner)
        while (hi - lo > 1) {
          const int mid = (lo + hi) / 2;
          if (wave_sum(max(tiles - mid, 0)) > rank) lo = mid;
          else hi = mid;
        }
        z = lo;
        const int nth = rank - wave_sum(max(tiles - lo - 1, 0));  // among the sequences that have tile z
        const uint64_t have = __ballot(tiles > lo);
        const bool mine = tiles > lo && __builtin_amdgcn_mbcnt_hi((uint32_t)(have >> 32),
                                            __builtin_amdgcn_mbcnt_lo((uint32_t)have, 0)) == nth;
        found = s0 + __builtin_ctzll(__ballot(mine));
        break;
      }
      base += all;
    }
    if (lane == 0) s_seq[0] = found, s_seq[1] = z, s_seq[2] = base, s_again = 0;
  }
  __syncthreads();
  const int seq = __builtin_amdgcn_readfirstlane(s_seq[0]);
  if (seq < 0) {
    // Past the last tile: rows behind the last sequence become zeros.
    const int tiles = s_seq[2];
    if (split != 0) return;
    const int last = min(max(p.query_start_loc[p.num_seqs], 0), p.num_tokens);
    const int items = gridDim.x / p.num_kv_heads;
    const int share = (p.num_tokens - last + items - tiles - 1) / (items - tiles);
    const int64_t t0 = last + (int64_t)(item - tiles) * share;
    zero_tokens<QT, kPromptThreads>(p, D, t0, min(t0 + share, (int64_t)p.num_tokens), h0, group);
    return;
  }
  const int z = __builtin_amdgcn_readfirstlane(s_seq[1]);
  const PromptSeq q = prompt_seq(p, seq);
  const int first_pos = q.ctx - q.count;  // position of the sequence's first query token
  const int rows = q.count * group;
  const int row0 = z * kExtendRows;
  const int row_end = min(row0 + kExtendRows, rows);
  // Positions of the workgroup's rows; tokens before position 0 see nothing.
  const int pmin = first_pos + p.by_group.of(row0), pmax = first_pos + p.by_group.of(row_end - 1);

  // This lane's row.
  const int wr0 = row0 + wave * 32, wr1 = min(wr0 + 32, rows);
  const int row = wr0 + col;
  const bool live = row < rows;
  const int tok = live ? p.by_group.of(row) : 0;
  const int head = h0 + (live ? row - tok * group : 0);
  const int64_t qrow = q.start + tok;
  const int pos = live ? first_pos + tok : -1;
  // Positions of the wavefront's rows (uniform): none where w_min > w_max.
  const bool w_any = wr0 < wr1;
  const int w_min = w_any ? first_pos + p.by_group.of(wr0) : 0, w_max = w_any ? first_pos + p.by_group.of(wr1 - 1) : -1;

  // The tiles to visit: those of the sinks, then those of the window.
  const int window = p.window > 0 ? p.window : 1 << 30;
  const int sinks = p.window > 0 ? p.sinks : 0;
  int lead = 0, base_tile = 0, ntiles = 0;
  if (pmax >= 0) {
    const int lo = max(0, max(pmin, 0) - window + 1);
    lead = (min(sinks, lo) + kPromptTile - 1) / kPromptTile;
    base_tile = max(lo / kPromptTile, lead);
    ntiles = lead + max(0, pmax / kPromptTile + 1 - base_tile);
  }
  const int per = (ntiles + p.splits - 1) / p.splits;
  const int v0 = min(split * per, ntiles), v1 = min(v0 + per, ntiles);
  auto tile_start = [&](int v) { return (v < lead ? v : base_tile + v - lead) * kPromptTile; };

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

  // Addresses that follow from the lane alone, made opaque to the compiler at each tile:
  // it would otherwise hold what it derives from them in 80 registers over the loop.
  //   k_at: of chunk 2 j + half of row col of K's image, but for j (which flips its bits);
  //   v_at: of this lane's 8 bytes for the transposing read of rows 4 half .. (+ 8 i), dim 32 dt;
  //   k_row, v_row, load_chunk: this lane's row in the first load of a tile, its 16 bytes there.
  uint32_t k_at = (lane & 31) * (ROW * 16) + 16 * (half ^ prompt_swizzle<ROW>(lane & 31)), v_at[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int r = 4 * half + (lane % 16) / 4 + 8 * i, c = 2 * ((lane / 16) % 2) + (lane % 4) / 2;
    v_at[i] = r * (ROW * 16) + 16 * (c ^ prompt_swizzle<ROW>(r)) + 8 * (lane & 1);
  }
  constexpr int RL = 64 / ROW;  // rows of a load
  const int load_row = SR * wave + lane / ROW;
  uint32_t k_row = load_row * (uint32_t)p.k_stride * 2, v_row = load_row * (uint32_t)p.v_stride * 2;
  uint32_t load_chunk = 16 * ((lane % ROW) ^ prompt_swizzle<ROW>(load_row));
  auto lane_again = [&]() __attribute__((always_inline)) {
    asm volatile("" : "+v"(k_at), "+v"(v_at[0]), "+v"(v_at[1]), "+v"(k_row), "+v"(v_row), "+v"(load_chunk));
  };
  // A wavefront stages SR rows of a tile of K or V, 16 bytes a lane, by buffer loads: what
  // lies behind the sequence's last row, or behind a row that is shorter than its image,
  // is out of the buffer's range and becomes zeros.  (One buffer a tile: with one for each
  // load their scalar instructions took 568 us instead of 554 for 8192 tokens.)
  const char* k_rows = static_cast<const char*>(p.k_cache) + (q.key * p.k_stride + (int64_t)kvh * D) * 2;
  const char* v_rows = static_cast<const char*>(p.v_cache) + (q.key * p.v_stride + (int64_t)kvh * D) * 2;
  auto stage = [&](uint4* image, const char* rows_of, int64_t stride, uint32_t row_at, int t0)
                   __attribute__((always_inline)) {
    const uint32_t bytes = (uint32_t)stride * 2;  // (64 rows stay below 2^31)
    const int rows_left = min(q.ctx - t0, kPromptTile);
    const auto rsrc = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<char*>(rows_of + (int64_t)t0 * stride * 2), 0,
        rows_left > 0 ? (int)((uint32_t)(rows_left - 1) * bytes + 2 * D) : 0, 0x00027000);
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      // (A load's rows and a wavefront's have their bits apart: the swizzles add up.)  The
      // whole offset stands in the lane's part of the address: the range check counts that
      // part, not the scalar one.
      const uint32_t c = load_chunk ^ (16 * prompt_swizzle<ROW>(RL * i));
      uint32_t at = row_at + RL * i * bytes + c;
      if (D != 8 * ROW) at = c < 2 * D ? at : 0xfffffff0u;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          rsrc, (__attribute__((address_space(3))) void*)(image + SR * wave * ROW + 64 * i), 16, (int)at, 0, 0, 0);
    }
  };
  auto stage_k = [&](auto k, int v) __attribute__((always_inline)) {
    if (v < v1) stage(k_image(k), k_rows, p.k_stride, k_row, tile_start(v));
  };
  auto stage_v = [&](auto k, int v) __attribute__((always_inline)) {
    if (v < v1) stage(v_image(k), v_rows, p.v_stride, v_row, tile_start(v));
  };
  // The workgroup meets at a bare s_barrier, each wavefront's own loads and LDS accesses
  // awaited before.
  auto meet = [] __attribute__((always_inline)) {
    __builtin_amdgcn_s_waitcnt(0x0070);  // vmcnt(0) lgkmcnt(0)
    asm volatile("s_barrier" ::: "memory");
  };

  // Register r of sub of a tile's scores is token 32 sub + r % 4 + 8 (r / 4) + 4 half.  K's
  // part of the product of dimensions 16 j ..+15 with tokens 32 sub ..+31:
  auto k_piece = [&](auto k, int sub, int j) __attribute__((always_inline)) {
    const char* at = reinterpret_cast<const char*>(k_image(k)) + 32 * sub * ROW * 16;
    return *reinterpret_cast<const uint4*>(at + (k_at ^ (32 * j)));
  };
  // Tokens 32 sub + 16 st + 8 i + 4 half ..+3, i = 0 and 1, of dimension 32 dt + col.
  auto v_piece = [&](auto k, int dt, int sub, int st) __attribute__((always_inline)) {
    typedef short s16x4 __attribute__((ext_vector_type(4)));
    uint2 x[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const char* at = reinterpret_cast<const char*>(v_image(k)) + (32 * sub + 16 * st) * ROW * 16;
      x[i] = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                           (__attribute__((address_space(3))) s16x4*)(at + (v_at[i] ^ (64 * dt)))));
    }
    return make_uint4(x[0].x, x[0].y, x[1].x, x[1].y);
  };
  // Bits of a lane's 8 tokens of (sub, st) among the 32 of sub.
  auto lane_bits = [&](uint32_t seen, int st) {
    const uint32_t a = seen >> (16 * st + 4 * half);
    return (a & 0xfu) | ((a >> 4) & 0xf0u);
  };
  auto mask = [&](f32x16 (&s)[2], int t0) __attribute__((always_inline)) {
#pragma unroll
    for (int sub = 0; sub < 2; ++sub) {
      const uint32_t sees = seen32(pos, t0 + 32 * sub, window, sinks) >> (4 * half);
#pragma unroll
      for (int r = 0; r < 16; ++r) s[sub][r] = sees >> ((r & 3) + 8 * (r >> 2)) & 1u ? s[sub][r] : kNoScore;
    }
  };
  // Moves the rows' reference points where the scores pass them by the slack.
  auto refer = [&](const f32x16 (&s)[2]) __attribute__((always_inline)) {
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
  };
  auto weigh = [&](const f32x16 (&s)[2], uint32_t (&w)[2][8]) __attribute__((always_inline)) {
    // (A row that has seen nothing keeps a finite reference point: no inf - inf.)
    const float ref = (m == kNoScore ? 0.f : m * scale) - weight_shift<QT>(kExtendSlack<QT>);
#pragma unroll
    for (int sub = 0; sub < 2; ++sub)
#pragma unroll
      for (int r = 0; r < 16; r += 2) {
        const float a = __builtin_amdgcn_exp2f(__builtin_fmaf(s[sub][r], scale, -ref));
        const float b = __builtin_amdgcn_exp2f(__builtin_fmaf(s[sub][r + 1], scale, -ref));
        l += a + b;
        w[sub][r / 2] = pack_weights<QT>(a, b);
      }
  };
  auto weights = [&](const uint32_t (&w)[2][8], int sub, int st) {
    return make_uint4(w[sub][4 * st], w[sub][4 * st + 1], w[sub][4 * st + 2], w[sub][4 * st + 3]);
  };
  // The products of a step: s = S^T of the tile in K's image kk (SCORES), then the outputs
  // of the tile in V's image kv with the weights w (VALUES).  Pieces come from LDS four (or
  // two) products ahead of their use; the fences keep them there (left to itself the
  // compiler reads each right before its product and waits out LDS 32 times a tile: 870
  // instead of 1000 TFLOP/s for 8192 tokens with 32 heads of 128).
  auto run_products = [&](auto kk, auto kv, auto scores, auto values, f32x16 (&s)[2], const uint32_t (&w)[2][8])
                          __attribute__((always_inline)) {
    constexpr int NS = decltype(scores)::value ? 2 * KSTEPS : 0, NV = decltype(values)::value ? 4 * DT : 0;
    constexpr int N = NS + NV, G = prompt_waves(D) == 3 ? 2 : 4;
    auto piece = [&](int i) __attribute__((always_inline)) {
      return i < NS ? k_piece(kk, i % 2, i / 2)
                    : v_piece(kv, (i - NS) % DT, (i - NS) / DT / 2, (i - NS) / DT % 2);
    };
    uint4 x[2][G];
#pragma unroll
    for (int i = 0; i < G; ++i)
      if (i < N) x[0][i] = piece(i);
    if (NS > 0)
#pragma unroll
      for (int sub = 0; sub < 2; ++sub)
#pragma unroll
        for (int r = 0; r < 16; ++r) s[sub][r] = 0.f;
#pragma unroll
    for (int i0 = 0; i0 < N; i0 += G) {
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int i = 0; i < G; ++i)
        if (i0 + G + i < N) x[(i0 / G + 1) % 2][i] = piece(i0 + G + i);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int i = 0; i < G; ++i) {
        const int n = i0 + i;
        if (n >= N) continue;
        if (n < NS) {
          s[n % 2] = mma32<QT>(x[i0 / G % 2][i], qf[n / 2], s[n % 2]);
        } else {
          const int at = n - NS, dt = at % DT, sub = at / DT / 2, st = at / DT % 2;
          o[dt] = mma32<QT>(x[i0 / G % 2][i], weights(w, sub, st), o[dt]);
        }
      }
    }
    __builtin_amdgcn_sched_barrier(0);
  };
  // A token that some rows do not see must not reach them, whatever its value, but a
  // weight of 0 times inf or NaN is NaN.  A product with zeros tells whether a partly
  // seen tile has such a value: the rows are then done again, with care.
  auto test = [&](auto k) __attribute__((always_inline)) {
    f32x16 zero;
#pragma unroll
    for (int r = 0; r < 16; ++r) zero[r] = 0.f;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int j = 0; j < 4; ++j) zero = mma32<QT>(v_piece(k, dt, j >> 1, j & 1), make_uint4(0, 0, 0, 0), zero);
    float sum = 0.f;
#pragma unroll
    for (int r = 0; r < 16; ++r) sum += zero[r];
    if (__any(sum != 0.f)) s_again = 1;
  };
  // One query position at a time, with the tokens that it does not see taken out of V;
  // the other positions' rows keep their sums.
  auto careful_products = [&](const uint32_t (&w)[2][8], int t0) __attribute__((always_inline)) {
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll 1
      for (int at = w_min; at <= w_max; ++at)
#pragma unroll
        for (int sub = 0; sub < 2; ++sub) {
          const uint32_t keep = seen32(at, t0 + 32 * sub, window, sinks);
          f32x16 n = o[dt];
#pragma unroll
          for (int st = 0; st < 2; ++st)
            n = mma32<QT>(keep8(v_piece(I0{}, dt, sub, st), lane_bits(keep, st)), weights(w, sub, st), n);
#pragma unroll
          for (int r = 0; r < 16; ++r) o[dt][r] = pos == at ? n[r] : o[dt][r];
        }
  };
  // Whether any of the wavefront's rows sees a token of the tile, and whether all see all.
  auto some_see = [&](int t0) { return w_max >= t0 && (t0 < sinks || t0 + kPromptTile > w_min - window + 1); };
  auto all_see = [&](int t0) {
    return t0 + kPromptTile - 1 <= w_min && (t0 > w_max - window || t0 + kPromptTile <= sinks);
  };

  // A step takes tile v's weights on the vector units, then tile v + 1's scores and tile
  // v's second product in one run on the matrix units, while V of tile v + 1 and K of tile
  // v + 2 load.
  if (v0 < v1) {
    f32x16 s[2];
    uint32_t w[2][8];
    // Tiles [first_whole, last_whole) are seen in full by every row: behind the sinks'
    // tiles and the window's edge, before the first row's position.
    const int first_whole = lead + max(0, (max(pmax - window + 1, 0) + kPromptTile - 1) / kPromptTile - base_tile);
    const int last_whole = min(v1, lead + (pmin + 1) / kPromptTile - base_tile);
    stage_k(I0{}, v0);
    stage_v(I0{}, v0);
    stage_k(I1{}, v0 + 1);
    meet();
    if (some_see(tile_start(v0))) run_products(I0{}, I0{}, std::true_type{}, std::false_type{}, s, w);
    auto step = [&](auto k, int v) __attribute__((always_inline)) {
      using KN = std::integral_constant<int, decltype(k)::value ^ 1>;
      const int t0 = tile_start(v);
      lane_again();
      meet();  // V of tile v and K of tile v + 1 have landed; K of tile v and V of tile v - 1 have been read
      stage_k(k, v + 2);
      stage_v(KN{}, v + 1);
      const bool seen = some_see(t0), sees = v + 1 < v1 && some_see(tile_start(v + 1));
      if (seen) {
        if (!all_see(t0)) mask(s, t0);
        refer(s);
        weigh(s, w);
      }
      // (With a third way, both in one run, what they share was copied between registers: 18
      // us instead of 12 for 23 tokens at head size 256, 264 instead of 205 for 4096.)
      if (seen) run_products(KN{}, k, std::false_type{}, std::true_type{}, s, w);
      if (sees) run_products(KN{}, k, std::true_type{}, std::false_type{}, s, w);
      if (seen && !all_see(t0)) test(k);
    };
    // The same where every row of the workgroup sees both tiles in full: no branch but
    // that of a moved reference point.  (In one loop with the others, the outputs were
    // copied between registers where their ways meet, at each tile.)  The products come
    // first on a SIMD whose other wavefront takes weights: 544 us instead of 552.
    auto whole_step = [&](auto k, int v) __attribute__((always_inline)) {
      using KN = std::integral_constant<int, decltype(k)::value ^ 1>;
      lane_again();
      meet();
      stage_k(k, v + 2);
      stage_v(KN{}, v + 1);
      refer(s);
      weigh(s, w);
      __builtin_amdgcn_s_setprio(1);
      run_products(KN{}, k, std::true_type{}, std::true_type{}, s, w);
      __builtin_amdgcn_s_setprio(0);
    };
    int v = v0;
    while (v < v1) {
      if (v >= first_whole) {
#pragma unroll 1
        while (v + 2 < last_whole) {
          whole_step(I0{}, v);
          whole_step(I1{}, v + 1);
          v += 2;
        }
      }
      step(I0{}, v);
      if (++v >= v1) break;
      step(I1{}, v);
      ++v;
    }
    meet();
    if (__builtin_expect(s_again, 0)) {
      reset();
#pragma unroll 1
      for (int v = v0; v < v1; ++v) {
        const int t0 = tile_start(v);
        meet();
        stage_k(I0{}, v);
        stage_v(I0{}, v);
        meet();
        if (!some_see(t0)) continue;
        run_products(I0{}, I0{}, std::true_type{}, std::false_type{}, s, w);
        mask(s, t0);
        refer(s);
        weigh(s, w);
        careful_products(w, t0);
      }
    }
  }

  l = xchg32_sum(l);
  if (!live) return;
  if (p.splits == 1) {
    const float inv = l > 0.f ? 1.f / l : l == 0.f ? 0.f : l;  // (NaN stays NaN)
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

template <class QT, int D> hipError_t launch_prompt_d(const PromptParams& p, hipStream_t stream) {
  const int64_t items = extend_items(p.num_tokens, p.num_seqs, p.group);
  hipLaunchKernelGGL((prompt_kernel<QT, D>), dim3((unsigned)(items * p.num_kv_heads), (unsigned)p.splits),
                     dim3(kPromptThreads), 0, stream, p);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || p.splits == 1) return e;
  const int64_t rows = (int64_t)p.num_tokens * p.num_heads;
  hipLaunchKernelGGL((extend_merge_kernel<QT, D>), dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, stream,
                     static_cast<const ExtendParams&>(p));
  return hipGetLastError();
}

template <class QT> hipError_t launch_prompt(const PromptParams& p, int head_size, hipStream_t stream) {
  switch (head_size) {
    case 32: return launch_prompt_d<QT, 32>(p, stream);
    case 64: return launch_prompt_d<QT, 64>(p, stream);
    case 80: return launch_prompt_d<QT, 80>(p, stream);
    case 96: return launch_prompt_d<QT, 96>(p, stream);
    case 112: return launch_prompt_d<QT, 112>(p, stream);
    case 120: return launch_prompt_d<QT, 120>(p, stream);
    case 128: return launch_prompt_d<QT, 128>(p, stream);
    case 192: return launch_prompt_d<QT, 192>(p, stream);
    case 256: return launch_prompt_d<QT, 256>(p, stream);
  }
  return hipErrorInvalidValue;
}

}  // namespace pkv
