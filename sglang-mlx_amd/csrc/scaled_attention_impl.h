// Attention of single and drafted tokens over a paged cache of E4M3 codes with a scale
// for each (block, KV head) of K and of V.
//
// K_t = c_t ks_b, V_t = d_t vs_b for the codes c, d of token t in block b:
//   out = sum_t w_t vs_b d_t / sum_t w_t,   w_t = exp(scale ks_b (q . c_t) - m).
// The codes are exact in the queries' 16-bit type, so both products run on them as they
// are; ks multiplies a score in float32, vs a weight before it is rounded to 16 bits.
// There vs enters as vs / 2^e, 2^(m + e) being at least the largest product of exp(score)
// and scale that the row has seen: the weights keep the range that float16 has, whatever the
// scales' size (with e the largest exponent of a scale seen, a block of scale 2^16 and weight
// 2^-60 cost blocks of scale 2^-16 a third of their value), and the output returns to true
// size at the end (2^e; powers of two, so that nothing is rounded).
//
// Query rows, products and masks are those of extend_few_kernel (extend_impl.h): 16 rows
// of a sequence and KV head, straight from the cache to the matrix units' registers,
// S^T = K Q^T, O^T = V^T P^T.  A tile is 64 tokens; lane group g holds tokens 16 g ..+15
// of it, so that V's paged layout arrives in whole 16-byte pieces and a lane has one K
// scale and one V scale a tile (two of 8-token blocks): row i of score product u, of
// four, is token 16 (i / 4) + 4 u + i % 4.
//
// Schedule: a unit is 16 rows of a KV head, a crew one workgroup for each unit.  The
// sequences lie end to end, each its tiles and a start-up's worth of them long, and every
// crew takes an equal span of that line, so that ragged contexts load the chip evenly and
// one long context fills it.  The workgroups of a crew go through the same tokens at the
// same time, a block's heads side by side (with a span of single items for each workgroup
// 256 short sequences took 114 us instead of 110).  Pieces of a sequence leave their
// states in the workspace; the one that arrives last merges them in their order (no result
// depends on timing, nobody waits for another workgroup).
//
// Bound: this kernel's reads, behind a start and an end.  64 sequences of 533 .. 4097 tokens,
// 8 KV heads of 128: 65 .. 67 us, 4.5 .. 4.7 TB/s (68 at the time when the same schedule with
// the loads alone, nothing computed, took 66).  That is these loads' rate, not the card's: a K
// load touches 16 places of 64 bytes, at the default cache policy, where the decode kernel of
// caches with one scale reads runs of 1 KiB, non-temporal, and as many bytes in 52 us.  In a
// graph a call with one token takes 6.1 us (launch, lengths -> span -> blocks -> first tile,
// states in LDS, output), one sequence of 512, a piece, 8.0, one of 1024, several, 11.0: the
// arrival and the merge cost 3 us.  Beyond 16 rows of a KV head its codes are read again for
// each 16 (28 heads over 4, five drafted tokens: 138 MB for 45).
#pragma once

#include "extend_impl.h"

namespace pkv {

// Sequence s of a call: its query rows and the tiles of 64 tokens that they see.
struct ScaledSeq {
  ExtendSeq q;
  int lead, base, tiles;  // tiles [0, lead), then from base on; tiles in all
  __device__ __forceinline__ int start_of(int v) const { return (v < lead ? v : base + v - lead) * kScaledTile; }
};
__device__ __forceinline__ ScaledSeq scaled_seq(const ScaledAttentionParams& p, int s) {
  ScaledSeq r;
  r.q = extend_seq(p, s);
  r.lead = r.base = r.tiles = 0;
  if (r.q.ctx == 0 || r.q.count == 0) return r;
  const int window = p.window > 0 ? p.window : p.max_seq_len;
  const int sinks = p.window > 0 ? p.sinks : 0;
  const int lo = max(0, max(r.q.ctx - r.q.count, 0) - window + 1);
  r.lead = (min(sinks, lo) + kScaledTile - 1) / kScaledTile;
  r.base = max(lo / kScaledTile, r.lead);
  r.tiles = r.lead + max(0, (r.q.ctx - 1) / kScaledTile + 1 - r.base);
  return r;
}

template <class QT, int D, int BS, bool ONE>
__global__ __launch_bounds__(256, D <= 128 ? 2 : 1) void scaled_attention_kernel(ScaledAttentionParams p) {
  using QS = typename Elem<QT>::storage;
  constexpr int SHIFT = BS == 8 ? 3 : BS == 16 ? 4 : 5;
  constexpr int NB = BS == 8 ? 2 : 1;    // blocks of 16 tokens
  constexpr int KL = (D + 63) / 64;  // 16-byte loads of a K row's codes by a lane (each two products)
  constexpr int DT = D / 16;
  constexpr int NW = 4;
  __shared__ float s_o[NW][DT * 4][64];
  __shared__ float s_m[NW][16], s_l[NW][16], s_e[NW][16];
  __shared__ int s_sum[NW], s_long[NW], s_base, s_first, s_last;

  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int group = p.group, H = p.num_kv_heads;
  if ((int)blockIdx.x >= p.workgroups) {
    const int tail = blockIdx.x - p.workgroups, empty = (p.num_seqs + 255) / 256;
    if (tail < empty) {
      // Rows of sequences that have nothing to attend become zeros: each wavefront looks
      // at 64 sequences.
      const int lane = threadIdx.x & 63, s = tail * 256 + threadIdx.x;
      ScaledSeq q;
      q.q.count = 0;
      if (s < p.num_seqs) q = scaled_seq(p, s);
      uint64_t rows = __ballot(q.q.count > 0 && q.tiles == 0);
      for (; rows; rows &= rows - 1) {
        const int w = __builtin_ctzll(rows);
        const int64_t t0 = __shfl(q.q.start, w), n = __shfl(q.q.count, w);
        uint4* out = reinterpret_cast<uint4*>(static_cast<QS*>(p.out) + t0 * p.num_heads * D);
        for (int64_t i = lane; i < n * p.num_heads * (D / 8); i += 64) out[i] = make_uint4(0, 0, 0, 0);
      }
      return;
    }
    // Rows behind the last sequence become zeros.
    const int last = min(max(p.query_start_loc[p.num_seqs], 0), p.num_tokens);
    const int groups = gridDim.x - p.workgroups - empty;
    const int share = (p.num_tokens - last + groups - 1) / groups;
    const int64_t t0 = last + (int64_t)(tail - empty) * share;
    zero_tokens<QT, 256>(p, D, t0, min(t0 + share, (int64_t)p.num_tokens), 0, p.num_heads);
    return;
  }
  int tid = threadIdx.x, lane = tid & 63;
  // Length of one item of a sequence (none with nothing to attend).
  auto item_length = [](const ScaledSeq& q) { return q.tiles == 0 ? 0 : q.tiles + kScaledStart; };
  // The sum of all lengths (below 2^31), and the sequence in which this workgroup's span
  // begins: each thread sums a run of sequences.
  const int run = (p.num_seqs + 255) / 256;
  int mine = 0;
  for (int s = tid * run; s < min((tid + 1) * run, p.num_seqs); ++s) mine += item_length(scaled_seq(p, s));
  int sum = mine;  // of this lane and those before it: within 16 lanes, then by their last
  sum += __builtin_amdgcn_update_dpp(0, sum, 0x111, 0xf, 0xf, false);  // row_shr:1
  sum += __builtin_amdgcn_update_dpp(0, sum, 0x112, 0xf, 0xf, false);
  sum += __builtin_amdgcn_update_dpp(0, sum, 0x114, 0xf, 0xf, false);
  sum += __builtin_amdgcn_update_dpp(0, sum, 0x118, 0xf, 0xf, false);
  sum += __builtin_amdgcn_update_dpp(0, sum, 0x142, 0xa, 0xf, false);  // row_bcast:15
  sum += __builtin_amdgcn_update_dpp(0, sum, 0x143, 0xc, 0xf, false);  // row_bcast:31
  const bool any_long = __any(mine > kScaledWhole);
  if (lane == 63) s_sum[wave] = sum, s_long[wave] = any_long;
  __syncthreads();
  int total = 0, below = sum - mine, longer = run - 1;
#pragma unroll
  for (int w = 0; w < NW; ++w) {
    const int a = __builtin_amdgcn_readfirstlane(s_sum[w]);
    if (w < wave) below += a;
    total += a;
    longer |= __builtin_amdgcn_readfirstlane(s_long[w]);
  }
  // A wavefront pays for each instruction of a start in full: here the quotient comes by the
  // divisor's reciprocal (exact for the up to kScaledWorkgroups workgroups of several crews).
  // That, the sum over the lanes without trips through LDS and one division a row instead of
  // one an output element took a call with one token from 8.4 to 6.9 us.
  const int crews = p.crews, crew = crew_of(blockIdx.x, p.units, crews, p.unit_reciprocal);
  const int unit = blockIdx.x - crew * p.units;
  // Where all are short and there are crews enough, each sequence is one crew's (cut and
  // joined by the span, four of 8 .. 50 tokens took 13.1 us instead of 8.6, sixty of 300 ..
  // 512 21.8 instead of 16.4).
  const bool apiece = longer == 0 && p.num_seqs <= crews;
  int span = kScaledLeast;
  if (!apiece) span = max((total + crews - 1) / crews, kScaledLeast);
  if (apiece ? crew >= p.num_seqs : (int64_t)crew * span >= total) return;
  int x0 = crew * span, x1 = apiece ? 0 : min(span, total - x0) + x0;
  if (apiece) {
    if (tid == crew) s_first = crew, s_base = below, s_last = mine;
  } else if (x0 >= below && x0 < below + mine) {
    int at = below;
    int s = tid * run;
    for (;; ++s) {
      const int n = item_length(scaled_seq(p, s));
      if (x0 < at + n) break;
      at += n;
    }
    s_first = s, s_base = at;
  }
  __syncthreads();
  if (apiece) {
    x0 = __builtin_amdgcn_readfirstlane(s_base);
    x1 = x0 + __builtin_amdgcn_readfirstlane(s_last);
  }

  const int window = p.window > 0 ? p.window : p.max_seq_len;
  const int sinks = p.window > 0 ? p.sinks : 0;

  // A piece: tiles [v0, v1) of a sequence, one of `parts` pieces, the first by crew
  // w_first.  Everything here is the same for all threads.
  struct Piece {
    ScaledSeq q;
    int seq, nr, v0, v1, w_first, parts;
  };
  // (ONE: a sequence has one token's rows.)
  auto token_of = [&](int row) __attribute__((always_inline)) { return ONE ? 0 : row / group; };
  const int kvh = p.slices == 1 ? unit : unit / p.slices, row0 = 16 * (unit - kvh * p.slices), h0 = kvh * group;
  // The next sequence of this crew's span.
  int seq = __builtin_amdgcn_readfirstlane(s_first), base = __builtin_amdgcn_readfirstlane(s_base);
  auto next_piece = [&](Piece& c) __attribute__((always_inline)) -> bool {
    while (base < x1) {
      // (In scalar registers: loads in a loop that stores come back in vector ones, and
      // all that follows from them would stay there.)
      ScaledSeq q = scaled_seq(p, seq);
      q.q.start = __builtin_amdgcn_readfirstlane(q.q.start);
      q.q.count = __builtin_amdgcn_readfirstlane(q.q.count);
      q.q.ctx = __builtin_amdgcn_readfirstlane(q.q.ctx);
      q.lead = __builtin_amdgcn_readfirstlane(q.lead);
      q.base = __builtin_amdgcn_readfirstlane(q.base);
      q.tiles = __builtin_amdgcn_readfirstlane(q.tiles);
      const int begin = base, end = begin + item_length(q);
      c.seq = seq;
      base = end;
      ++seq;
      const ScaledPiece piece = scaled_piece(begin, end, x0, x1, span, crew, apiece);
      c.nr = min(16, q.q.count * group - row0);
      if (piece.from >= piece.to || c.nr <= 0) continue;
      c.parts = piece.parts;
      c.w_first = piece.first;
      c.v0 = max(piece.from - begin - kScaledStart, 0);
      c.v1 = piece.to - begin - kScaledStart;
      c.q = q;
      return true;
    }
    return false;
  };

  // (Opaque to the compiler: addresses of a lane that no piece changes would otherwise stay
  // in registers over the loop, 75 of them at head size 128.)
  asm volatile("" : "+v"(tid), "+v"(lane));
  int g = lane >> 4, col = lane & 15;
  Piece c;
  // What belongs to the piece: this lane's row and its position, the cache's pointers.
  ScaledSeq q;
  int pmin, pmax, pos, v0, v1;
  const int32_t* table;
  const uint8_t *kc, *vc;
  const float* scales;
  uint4 qf[2 * KL];
  f32x4 o[DT];
  // m: log2 of the weights' reference point; m + e: of the largest product of a weight and its
  // scale, whose reference point is 2^(m + ceil(e)).
  float m, l, e;
  auto begin_piece = [&]() __attribute__((always_inline)) {
    q = c.q;
    v0 = c.v0, v1 = c.v1;
    const int first_pos = q.q.ctx - q.q.count;
    pmin = first_pos + token_of(row0), pmax = first_pos + token_of(row0 + c.nr - 1);
    // Row row0 + i, i < nr, is head (row0 + i) % group of token (row0 + i) / group; this
    // lane's is i = col.
    const int my_row = row0 + min(col, c.nr - 1), token = token_of(my_row);
    pos = first_pos + token;
    const QS* src =
        static_cast<const QS*>(p.q) + (q.q.start + token) * p.q_stride + (int64_t)(h0 + (my_row - token * group)) * D;
#pragma unroll
    for (int j = 0; j < 2 * KL; ++j) {
      const int d = 64 * (j / 2) + 16 * g + 8 * (j & 1);
      qf[j] = col < c.nr && d < D ? *reinterpret_cast<const uint4*>(src + d) : make_uint4(0, 0, 0, 0);
    }
    table = p.block_tables + (int64_t)c.seq * p.max_blocks_per_seq;
    kc = static_cast<const uint8_t*>(p.k_cache) + (int64_t)kvh * p.k_head_stride;
    vc = static_cast<const uint8_t*>(p.v_cache) + (int64_t)kvh * p.v_head_stride;
    scales = p.scales + 2 * kvh;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) o[dt] = {0.f, 0.f, 0.f, 0.f};
    m = kNoScore, l = 0.f, e = kNoExponent;
  };
  // Blocks of this lane's K rows and of its V tokens (two of 8 tokens each).
  struct Blocks {
    int k[NB], v[NB];
  };
  auto load_blocks = [&](int v) __attribute__((always_inline)) {
    const int t0 = q.start_of(v);
    Blocks b;
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      const int tk = t0 + 16 * (col >> 2) + 8 * i, tv = t0 + 16 * g + 8 * i;
      b.k[i] = b.v[i] = -1;
      if (tk < q.q.ctx) b.k[i] = table[tk >> SHIFT];
      if (tv < q.q.ctx) b.v[i] = table[tv >> SHIFT];
    }
    return b;
  };
  auto check_blocks = [&](Blocks& b) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      b.k[i] = b.k[i] >= 0 && (int64_t)b.k[i] < p.num_blocks ? b.k[i] : -1;
      b.v[i] = b.v[i] >= 0 && (int64_t)b.v[i] < p.num_blocks ? b.v[i] : -1;
    }
  };
  uint4 kx[4][KL], vx[DT];
  float2 sx[NB];
  // (A missing block's loads go to block 0; its tokens are masked.)
  auto load_k = [&](const Blocks& b) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const uint8_t* at = kc + (int64_t)max(b.k[BS == 8 ? u / 2 : 0], 0) * p.k_block_stride + 16 * (col & 3);
      const int off = BS == 8 ? 4 * (u & 1) : BS == 16 ? 4 * u : 16 * ((col >> 2) & 1) + 4 * u;
#pragma unroll
      for (int j = 0; j < KL; ++j) {
        const int c = 4 * j + g;
        kx[u][j] = D % 64 == 0 || c * 16 < D ? *reinterpret_cast<const uint4*>(at + (c * BS + off) * 16)
                                              : make_uint4(0, 0, 0, 0);
      }
    }
  };
  auto load_v = [&](const Blocks& b) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < NB; ++i) sx[i] = *reinterpret_cast<const float2*>(scales + (int64_t)max(b.v[i], 0) * 2 * H);
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
      const int row = (16 * dt + col) * BS;
      const uint8_t* at = vc + (int64_t)max(b.v[0], 0) * p.v_block_stride;
      if constexpr (BS == 8) {
        const uint8_t* next = vc + (int64_t)max(b.v[NB - 1], 0) * p.v_block_stride;
        const uint2 x = *reinterpret_cast<const uint2*>(at + row), y = *reinterpret_cast<const uint2*>(next + row);
        vx[dt] = make_uint4(x.x, x.y, y.x, y.y);
      } else {
        vx[dt] = *reinterpret_cast<const uint4*>(at + row + (BS == 32 ? 16 * (g & 1) : 0));
      }
    }
  };
  // One branch a tile and product: with one at each conversion of codes the products
  // stood alone between waits.
  f32x4 s[4];
  auto scores = [&](auto careful) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < 4; ++u) s[u] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < KL; ++j)
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        constexpr bool SPECIAL = decltype(careful)::value;
        s[u] = Mma<QT>::k32(decode8<QT>(make_uint2(kx[u][j].x, kx[u][j].y), SPECIAL), qf[2 * j], s[u]);
        s[u] = Mma<QT>::k32(decode8<QT>(make_uint2(kx[u][j].z, kx[u][j].w), SPECIAL), qf[2 * j + 1], s[u]);
      }
  };
  auto special4 = [](uint4 x) {
    return fp8x4_special(x.x) | fp8x4_special(x.y) | fp8x4_special(x.z) | fp8x4_special(x.w);
  };
  // Tile v, whose K and V are in registers (or on their way); the next one's, v + NW, is
  // loaded behind the last use of each, where there is one.
  auto attend = [&](int v, Blocks& b, const Blocks& next, auto more) __attribute__((always_inline)) {
    const int t0 = q.start_of(v), tv = t0 + 16 * g;
    const bool held = NB == 1 ? b.v[0] >= 0 : b.v[0] >= 0 && b.v[NB - 1] >= 0;
    // (K's blocks are V's, of other lanes.)
    const bool whole = t0 + kScaledTile - 1 <= pmin && (t0 > pmax - window || t0 + kScaledTile <= sinks) && __all(held);
    uint32_t probe = 0;
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
      for (int j = 0; j < KL; ++j) probe |= special4(kx[u][j]);
    if (__any(probe != 0u))
      scores(std::true_type{});
    else
      scores(std::false_type{});
    if constexpr (decltype(more)::value) load_k(next);
    // Bit r: this lane's row sees token tv + r.
    uint32_t have = 0xffffu;
    if (!whole) {
      have = (b.v[0] >= 0 ? (NB == 1 ? 0xffffu : 0xffu) : 0u) | (NB == 2 && b.v[NB - 1] >= 0 ? 0xff00u : 0u);
    }
    const uint32_t sees = whole ? 0xffffu : have & seen16(pos, tv, window, sinks);
    float ks[NB], top[NB];
#pragma unroll
    for (int i = 0; i < NB; ++i) ks[i] = sx[i].x * p.scale_log2, top[i] = kNoScore;
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
      for (int r = 0; r < 4; ++r) s[u][r] *= ks[NB == 2 ? u / 2 : 0];
    if (!whole)
#pragma unroll
      for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int r = 0; r < 4; ++r) s[u][r] = sees >> (4 * u + r) & 1u ? s[u][r] : kNoScore;
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
      for (int r = 0; r < 4; ++r) top[NB == 2 ? u / 2 : 0] = fmaxf(top[NB == 2 ? u / 2 : 0], s[u][r]);
    float mt = fmaxf(top[0], top[NB - 1]);
    // log2 of the largest product of a weight, 2^(score - from), and its scale.  (A block of
    // zeros has no say, nor one without weight: nothing that the row sees, or less than
    // float32's normal range holds.)
    auto weighs = [&](int i, float from) { return top[i] - from >= kLeastWeight; };
    auto product = [&](float from) __attribute__((always_inline)) {
      float x = kNoScore;
#pragma unroll
      for (int i = 0; i < NB; ++i)
        if (weighs(i, from) && sx[i].y > 0.f)
          x = fmaxf(x, top[i] - from + (float)__builtin_amdgcn_frexp_expf(sx[i].y));
      return x;
    };
    if (__any(mt > m + kExtendSlack<QT> || product(m) > e + kExtendSlack<QT> || (m == kNoScore && mt != kNoScore))) {
      // (m is the largest score itself: a row's heaviest weight is then a power of two, and
      // nothing of it is lost when it is rounded.  With m moved by whole steps errors against
      // 64 bits were 0.0024 instead of 0.0017.)
      mt = fmaxf(column_max(mt), m);
      const float by = m - (mt == kNoScore ? 0.f : mt), was = __builtin_ceilf(e);
      e = fmaxf(fmaxf(e - (mt - m), column_max(product(mt))), kNoExponent);
      m = mt;
      const float alpha = __builtin_amdgcn_exp2f(by), alpha_o = __builtin_amdgcn_exp2f(by + (was - __builtin_ceilf(e)));
      l *= alpha;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int r = 0; r < 4; ++r) o[dt][r] *= alpha_o;
    }
    const float from = (m == kNoScore ? 0.f : m) - (weight_shift<QT>(kExtendSlack<QT>) + kSumShift);
    float vs[NB];
#pragma unroll
    for (int i = 0; i < NB; ++i)
      vs[i] = weighs(i, m) ? __builtin_amdgcn_ldexpf(sx[i].y, -(int)__builtin_ceilf(e) - kSumShift) : 0.f;
    uint4 wf[2];
    {
      uint32_t w[8];
#pragma unroll
      for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int r = 0; r < 4; r += 2) {
          const float a = __builtin_amdgcn_exp2f(s[u][r] - from), c = __builtin_amdgcn_exp2f(s[u][r + 1] - from);
          l += a + c;
          w[2 * u + r / 2] = pack_weights<QT>(a * vs[NB == 2 ? u / 2 : 0], c * vs[NB == 2 ? u / 2 : 0]);
        }
      wf[0] = make_uint4(w[0], w[1], w[2], w[3]);
      wf[1] = make_uint4(w[4], w[5], w[6], w[7]);
    }
    probe = 0;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) probe |= special4(vx[dt]);
    const bool special = __any(probe != 0u);
    // (Tokens that a row does not see have weight 0, and finite values: nothing reaches it.)
    if (!special) {
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        o[dt] = Mma<QT>::k32(decode8<QT>(make_uint2(vx[dt].x, vx[dt].y), false), wf[0], o[dt]);
        o[dt] = Mma<QT>::k32(decode8<QT>(make_uint2(vx[dt].z, vx[dt].w), false), wf[1], o[dt]);
      }
    } else {
      // A weight of 0 times inf or NaN is NaN: what a row does not see is taken out of V,
      // one query position at a time where the rows see different tokens.
      const bool one = ONE || (t0 + kScaledTile - 1 <= pmin && (t0 > pmax - window || t0 + kScaledTile <= sinks));
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        const uint4 y0 = decode8<QT>(make_uint2(vx[dt].x, vx[dt].y), true);
        const uint4 y1 = decode8<QT>(make_uint2(vx[dt].z, vx[dt].w), true);
        if (one) {
          o[dt] = Mma<QT>::k32(keep8(y0, sees), wf[0], o[dt]);
          o[dt] = Mma<QT>::k32(keep8(y1, sees >> 8), wf[1], o[dt]);
        } else {
#pragma unroll 1
          for (int at = pmin; at <= pmax; ++at) {
            const uint32_t keep = have & seen16(at, tv, window, sinks);
            f32x4 n = Mma<QT>::k32(keep8(y0, keep), wf[0], o[dt]);
            n = Mma<QT>::k32(keep8(y1, keep >> 8), wf[1], n);
#pragma unroll
            for (int r = 0; r < 4; ++r) o[dt][r] = pos == at ? n[r] : o[dt][r];
          }
        }
      }
    }
    if constexpr (decltype(more)::value) load_v(next);
  };
  while (next_piece(c)) {
    begin_piece();
    // Each wavefront takes every fourth tile.
    if (v0 + wave < v1) {
      Blocks b0 = load_blocks(v0 + wave), b1 = load_blocks(v0 + wave + NW);
      check_blocks(b0);
      load_k(b0);
      load_v(b0);
      int v = v0 + wave;
      if (v + NW < v1) {
        for (; v + 2 * NW < v1; v += NW) {
          check_blocks(b1);
          const Blocks after = load_blocks(v + 2 * NW);
          attend(v, b0, b1, std::true_type{});
          b0 = b1;
          b1 = after;
        }
        check_blocks(b1);
        attend(v, b0, b1, std::true_type{});
        b0 = b1;
        v += NW;
      }
      attend(v, b0, b0, std::false_type{});
    }

    // The wavefronts' states: column col is row row0 + col.
    l = column_sum(l) * (1.f / (1 << kSumShift));
    e = __builtin_ceilf(e);
    if (g == 0) s_m[wave][col] = m, s_l[wave][col] = l, s_e[wave][col] = e;
    __syncthreads();
    float M = kNoScore, L = 0.f, E = kNoExponent;
#pragma unroll
    for (int w = 0; w < NW; ++w) M = fmaxf(M, s_m[w][col]);
    {
      const float ref = M == kNoScore ? 0.f : M;
#pragma unroll
      for (int w = 0; w < NW; ++w) {
        const float by = s_m[w][col] - ref;
        L += s_l[w][col] * __builtin_amdgcn_exp2f(by);
        E = fmaxf(E, __builtin_ceilf(by + s_e[w][col]));
      }
      const float f = __builtin_amdgcn_exp2f(m - ref + (e - E));
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int r = 0; r < 4; ++r) s_o[wave][dt * 4 + r][lane] = o[dt][r] * f;
    }
    const Piece& done = c;
    __syncthreads();
    auto row_of = [&](int i) {
      const int tok = token_of(row0 + i);
      return ((int64_t)done.q.q.start + tok) * p.num_heads + h0 + (row0 + i - tok * group);
    };
    // out = O 2^E / L (NaN stays NaN, a row without tokens is zero).
    auto inverse = [](float l) { return l > 0.f ? 1.f / l : l == 0.f ? 0.f : l; };
    const float inv = inverse(L);
    // Wavefront w sums the 16-dimension tiles w, w + 4, ...
    const int nr = done.nr;
    const int64_t slot = (int64_t)blockIdx.x * 2 + (crew == done.w_first ? 1 : 0);
    float* state = p.ws_o + slot * (16 * D);
    const int64_t row = row_of(min(col, nr - 1));
#pragma unroll
    for (int k = 0; k < (DT + 3) / 4; ++k) {
      const int dt = 4 * k + wave;
      const int d = 16 * dt + 4 * g;
      if (dt >= DT || col >= nr) continue;
      float y[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int at = dt * 4 + r;
        const float sum = s_o[0][at][lane] + s_o[1][at][lane] + s_o[2][at][lane] + s_o[3][at][lane];
        y[r] = __builtin_amdgcn_ldexpf(sum * inv, (int)E);
      }
      if (done.parts == 1) {
        uint2 z;
        z.x = pack2(from_f32<QT>(y[0]), from_f32<QT>(y[1]));
        z.y = pack2(from_f32<QT>(y[2]), from_f32<QT>(y[3]));
        *reinterpret_cast<uint2*>(static_cast<QS*>(p.out) + row * D + d) = z;
      } else {
        store_agent(state + col * D + d, y[0], y[1]);
        store_agent(state + col * D + d + 2, y[2], y[3]);
      }
    }
    if (done.parts > 1) {
      if (wave == 0 && g == 0 && col < nr) store_agent(p.ws_ml + (slot * 16 + col) * 2, M, L);
      // The piece that arrives last merges all, in their order.
      wait_agent_stores();
      __syncthreads();
      if (tid == 0) s_last = arrived_last(p.counters + done.w_first * p.units + unit, done.parts);
      __syncthreads();
      if (s_last) {
        // Four dimensions of a row a thread; where that leaves threads over, several
        // share the parts of a row and meet in LDS.  Many loads in flight: a part at a
        // time took 20 us for 32 of them.
        const int quads = nr * (D / 4);
        auto merge = [&](auto at_once, auto shared) __attribute__((always_inline)) {
          constexpr int U = decltype(at_once)::value;
          constexpr bool SHARED = decltype(shared)::value;
          const int sharers = SHARED ? min(256 / quads, 4) : 1;
          const int each = SHARED ? (done.parts + sharers - 1) / sharers : done.parts;
          for (int i = tid; i < quads * sharers; i += 256) {
            const int who = SHARED ? i / quads : 0, quad = i - who * quads;
            const int r = quad / (D / 4), d = 4 * (quad - r * (D / 4));
            const int first = who * each, last = min(first + each, done.parts);
            float mm = kNoScore, ll = 0.f, y[4] = {0.f, 0.f, 0.f, 0.f};
            for (int k0 = first; k0 < last; k0 += U) {
              float2 ml[U], xa[U], xb[U];
#pragma unroll
              for (int k = 0; k < U; ++k) {
                const int part = min(k0 + k, last - 1);
                const int64_t from = ((int64_t)(done.w_first + part) * p.units + unit) * 2 + (part == 0 ? 1 : 0);
                ml[k] = load_agent(p.ws_ml + (from * 16 + r) * 2);
                xa[k] = load_agent(p.ws_o + from * (16 * D) + r * D + d);
                xb[k] = load_agent(p.ws_o + from * (16 * D) + r * D + d + 2);
              }
              const float before = mm;
#pragma unroll
              for (int k = 0; k < U; ++k) mm = fmaxf(mm, ml[k].x);
              const float rf = mm == kNoScore ? 0.f : mm, f0 = __builtin_amdgcn_exp2f(before - rf);
              ll *= f0;
#pragma unroll
              for (int j = 0; j < 4; ++j) y[j] *= f0;
#pragma unroll
              for (int k = 0; k < U; ++k) {
                if (k0 + k >= last) continue;
                const float f = __builtin_amdgcn_exp2f(ml[k].x - rf) * ml[k].y;
                ll += f;
                y[0] += f * xa[k].x, y[1] += f * xa[k].y, y[2] += f * xb[k].x, y[3] += f * xb[k].y;
              }
            }
            if constexpr (SHARED) {
              float* mine = &s_o[0][0][0] + i * 8;
              mine[0] = mm, mine[1] = ll, mine[2] = y[0], mine[3] = y[1], mine[4] = y[2], mine[5] = y[3];
            } else {
              const float by = inverse(ll);
              uint2 z;
              z.x = pack2(from_f32<QT>(y[0] * by), from_f32<QT>(y[1] * by));
              z.y = pack2(from_f32<QT>(y[2] * by), from_f32<QT>(y[3] * by));
              *reinterpret_cast<uint2*>(static_cast<QS*>(p.out) + row_of(r) * D + d) = z;
            }
          }
          if constexpr (SHARED) {
            __syncthreads();
            if (tid < quads) {
              const int r = tid / (D / 4), d = 4 * (tid - r * (D / 4));
              float mm = kNoScore, ll = 0.f, y[4] = {0.f, 0.f, 0.f, 0.f};
              for (int k = 0; k < sharers; ++k) mm = fmaxf(mm, (&s_o[0][0][0])[(k * quads + tid) * 8]);
              const float rf = mm == kNoScore ? 0.f : mm;
              for (int k = 0; k < sharers; ++k) {
                const float* from = &s_o[0][0][0] + (k * quads + tid) * 8;
                const float f = __builtin_amdgcn_exp2f(from[0] - rf);
                ll += f * from[1];
#pragma unroll
                for (int j = 0; j < 4; ++j) y[j] += f * from[2 + j];
              }
              const float by = inverse(ll);
              uint2 z;
              z.x = pack2(from_f32<QT>(y[0] * by), from_f32<QT>(y[1] * by));
              z.y = pack2(from_f32<QT>(y[2] * by), from_f32<QT>(y[3] * by));
              *reinterpret_cast<uint2*>(static_cast<QS*>(p.out) + row_of(r) * D + d) = z;
            }
          }
        };
        static_assert(sizeof(s_o) >= 256 * 8 * sizeof(float), "room for the sharers' sums");
        if (done.parts <= 4)
          merge(std::integral_constant<int, 4>{}, std::false_type{});
        else if (quads <= 128)
          merge(std::integral_constant<int, 16>{}, std::true_type{});
        else
          merge(std::integral_constant<int, 16>{}, std::false_type{});
      }
    }
    __syncthreads();  // (the next piece writes the wavefronts' states again)
  }
}

template <class QT, int D, int BS> hipError_t launch_scaled_d(const ScaledAttentionParams& p, hipStream_t stream) {
  const dim3 grid((unsigned)scaled_groups(p.workgroups, p.num_tokens, p.num_seqs, p.num_heads, D, p.query_start_loc != nullptr));
  if (p.max_query_len == 1)
    hipLaunchKernelGGL((scaled_attention_kernel<QT, D, BS, true>), grid, dim3(256), 0, stream, p);
  else
    hipLaunchKernelGGL((scaled_attention_kernel<QT, D, BS, false>), grid, dim3(256), 0, stream, p);
  return hipGetLastError();
}

template <class QT, int BS>
hipError_t launch_scaled_attention(const ScaledAttentionParams& p, int head_size, hipStream_t stream) {
  switch (head_size) {
    case 32: return launch_scaled_d<QT, 32, BS>(p, stream);
    case 64: return launch_scaled_d<QT, 64, BS>(p, stream);
    case 80: return launch_scaled_d<QT, 80, BS>(p, stream);
    case 96: return launch_scaled_d<QT, 96, BS>(p, stream);
    case 112: return launch_scaled_d<QT, 112, BS>(p, stream);
    case 128: return launch_scaled_d<QT, 128, BS>(p, stream);
    case 192: return launch_scaled_d<QT, 192, BS>(p, stream);
    case 256: return launch_scaled_d<QT, 256, BS>(p, stream);
  }
  return hipErrorInvalidValue;
}

}  // namespace pkv
