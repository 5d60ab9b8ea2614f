// Attention of single and drafted tokens over a paged cache of E4M3 codes with a scale
// for each (block, KV head) of K and of V.
//
// K_t = c_t ks_b, V_t = d_t vs_b for the codes c, d of token t in block b:
//   out = sum_t w_t vs_b d_t / sum_t w_t,   w_t = exp(scale ks_b (q . c_t) - m).
// The codes are exact in the queries' 16-bit type, so both products run on them as they
// are; ks multiplies a score in float32, vs a weight before it is rounded to 16 bits.
// There vs enters as vs / 2^e, e the largest exponent of a scale that the row has seen: the
// weights keep the range that float16 has, whatever the scales' size, and the output
// returns to true size at the end (2^e; powers of two, so that nothing is rounded).
//
// Query rows, products and masks are those of extend_few_kernel (extend_impl.h): 16 rows
// of a sequence and KV head, 32-token tiles straight from the cache to the matrix units'
// registers, S^T = K Q^T, O^T = V^T P^T, lane group g holding tokens 8 g ..+7 of a tile.
// Eight tokens never cross a block, so a lane has one K scale and one V scale a tile.
//
// Schedule: the items (sequence, KV head, 16 rows) lie end to end, each its tiles and a
// start-up's worth of them long, and every workgroup takes an equal span, so that ragged
// contexts load the chip evenly and one long context fills it.  Pieces of an item leave
// their states in the workspace; the one that arrives last merges them in their order
// (no result depends on timing, nobody waits for another workgroup).
#pragma once

#include "extend_impl.h"

namespace pkv {

constexpr int kScaledTile = 32;

// Sequence s of a call: its query rows and the tiles of 32 tokens that they see.
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
  constexpr int KL = (D + 63) / 64;  // 16-byte loads of a K row's codes by a lane (each two products)
  constexpr int DT = D / 16;
  constexpr int NW = 4;
  __shared__ float s_o[NW][DT * 4][64];
  __shared__ float s_m[NW][16], s_l[NW][16], s_e[NW][16];
  __shared__ int s_sum[NW], s_base, s_first, s_last;

  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int group = p.group, H = p.num_kv_heads;
  if ((int)blockIdx.x >= p.workgroups) {
    // Rows behind the last sequence become zeros.
    const int last = min(max(p.query_start_loc[p.num_seqs], 0), p.num_tokens);
    const int groups = gridDim.x - p.workgroups;
    const int share = (p.num_tokens - last + groups - 1) / groups;
    const int64_t t0 = last + (int64_t)(blockIdx.x - p.workgroups) * share;
    zero_tokens<QT, 256>(p, D, t0, min(t0 + share, (int64_t)p.num_tokens), 0, p.num_heads);
    return;
  }
  int tid = threadIdx.x, lane = tid & 63;
  // Length of one item of sequence s (a sequence without rows has none).
  auto item_length = [](const ScaledSeq& q) { return q.q.count == 0 ? 0 : q.tiles + kScaledStart; };
  // The sum of all lengths (below 2^31), and the sequence in which this workgroup's span
  // begins: each thread sums a run of sequences.
  const int run = (p.num_seqs + 255) / 256;
  int mine = 0;
  for (int s = tid * run; s < min((tid + 1) * run, p.num_seqs); ++s) mine += item_length(scaled_seq(p, s)) * p.units;
  int sum = mine;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int a = __shfl_up(sum, d);
    if (lane >= d) sum += a;
  }
  if (lane == 63) s_sum[wave] = sum;
  __syncthreads();
  int total = 0, below = sum - mine;
#pragma unroll
  for (int w = 0; w < NW; ++w) {
    const int a = __builtin_amdgcn_readfirstlane(s_sum[w]);
    if (w < wave) below += a;
    total += a;
  }
  const int span = max((total + p.workgroups - 1) / p.workgroups, kScaledLeast);
  if ((int64_t)blockIdx.x * span >= total) return;
  const int x0 = blockIdx.x * span, x1 = min(span, total - x0) + x0;
  if (x0 >= below && x0 < below + mine) {
    int at = below;
    int s = tid * run;
    for (;; ++s) {
      const int n = item_length(scaled_seq(p, s)) * p.units;
      if (x0 < at + n) break;
      at += n;
    }
    s_first = s, s_base = at;
  }
  __syncthreads();
  int seq = __builtin_amdgcn_readfirstlane(s_first);
  int base = __builtin_amdgcn_readfirstlane(s_base);  // where the sequence's first item begins

  const int window = p.window > 0 ? p.window : p.max_seq_len;
  const int sinks = p.window > 0 ? p.sinks : 0;
  constexpr int shift = BS == 8 ? 3 : BS == 16 ? 4 : 5, bs = BS;

  int x = x0;
  while (x < x1) {
    const ScaledSeq q = scaled_seq(p, seq);
    const int length = item_length(q);
    if (x - base >= length * p.units) {
      base += length * p.units;
      ++seq;
      continue;
    }
    const int unit = (x - base) / length;
    const int begin = base + unit * length, end = begin + length;
    // Tile v sits at position begin + kScaledStart + v.
    const int tile0 = begin + kScaledStart;
    const int v0 = max(x - tile0, 0), v1 = max(min(x1, end) - tile0, 0);
    x = min(x1, end);
    // (Opaque to the compiler: addresses of a lane that no item changes would otherwise
    // stay in registers over the loop, 75 of them at head size 128.)
    asm volatile("" : "+v"(tid), "+v"(lane));
    const int g = lane >> 4, col = lane & 15;
    const int kvh = unit / p.slices, slice = unit - kvh * p.slices;
    const int h0 = kvh * group;
    if (q.tiles == 0) {
      // Nothing to attend: the rows are zeros, by the workgroup that has the item's end.
      if (x == end && slice == 0) zero_tokens<QT, 256>(p, D, q.q.start, q.q.start + q.q.count, h0, group);
      continue;
    }
    if (v0 >= v1) continue;  // (only the start-up of the item)
    const int w_first = tile0 / span, parts = (end - 1) / span - w_first + 1;
    // Row row0 + c, c < nr, is head (row0 + c) % group of token (row0 + c) / group;
    // this lane's is c = col.
    const int row0 = 16 * slice, nr = min(16, q.q.count * group - row0);
    if (nr <= 0) continue;
    const int first_pos = q.q.ctx - q.q.count;
    const int pmin = first_pos + row0 / group, pmax = first_pos + (row0 + nr - 1) / group;  // (uniform)
    const bool live = col < nr;
    const int my_row = row0 + min(col, nr - 1), token = my_row / group;
    const int pos = first_pos + token;
    auto row_of = [&](int c) {
      const int tok = (row0 + c) / group;
      return ((int64_t)q.q.start + tok) * p.num_heads + h0 + (row0 + c - tok * group);
    };
    uint4 qf[2 * KL];
    {
      const QS* src =
          static_cast<const QS*>(p.q) + (q.q.start + token) * p.q_stride + (int64_t)(h0 + (my_row - token * group)) * D;
#pragma unroll
      for (int j = 0; j < 2 * KL; ++j) {
        const int d = 64 * (j / 2) + 16 * g + 8 * (j & 1);
        qf[j] = live && d < D ? *reinterpret_cast<const uint4*>(src + d) : make_uint4(0, 0, 0, 0);
      }
    }
    const int32_t* table = p.block_tables + (int64_t)seq * p.max_blocks_per_seq;
    const uint8_t* kc = static_cast<const uint8_t*>(p.k_cache) + (int64_t)kvh * p.k_head_stride;
    const uint8_t* vc = static_cast<const uint8_t*>(p.v_cache) + (int64_t)kvh * p.v_head_stride;
    const float* scales = p.scales + 2 * kvh;

    f32x4 o[DT];
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) o[dt] = {0.f, 0.f, 0.f, 0.f};
    float m = kNoScore, l = 0.f;
    int e = kNoExponent;

    struct Blocks {
      int k, v;  // of this lane's K row and of its V pieces (and scales)
    };
    auto load_blocks = [&](int v) __attribute__((always_inline)) {
      Blocks b{-1, -1};
      if (v < v1) {
        const int t0 = q.start_of(v), tk = t0 + 8 * (col >> 2), tv = t0 + 8 * g;
        if (tk < q.q.ctx) b.k = table[tk >> shift];
        if (tv < q.q.ctx) b.v = table[tv >> shift];
      }
      auto valid = [&](int id) { return id >= 0 && (int64_t)id < p.num_blocks ? id : -1; };
      return Blocks{valid(b.k), valid(b.v)};
    };
    struct Tile {
      uint4 k[2][KL];
      uint2 v[DT];
      float2 scale;
    };
    // (A missing block's loads go to block 0; its tokens are masked.)
    auto load_tile = [&](Tile& t, int v, const Blocks& b) __attribute__((always_inline)) {
      const int t0 = q.start_of(v), tk = t0 + 8 * (col >> 2), tv = t0 + 8 * g;
      const uint8_t* kp = kc + (int64_t)max(b.k, 0) * p.k_block_stride + ((tk & (bs - 1)) + (col & 3)) * 16;
      const uint8_t* vp = vc + (int64_t)max(b.v, 0) * p.v_block_stride + (tv & (bs - 1));
      t.scale = *reinterpret_cast<const float2*>(scales + (int64_t)max(b.v, 0) * 2 * H);
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int j = 0; j < KL; ++j) {
          const int c = 4 * j + g;
          t.k[u][j] = c * 16 < D ? *reinterpret_cast<const uint4*>(kp + (c * bs + 4 * u) * 16) : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) t.v[dt] = *reinterpret_cast<const uint2*>(vp + (16 * dt + col) * bs);
    };
    auto attend = [&](const Tile& t, int v, const Blocks& b) __attribute__((always_inline)) {
      const int t0 = q.start_of(v), tv = t0 + 8 * g;
      uint32_t probe = 0;
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int j = 0; j < KL; ++j)
          probe |= fp8x4_special(t.k[u][j].x) | fp8x4_special(t.k[u][j].y) | fp8x4_special(t.k[u][j].z) |
                   fp8x4_special(t.k[u][j].w);
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) probe |= fp8x4_special(t.v[dt].x) | fp8x4_special(t.v[dt].y);
      const bool special = __any(probe != 0u);
      f32x4 s[2];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        s[u] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < KL; ++j) {
          s[u] = Mma<QT>::k32(decode8<QT>(make_uint2(t.k[u][j].x, t.k[u][j].y), special), qf[2 * j], s[u]);
          s[u] = Mma<QT>::k32(decode8<QT>(make_uint2(t.k[u][j].z, t.k[u][j].w), special), qf[2 * j + 1], s[u]);
        }
      }
      // Bit r: this lane's row sees token tv + r.
      const uint32_t sees = b.v >= 0 ? seen16(pos, tv, window, sinks) & 0xffu : 0u;
      const float ks = t.scale.x * p.scale_log2;
      float mt = kNoScore;
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          s[u][r] = sees >> (4 * u + r) & 1u ? s[u][r] * ks : kNoScore;
          mt = fmaxf(mt, s[u][r]);
        }
      // (A block of zeros, or without tokens that the rows see, has no say.)
      const int ve = sees != 0u && t.scale.y > 0.f ? __builtin_amdgcn_frexp_expf(t.scale.y) : kNoExponent;
      mt = fmaxf(column_max(mt), m);
      const int et = max(e, (int)column_max((float)ve));
      const float ref = mt == kNoScore ? 0.f : mt;
      const float alpha = __builtin_amdgcn_exp2f(m - ref);
      const float alpha_o = __builtin_amdgcn_ldexpf(alpha, max(e - et, -200));
      m = mt;
      e = et;
      l *= alpha;
      const float from = ref - weight_shift<QT>(1.f);
      const float vs = sees != 0u ? __builtin_amdgcn_ldexpf(t.scale.y, -max(e, kNoExponent + 1)) : 0.f;
      uint32_t w[4];
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int r = 0; r < 4; r += 2) {
          const float a = __builtin_amdgcn_exp2f(s[u][r] - from), c = __builtin_amdgcn_exp2f(s[u][r + 1] - from);
          l += a + c;
          w[2 * u + r / 2] = pack_weights<QT>(a * vs, c * vs);
        }
      const uint4 wf = make_uint4(w[0], w[1], w[2], w[3]);
      // What a token that a row does not see holds must not matter: it is taken out of
      // V, one query position at a time where the rows see different tokens.
      const bool one = ONE || (t0 + kScaledTile - 1 <= pmin && (t0 > pmax - window || t0 + kScaledTile <= sinks));
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        const uint4 y = decode8<QT>(t.v[dt], special);
#pragma unroll
        for (int r = 0; r < 4; ++r) o[dt][r] *= alpha_o;
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
    // Each wavefront takes every fourth tile; the next one loads while one is attended.
    Blocks b0 = load_blocks(v0 + wave), b1 = load_blocks(v0 + wave + NW);
    Tile x0t, x1t;
    if (v0 + wave < v1) load_tile(x0t, v0 + wave, b0);
    for (int v = v0 + wave; v < v1; v += 2 * NW) {
      Blocks b2 = load_blocks(v + 2 * NW);
      if (v + NW < v1) load_tile(x1t, v + NW, b1);
      attend(x0t, v, b0);
      if (v + NW >= v1) break;
      b0 = b2;
      b2 = load_blocks(v + 3 * NW);
      if (v + 2 * NW < v1) load_tile(x0t, v + 2 * NW, b0);
      attend(x1t, v + NW, b1);
      b1 = b2;
    }

    // The wavefronts' states: column col is row row0 + col.
    l = column_sum(l);
    if (g == 0) s_m[wave][col] = m, s_l[wave][col] = l, s_e[wave][col] = (float)e;
    __syncthreads();
    float M = kNoScore, L = 0.f, E = (float)kNoExponent;
#pragma unroll
    for (int w = 0; w < NW; ++w) M = fmaxf(M, s_m[w][col]), E = fmaxf(E, s_e[w][col]);
    {
      const float ref = M == kNoScore ? 0.f : M;
#pragma unroll
      for (int w = 0; w < NW; ++w) L += s_l[w][col] * __builtin_amdgcn_exp2f(s_m[w][col] - ref);
      const float f = __builtin_amdgcn_exp2f(m - ref) * __builtin_amdgcn_exp2f(fmaxf((float)e - E, -126.f));
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int r = 0; r < 4; ++r) s_o[wave][dt * 4 + r][lane] = o[dt][r] * f;
    }
    __syncthreads();
    // out = O 2^E / L (NaN stays NaN).
    auto finish = [](float o, float l, float e) {
      return l > 0.f ? __builtin_amdgcn_ldexpf(o / l, (int)e) : l == 0.f ? 0.f : l;
    };
    // Wavefront w sums the 16-dimension tiles w, w + 4, ...
    const int64_t slot = (int64_t)blockIdx.x * 2 + ((int)blockIdx.x == w_first ? 1 : 0);
    float* state = p.ws_o + slot * (16 * D);
    const int64_t row = row_of(min(col, nr - 1));
#pragma unroll
    for (int k = 0; k < (DT + 3) / 4; ++k) {
      const int dt = 4 * k + wave;
      const int d = 16 * dt + 4 * g;
      if (dt >= DT || !live) continue;
      float y[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int at = dt * 4 + r;
        y[r] = s_o[0][at][lane] + s_o[1][at][lane] + s_o[2][at][lane] + s_o[3][at][lane];
      }
      if (parts == 1) {
        uint2 z;
        z.x = pack2(from_f32<QT>(finish(y[0], L, E)), from_f32<QT>(finish(y[1], L, E)));
        z.y = pack2(from_f32<QT>(finish(y[2], L, E)), from_f32<QT>(finish(y[3], L, E)));
        *reinterpret_cast<uint2*>(static_cast<QS*>(p.out) + row * D + d) = z;
      } else {
        store_agent(state + col * D + d, y[0], y[1]);
        store_agent(state + col * D + d + 2, y[2], y[3]);
      }
    }
    if (parts > 1) {
      if (wave == 0 && g == 0 && live) {
        store_agent(p.ws_ml + (slot * 16 + col) * 4, M, L);
        store_agent(p.ws_ml + (slot * 16 + col) * 4 + 2, E, 0.f);
      }
      // The piece that arrives last merges all, in their order.
      wait_agent_stores();
      __syncthreads();
      if (tid == 0) s_last = arrived_last(p.counters + w_first, parts);
      __syncthreads();
      if (s_last) {
        for (int i = tid; i < nr * (D / 2); i += 256) {
          const int c = i / (D / 2), d = 2 * (i - c * (D / 2));
          auto slot_of = [&](int k) { return (int64_t)(w_first + k) * 2 + (k == 0 ? 1 : 0); };
          float mm = kNoScore, ee = (float)kNoExponent;
          for (int k = 0; k < parts; ++k) {
            const float* ml = p.ws_ml + (slot_of(k) * 16 + c) * 4;
            mm = fmaxf(mm, load_agent(ml).x);
            ee = fmaxf(ee, load_agent(ml + 2).x);
          }
          const float rf = mm == kNoScore ? 0.f : mm;
          float ll = 0.f, y = 0.f, z = 0.f;
          for (int k = 0; k < parts; ++k) {
            const float* ml = p.ws_ml + (slot_of(k) * 16 + c) * 4;
            const float2 a = load_agent(ml);
            const float f = __builtin_amdgcn_exp2f(a.x - rf);
            const float fo = f * __builtin_amdgcn_exp2f(fmaxf(load_agent(ml + 2).x - ee, -126.f));
            const float2 v = load_agent(p.ws_o + slot_of(k) * (16 * D) + c * D + d);
            ll += f * a.y;
            y += fo * v.x;
            z += fo * v.y;
          }
          *reinterpret_cast<uint32_t*>(static_cast<QS*>(p.out) + row_of(c) * D + d) =
              pack2(from_f32<QT>(finish(y, ll, ee)), from_f32<QT>(finish(z, ll, ee)));
        }
      }
    }
    __syncthreads();  // (the next item writes the wavefronts' states again)
  }
}

template <class QT, int D, int BS> hipError_t launch_scaled_d(const ScaledAttentionParams& p, hipStream_t stream) {
  const int64_t tail = p.query_start_loc != nullptr ? extend_tail_groups(p.num_tokens, p.num_heads, D, 1) : 0;
  const dim3 grid((unsigned)(p.workgroups + tail));
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
