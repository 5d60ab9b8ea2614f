// Block tables, slots and positions of one step, from request lengths.
//
// Sequence s of the step belongs to row r = rows[s] of the request table, holds
// c tokens when the step is done, n of them new.  Its blocks number have =
// ceil((c - n) / bs) before and need = ceil(c / bs) after; with off the sum of
// need - have over the sequences before it, its table is
//   table[b] = request[r][b]                  for b < have
//              new_blocks[off + b - have]     for have <= b < need   (also stored to request[r][b])
//              -1                             beyond,
// and its i-th new token sits at position p = c - n + i, in slot
// table[p / bs] * bs + p % bs.  Tokens of all sequences lie end to end.
//
// Every workgroup computes the two prefix sums (new tokens, new blocks) over all
// sequences by itself, so that one launch does without a second pass or a wait
// between workgroups; a second launch would cost microseconds.  Each reads 12 bytes a
// sequence from the L2, twice, and there is one for each sequence: with one new
// token each, 64 sequences take 4.7 us in a captured graph, 512 7.7, 1024 14, 2048 55
// and 4096 188.  A new token's block comes from new_blocks directly, never from what
// this launch writes to the request table.
// Bound: the latency of the chain lengths -> sums -> block -> slot: 4.2 us for 64
// decodes and 9.4 us for 16384 new tokens of 211 sequences (16 workgroups, four
// rounds of search and dependent loads each) in a kernel trace, where the bytes (0.1
// and 0.9 MB) would take below 1 us.
#include "pkv_launch.h"

namespace pkv {

namespace {

constexpr int kThreads = 256;
constexpr int kTokensPerGroup = 1024;

struct Seq {
  int32_t row, first, have, need, tokens;  // first: position of the first new token
};

__device__ __forceinline__ Seq load_seq(const StepTablesParams& p, int s) {
  const int64_t capacity = (int64_t)p.max_blocks * p.block_size;
  const int32_t row = p.rows[s];
  int32_t c = p.context_lens[s], n = p.query_lens[s];
  // No request, no context, or one that the table cannot hold: an empty sequence.
  if (row < 0 || row >= p.num_requests || c <= 0 || c > capacity) c = 0;
  n = min(max(n, 0), c);
  const int32_t bs = p.block_size;
  Seq q;
  q.row = row;
  q.first = c - n;
  q.tokens = n;
  q.have = (int32_t)(((int64_t)q.first + (bs - 1)) / bs);
  q.need = (int32_t)(((int64_t)c + (bs - 1)) / bs);
  return q;
}

// The new block number i of the step, -1 if there are fewer.
__device__ __forceinline__ int32_t new_block(const StepTablesParams& p, int64_t i) {
  return i < p.num_new_blocks ? p.new_blocks[i] : -1;
}

__global__ __launch_bounds__(kThreads) void step_tables_kernel(StepTablesParams p, int token_groups) {
  // First token and first new block of every sequence, saturated at 2^31 - 1
  // (beyond the last token and new block that a call can have).
  __shared__ int32_t s_tok[kMaxStepSeqs + 1];
  __shared__ int32_t s_blk[kMaxStepSeqs];
  __shared__ int64_t s_sum[2][kThreads / 64];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int per = (p.num_seqs + kThreads - 1) / kThreads;
  const int s0 = min(tid * per, p.num_seqs), s1 = min(s0 + per, p.num_seqs);
  int64_t tok = 0, blk = 0;
  for (int s = s0; s < s1; ++s) {
    const Seq q = load_seq(p, s);
    tok += q.tokens;
    blk += q.need - q.have;
  }
  const int64_t own_tok = tok, own_blk = blk;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int64_t a = __shfl_up(tok, d), b = __shfl_up(blk, d);
    if (lane >= d) tok += a, blk += b;
  }
  if (lane == 63) s_sum[0][wave] = tok, s_sum[1][wave] = blk;
  __syncthreads();
  for (int w = 0; w < wave; ++w) tok += s_sum[0][w], blk += s_sum[1][w];
  tok -= own_tok;
  blk -= own_blk;
  for (int s = s0; s < s1; ++s) {
    const Seq q = load_seq(p, s);
    s_tok[s] = (int32_t)min(tok, (int64_t)INT32_MAX);
    s_blk[s] = (int32_t)min(blk, (int64_t)INT32_MAX);
    tok += q.tokens;
    blk += q.need - q.have;
  }
  if (p.num_seqs == 0 && tid == 0) s_tok[0] = 0;
  if (s1 == p.num_seqs && s0 < s1) s_tok[p.num_seqs] = (int32_t)min(tok, (int64_t)INT32_MAX);
  __syncthreads();

  if ((int)blockIdx.x < token_groups) {
    if (blockIdx.x == 0)
      for (int s = tid; s <= p.num_seqs; s += kThreads) p.query_start_loc[s] = s_tok[s];
    // (Counted from the group's first token: num_tokens may be 2^31 - 1.)
    const int t0 = blockIdx.x * kTokensPerGroup, count = min(kTokensPerGroup, p.num_tokens - t0);
    for (int i = tid; i < count; i += kThreads) {
      const int t = t0 + i;
      int32_t slot = -1, pos = 0;
      if (t < s_tok[p.num_seqs]) {
        int lo = 0, hi = p.num_seqs;  // s_tok[lo] <= t < s_tok[hi]
        while (hi - lo > 1) {
          const int mid = (lo + hi) >> 1;
          if (s_tok[mid] <= t) lo = mid;
          else hi = mid;
        }
        const Seq q = load_seq(p, lo);
        pos = q.first + (t - s_tok[lo]);
        const int32_t b = pos / p.block_size;
        const int32_t id = b < q.have ? p.request_blocks[(int64_t)q.row * p.max_blocks + b]
                                      : new_block(p, (int64_t)s_blk[lo] + b - q.have);
        const int64_t at = (int64_t)id * p.block_size + (pos - b * p.block_size);
        slot = id >= 0 && at <= INT32_MAX ? (int32_t)at : -1;
      }
      p.slot_mapping[t] = slot;
      p.positions[t] = pos;
    }
    return;
  }
  const int s = (int)blockIdx.x - token_groups;
  const Seq q = load_seq(p, s);
  for (int64_t b = tid; b < p.max_blocks; b += kThreads) {
    int32_t id = -1;
    if (b < q.have) {
      id = p.request_blocks[(int64_t)q.row * p.max_blocks + b];
    } else if (b < q.need) {
      id = new_block(p, (int64_t)s_blk[s] + b - q.have);
      p.request_blocks[(int64_t)q.row * p.max_blocks + b] = id;
    }
    p.block_tables[(int64_t)s * p.max_blocks + b] = id;
  }
}

}  // namespace

hipError_t launch_step_tables(const StepTablesParams& p, hipStream_t stream) {
  // (At least one token group: it writes query_start_loc.)
  const int groups = (int)((std::max<int64_t>(p.num_tokens, 1) + kTokensPerGroup - 1) / kTokensPerGroup);
  hipLaunchKernelGGL(step_tables_kernel, dim3((unsigned)(groups + p.num_seqs)), dim3(kThreads), 0, stream, p, groups);
  return hipGetLastError();
}

}  // namespace pkv
