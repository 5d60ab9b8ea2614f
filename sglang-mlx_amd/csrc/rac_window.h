// Runs of whole blocks among the tokens that a paged append writes, shared by
// the kernels that append (reshape_and_cache.hip, norm_rope.hip).
#pragma once

#include "pkv_launch.h"

namespace pkv {

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

}  // namespace pkv
