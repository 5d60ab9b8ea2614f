// Whole-number arithmetic with which launches find their work, the same on host and device
// (tests/schedule_check.cpp compares it with plain division and counting).
#pragma once

#include <cstdint>

namespace pkv {

// n / d for n below 2^31 by a product: with 2^shift the least power of two that is at least
// d, m = 2^(31 + shift) / d rounded up exceeds the quotient by under 2^-31, too little to
// reach n's next multiple of d.
struct Reciprocal {
  uint32_t m;
  int32_t shift;  // 0: d is 1
  __host__ __device__ __forceinline__ int of(int n) const {
    return shift == 0 ? n : (int)((uint32_t)((uint64_t)(uint32_t)n * m >> 32) >> (shift - 1));
  }
};
inline Reciprocal reciprocal(int64_t d) {
  Reciprocal r = {0, 0};
  while ((int64_t)1 << r.shift < d) ++r.shift;
  if (r.shift > 0) r.m = (uint32_t)((((uint64_t)1 << (31 + r.shift)) + (uint64_t)d - 1) / (uint64_t)d);
  return r;
}

// ---- attention over caches with a scale for each block and head (scaled_attention_impl.h) ----

constexpr int kScaledTile = 64;    // tokens
// What an item's start costs, in tiles (3, 5 and 8: four sequences of 4096 tokens 19.2, 17.7
// and 17.5 us, 64 of 533 .. 4097 69.1, 71.4 and 71.4, 256 of 300 .. 1700 114, 113 and 112).
constexpr int kScaledStart = 5;
// The least span of a workgroup, in tiles (5, 7 and 9: one sequence of 500 tokens 11.5, 11.6
// and 10.4 us, four of 4096 18.8, 18.9 and 17.6, one of 8190 16.5, 15.7 and 16.5).
constexpr int kScaledLeast = 9;
constexpr int kScaledWhole = 13;   // the longest item, its start with it, of sequences that get a crew each
constexpr int kScaledWorkgroups = 512;  // two a CU stay resident (one above head size 128)

// Crew of a workgroup, of crews of `units` workgroups each: by 2^32 / units rounded up (units
// of one crew alone are never taken apart, nor is a crew of one).
inline uint32_t unit_reciprocal(int64_t units) {
  const int64_t r = (((int64_t)1 << 32) + units - 1) / units;
  return r > UINT32_MAX ? UINT32_MAX : (uint32_t)r;
}
__host__ __device__ __forceinline__ int crew_of(uint32_t block, int units, int crews, uint32_t reciprocal) {
  const int quotient = units == 1 ? (int)block : (int)((uint64_t)block * reciprocal >> 32);
  return crews == 1 ? 0 : quotient;
}

// What the crew of span [x0, x1) takes of the item [begin, end) of the line: [from, to), empty
// or one of `parts` pieces, the first of them by crew `first`.
struct ScaledPiece {
  int from, to, parts, first;
};
__host__ __device__ __forceinline__ ScaledPiece scaled_piece(int begin, int end, int x0, int x1, int span, int crew,
                                                             bool apiece) {
  const int snap = span / 4 < 4 ? span / 4 : 4;
  // A cut near a sequence's begin or end moves there: a piece costs about kScaledStart
  // tiles, wherever it is.
  auto cut = [&](int x) {
    return x <= begin || x - begin < kScaledStart + snap ? begin : x >= end || end - x < snap ? end : x;
  };
  ScaledPiece c;
  c.from = x0 <= begin ? begin : cut(x0);
  c.to = x1 >= end ? end : cut(x1);
  c.parts = 1;
  c.first = crew;
  if (!apiece) {
    const int k0 = (begin + kScaledStart + snap + span - 1) / span, k1 = (end - snap) / span;
    c.parts = (k1 - k0 + 1 > 0 ? k1 - k0 + 1 : 0) + 1;
    if (c.parts > 1) c.first = k0 - 1;
  }
  return c;
}

}  // namespace pkv
