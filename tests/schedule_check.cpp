// The launches' arithmetic (csrc/pkv_schedule.h) against plain division and counting, on the
// host.  Prints what is wrong; 0 where nothing is.
#include <cstdio>
#include <cstdlib>
#include <random>
#include <vector>

#define __host__
#define __device__
#define __forceinline__ inline
#include "pkv_schedule.h"

using namespace pkv;

static int wrong(const char* what, long long a, long long b, long long c) {
  std::printf("%s: %lld %lld %lld\n", what, a, b, c);
  return 1;
}

static int reciprocals(std::mt19937_64& rng) {
  const int64_t top = (int64_t)1 << 31;
  std::vector<int64_t> divisors;
  for (int64_t d = 1; d < 300; ++d) divisors.push_back(d);
  for (int i = 0; i < 3000; ++i) divisors.push_back(1 + (int64_t)(rng() % (uint64_t)(1 << 30)) >> rng() % 30);
  for (int s = 8; s <= 30; ++s)
    for (int64_t d : {((int64_t)1 << s) - 1, (int64_t)1 << s, ((int64_t)1 << s) + 1})
      if (d <= (int64_t)1 << 30) divisors.push_back(d);
  for (int64_t d : divisors) {
    if (d < 1) continue;
    const Reciprocal r = reciprocal(d);
    const int64_t last = (top - 1) / d * d;  // (the last multiple)
    std::vector<int64_t> ns = {0, 1, d - 1, d, d + 1, last - 1, last, top - 1};
    for (int i = 0; i < 40; ++i) {
      ns.push_back((int64_t)(rng() % (uint64_t)top));
      const int64_t multiple = (int64_t)(rng() % (uint64_t)(last / d + 1)) * d;
      ns.push_back(multiple);
      ns.push_back(multiple - 1);
    }
    for (int64_t n : ns)
      if (n >= 0 && n < top && r.of((int)n) != n / d) return wrong("reciprocal", n, d, r.of((int)n));
  }
  return 0;
}

static int crews() {
  for (int units = 1; units <= kScaledWorkgroups; ++units)
    for (int crews : {1, kScaledWorkgroups / units}) {
      const uint32_t r = unit_reciprocal(units);
      for (int block = 0; block < crews * units; ++block)
        if (crew_of(block, units, crews, r) != block / units) return wrong("crew", block, units, crews);
    }
  // A single crew may have more units.
  for (int units : {513, 4096, 1 << 20, (1 << 24) - 1})
    if (crew_of(units - 1, units, 1, unit_reciprocal(units)) != 0) return wrong("crew", units - 1, units, 1);
  return 0;
}

// The pieces of a line of sequences: each sequence's meet end to end, none is empty, their
// number is what each of them counts, the first's crew is the one they name, and no crew
// leaves more than one piece in either of its two places (first of a sequence, or not).
static int pieces(std::mt19937_64& rng, bool apiece) {
  auto any = [&](int lo, int hi) { return lo + (int)(rng() % (uint64_t)(hi - lo + 1)); };
  const int crews = any(1, 3) == 1 ? any(1, 8) : any(1, kScaledWorkgroups), n = apiece ? any(1, crews) : any(1, 700);
  const int longest = apiece ? kScaledWhole - kScaledStart : 1 << any(0, 11);
  std::vector<int> begin(n + 1, 0);
  for (int s = 0; s < n; ++s) {
    const int tiles = any(0, longest);
    begin[s + 1] = begin[s] + (tiles == 0 ? 0 : tiles + kScaledStart);
  }
  const int total = begin[n];
  const int span = apiece ? kScaledLeast : std::max((total + crews - 1) / crews, kScaledLeast);
  std::vector<int> firsts(crews, 0), others(crews, 0);
  for (int s = 0; s < n; ++s) {
    const int b = begin[s], e = begin[s + 1];
    if (b == e) continue;
    int at = b, count = 0, parts = -1, first = -1;
    for (int crew = 0; crew < crews; ++crew) {
      const int64_t start = (int64_t)crew * span;
      if (!apiece && start >= total) break;
      const int x0 = apiece ? b : (int)start, x1 = apiece ? e : std::min(span, total - x0) + x0;
      if (apiece ? crew != s : x1 <= b || x0 >= e) continue;
      const ScaledPiece c = scaled_piece(b, e, x0, x1, span, crew, apiece);
      if (c.from >= c.to) continue;
      if (c.from != at) return wrong("piece begins", c.from, at, s);
      // (Its tiles: behind the start.)
      if (std::max(c.from - b - kScaledStart, 0) >= c.to - b - kScaledStart) return wrong("no tile", c.from, c.to, b);
      if (parts < 0) parts = c.parts, first = crew;
      if (c.parts != parts || c.first != first) return wrong("parts", c.parts, parts, c.first);
      if (c.parts > 1 && first + count != crew) return wrong("crews of pieces", first, count, crew);
      if (c.parts > 1 && ++(crew == c.first ? firsts : others)[crew] > 1) return wrong("a place twice", crew, s, 0);
      at = c.to;
      ++count;
    }
    if (at != e) return wrong("piece ends", at, e, s);
    if (count != parts) return wrong("count", count, parts, s);
  }
  return 0;
}

int main() {
  std::mt19937_64 rng(7);
  if (reciprocals(rng) || crews()) return 1;
  for (int i = 0; i < 4000; ++i)
    if (pieces(rng, i % 4 == 0)) return 1;
  std::puts("as counted");
  return 0;
}
