// Host check of the cache attention's walk (cache_geom.h) against the mask's
// definition: every key that some row of a tile sees is in exactly one step,
// tiles called full are seen by every row, the parts of a split cover the steps
// once, the 32-bit words of the keys that a row sees are those keys, and page and slot numbers outside the cache are refused.
#include <climits>
#include <cstdio>
#include <cstdlib>
#include <vector>

#include "cache_geom.h"

using namespace chia;

static bool sees(const CacheMask& m, int i, int j, int S) {
  if (i < 0 || j < 0 || j >= S) return false;
  if (j < m.prefix) return true;
  const int d = i - j;
  if (m.causal && d < 0) return false;
  if (m.window > 0 && (m.causal ? d >= m.window : std::abs(d) >= m.window)) return false;
  if (m.blk > 0 && i / m.blk != j / m.blk) return false;
  return d % m.dil == 0;
}

int main() {
  long failures = 0, checked = 0;
  unsigned seed = 7;
  auto rnd = [&](int n) {
    seed = seed * 1664525u + 1013904223u;
    return (int)((seed >> 8) % (unsigned)n);
  };
  for (int it = 0; it < 30000; ++it) {
    CacheMask m;
    m.causal = rnd(2);
    m.window = rnd(3) ? 0 : 1 + rnd(150);
    m.dil = rnd(4) ? 1 : 2 + rnd(6);
    m.blk = rnd(3) ? 0 : 1 + rnd(120);
    m.prefix = m.dil > 1 || rnd(2) ? 0 : 1 + rnd(200);
    m.div_blk = make_udiv(m.blk > 0 ? m.blk : 1);
    m.div_dil = make_udiv(m.dil);
    m.comb = cache_comb(m.dil);
    const int S = rnd(10) ? rnd(400) : rnd(3);
    const int n = 1 + rnd(40), i0 = S - n + rnd(n), i1 = i0 + rnd(S - i0 > 0 ? S - i0 : 1);
    if (i1 >= S && S > 0) continue;
    const int kStepKeys = rnd(2) ? 32 : 64;
    const TileWalk w = cache_tile_walk(m, i0, i1, S, kStepKeys);
    std::vector<int> times(S + 64, 0);
    for (int s = 0; s < w.n; ++s) {
      const int c = walk_key(w, s);
      if (c < 0 || c % kStepKeys || c >= S + kStepKeys) ++failures;
      for (int x = 0; x < kStepKeys; ++x)
        if (c + x < S + 64) ++times[c + x];
      for (int len : {16, 32, 64}) {
        bool all = true;
        for (int i = i0; i <= i1; ++i)
          for (int x = 0; x < len; ++x) all = all && sees(m, i, c + x, S);
        if (walk_full(w, c, len) && !all) ++failures;
      }
    }
    for (int j = 0; j < S; ++j) {
      bool any = false;
      for (int i = i0; i <= i1; ++i) {
        const RowKeys k = cache_row_keys(m, i, S);
        const bool got = (j >= k.lo && j < k.hi && (i - j) % m.dil == 0) || j < k.pre;
        if (got != sees(m, i, j, S)) ++failures;
        any = any || got;
      }
      if (times[j] > 1 || (any && times[j] != 1)) ++failures;
      ++checked;
    }
    for (int i = i0; i <= i1; ++i) {
      const RowKeys k = cache_row_keys(m, i, S);
      for (int c = 0; c < S + 64; c += 16) {
        const uint32_t word = cache_seen(m, k, i, c);
        for (int x = 0; x < 32; ++x)
          if (((word >> x) & 1u) != (sees(m, i, c + x, S) ? 1u : 0u)) ++failures;
      }
    }
    for (int parts : {1, 2, 3, 7})
      for (int chunk : {1, 4, 8}) {
        const int c = walk_chunk(w.n, parts, chunk), used = (w.n + c - 1) / c;
        if (c < 1 || used > parts || (int64_t)used * c < w.n) ++failures;
      }
  }
  // causal walks skip what lies behind: a decoding step under a window reads only the window
  CacheMask m{1, 64, 1, 0, 0, make_udiv(1), make_udiv(1)};
  if (cache_tile_walk(m, 9999, 9999, 10000, 32).n > 3) ++failures;
  // far positions and reaches do not overflow
  const int big = (1 << 28) - 1;
  CacheMask f{0, big, 1, big, 1 << 28, make_udiv(big), make_udiv(1)};
  const RowKeys k = cache_row_keys(f, big - 1, big);
  if (k.lo != 0 || k.hi != big || k.pre != big) ++failures;
  // dilations at and past the word's width
  for (int dil : {31, 32, 33, 100, 1 << 28}) {
    const CacheMask far{1, 0, dil, 0, 0, make_udiv(1), make_udiv(dil), cache_comb(dil)};
    for (int i : {0, 31, 63, 200, 4095, big - 1}) {
      const RowKeys rk = cache_row_keys(far, i, i + 1);
      for (int c = i > 300 ? i - 300 : 0; c <= i; c += 16) {
        const uint32_t word = cache_seen(far, rk, i, c);
        for (int x = 0; x < 32; ++x)
          if (((word >> x) & 1u) != (sees(far, i, c + x, i + 1) ? 1u : 0u)) ++failures;
      }
    }
  }
  for (int bad : {-1, INT_MIN, 10, 11, INT_MAX})
    if (cache_page(bad, 10) != -1 || cache_slot(bad, 10) != -1) ++failures;
  for (int good : {0, 9})
    if (cache_page(good, 10) != good || cache_slot(good, 10) != good) ++failures;
  std::printf("%ld keys checked, %ld failures\n", checked, failures);
  return failures != 0;
}
