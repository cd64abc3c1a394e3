// cache_geom.h -- which keys of the paged cache a query sees, and how a row
// tile's keys are walked and split; shared by the kernels, the launch code and
// host checks.
//
// For one query at position i of a request with S tokens the mask of mask.h is
//   visible(j) = j < S and (j < pre  or  (lo <= j < hi and (i - j) % dil == 0)).
// A row tile holds queries at positions i0 .. i1 (times the query heads of one
// K/V head).  Its keys are walked in steps of 32 or 64: the prefix's steps, then
// those of the band that lie behind them.  The steps are split evenly enough: `parts`
// workgroups take `chunk` steps each, chunk being the launch's, or more where a
// request is longer than the launch was told.
#pragma once
#include "mask.h"

namespace chia {


// A table's page number, or -1 for one outside the cache: such a page is not read.
CHIA_HD int32_t cache_page(int32_t id, int32_t num_blocks) { return (uint32_t)id < (uint32_t)num_blocks ? id : -1; }

// A slot, or -1 for one outside the cache: such a token is not written.
CHIA_HD int32_t cache_slot(int32_t slot, int32_t num_slots) { return (uint32_t)slot < (uint32_t)num_slots ? slot : -1; }

struct CacheMask {
  int32_t causal, window, dil, blk, prefix;  // window, blk, prefix below 2^28; 0 = off
  UDiv div_blk, div_dil;
  uint32_t comb;  // bits 0, dil, 2 dil, ... below 32
};

CHIA_HD uint32_t cache_comb(int32_t dil) {
  uint32_t bits = 1;
  for (int32_t d = dil; d < 32; d += dil) bits |= 1u << d;
  return bits;
}

struct RowKeys {
  int32_t lo, hi, pre;  // lo <= j < hi (and the dilation), or j < pre
};

CHIA_HD RowKeys cache_row_keys(const CacheMask& m, int32_t i, int32_t S) {
  if (i < 0) return {0, 0, 0};
  int32_t lo = 0, hi = S;
  if (m.causal) hi = imin32(hi, i + 1);
  if (m.window > 0) {
    lo = imax32(lo, i - m.window + 1);
    if (!m.causal) hi = imin32(hi, i + m.window);
  }
  if (m.blk > 0) {
    const int32_t b = udiv(i, m.div_blk) * m.blk;
    lo = imax32(lo, b);
    hi = imin32(hi, b + m.blk);
  }
  return {lo, hi, imin32(m.prefix, S)};
}

// Bits below n, of 32.
CHIA_HD uint32_t bits_below(int32_t n) { return n <= 0 ? 0u : n >= 32 ? ~0u : (1u << n) - 1u; }

// Bit d: the row at position i sees key j0 + d (j0 >= 0).  The band and the prefix are
// ranges of bits, the dilation one comb of them, moved to the first key of i's class:
// one division for 32 keys.
CHIA_HD uint32_t cache_seen(const CacheMask& m, const RowKeys& k, int32_t i, int32_t j0) {
  uint32_t bits = bits_below(k.hi - j0) & ~bits_below(k.lo - j0);
  if (m.dil > 1) {
    const int32_t at = imax32(i, 0);  // (a row at i < 0 sees nothing)
    int32_t first = (at - udiv(at, m.div_dil) * m.dil) - (j0 - udiv(j0, m.div_dil) * m.dil);
    if (first < 0) first += m.dil;
    bits &= first < 32 ? m.comb << first : 0u;
  }
  return bits | bits_below(k.pre - j0);
}

// The walk of a row tile: step s covers the `step` keys from walk_key(s) on.
struct TileWalk {
  int32_t step;
  int32_t n_pre, first, n;          // prefix steps, first band step, steps in all
  int32_t full_lo, full_hi, full_pre;  // every row sees [full_lo, full_hi) and [0, full_pre) (dilation 1)
};

CHIA_HD TileWalk cache_tile_walk(const CacheMask& m, int32_t i0, int32_t i1, int32_t S, int32_t step) {
  // lo and hi never fall with the position: the first row reaches lowest, the last highest.
  const RowKeys a = cache_row_keys(m, imax32(i0, 0), S), b = cache_row_keys(m, i1, S);
  TileWalk w;
  w.step = step;  // a power of two known to the compiler where this is called
  const int32_t pre = b.pre;
  w.n_pre = (pre + step - 1) / step;
  w.first = imax32(w.n_pre, a.lo / step);
  w.n = w.n_pre + imax32(0, (b.hi + step - 1) / step - w.first);
  if (i1 < 0) w.n_pre = w.n = 0;
  w.full_lo = b.lo;
  w.full_hi = i0 < 0 || m.dil > 1 ? 0 : a.hi;
  w.full_pre = i0 < 0 ? 0 : pre;
  return w;
}

CHIA_HD int32_t walk_key(const TileWalk& w, int32_t s) {
  return w.step * (s < w.n_pre ? s : w.first + (s - w.n_pre));
}

// Whether every row of the tile sees all of keys c .. c + n - 1.
CHIA_HD bool walk_full(const TileWalk& w, int32_t c, int32_t n) {
  return (c >= w.full_lo && c + n <= w.full_hi) || c + n <= w.full_pre;
}

// Steps of each part, of at most `parts`.
CHIA_HD int32_t walk_chunk(int32_t steps, int32_t parts, int32_t chunk) {
  return imax32(chunk, (steps + parts - 1) / parts);
}

}  // namespace chia
