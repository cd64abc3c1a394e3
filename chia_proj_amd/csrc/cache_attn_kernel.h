// cache_attn_kernel.h -- attention of a few queries over the paged 8-bit cache (gfx950).
//
// Per row (query x head of a K/V head), over the keys j the mask shows it:
//   s_j = mod(ks[page] scale hs (q . k8_j)),  o = sum_j p_j vs[page] v8_j  (/ sum_j p_j for softmax)
// with k8, v8 the float8 codes and ks, vs their page's scales.
//
// A decoding step reads every cached code once for a handful of rows: it is
// bound by HBM.  So the codes go from memory straight into registers (no LDS,
// no barrier in the loop; every wavefront walks its own keys with the next
// step's loads in flight) and the rows of one K/V head share them:
//   S^T[key, row]  = K Q^T    v_mfma_f32_16x16x32_bf16, A = K: lane (m = l % 16,
//       g = l / 16) takes 16-byte pieces 64 c + 16 g of key m's row and uses them
//       as channels (the order of a contraction is free; Q is loaded in the same);
//   O^T[d, row]   += V^T P^T  A = V^T: the lane takes columns d = n D/16 + c
//       (n = l % 16, c = 0 .. D/16 - 1) of keys 4 g + {0 .. 3} and 16 + 4 g + {0 .. 3}
//       of the step, the very keys whose scores the first product left in this
//       lane, so P goes from accumulator to operand in place.  A byte
//       permutation of two keys' dwords pairs them for the conversion.
// float8 -> bf16 is exact (v_cvt_scalef32_pk_bf16_fp8 / bf8); V's conversion
// applies the power of two of its scale, the fraction of one that is no power of
// two goes to P.  K's scale joins the fp32 score.  P is rounded to bf16; the row
// sum adds the rounded weights.  The softmax maximum moves only when a score
// exceeds it by more than 8 (log2), which one vote per step finds out.
//
// Rows come in tiles of 16 NT; the NW wavefronts of a workgroup split a tile's keys
// and merge through LDS.  The keys are further split over workgroups
// (cache_geom.h), whose partial rows a second kernel joins.  Prompts, with many
// rows to a K/V head, have a kernel of their own (cache_prompt_kernel.h).
//
// 64 requests of 97 .. 8192 tokens, H32/8, D = 128 (469 MB): 103 us, 4.6 TB/s; two of 131072
// (489 MB, reads only): 92 us, 5.3 TB/s; one of 512, 8 heads, D = 64: 8.2 us, the chain length ->
// table -> scales and keys -> merge.
#pragma once
#include <hip/hip_runtime.h>

#include "cache_geom.h"

namespace chia {

typedef __bf16 cbf16x8_t __attribute__((ext_vector_type(8)));
typedef __bf16 cbf16x2_t __attribute__((ext_vector_type(2)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef uint32_t cu32x4_t __attribute__((ext_vector_type(4)));
typedef uint32_t cu32x2_t __attribute__((ext_vector_type(2)));

enum CacheScore : int { CACHE_SOFTMAX = 0, CACHE_SOFTMAX_MOD = 1, CACHE_SIGMOID = 2, CACHE_RELU = 3 };

struct CacheAttnParams {
  const uint16_t* q;
  uint16_t* o;
  const uint8_t *k, *v;
  const float *ks, *vs;
  int64_t q_st, q_sh, o_st, o_sh;
  int64_t k_sb, k_sh, k_st, v_sb, v_sh, v_st;
  int64_t ks_sb, ks_sh, vs_sb, vs_sh;
  const int32_t* table;
  int64_t table_stride;
  const int32_t *lens, *cu;
  const float *head_scale, *alibi;
  CacheMask mask;
  int32_t R, H, Hkv, G, T, width, num_blocks, bshift;
  int32_t tiles, parts, chunk;  // row tiles and key parts per (request, K/V head); steps per part
  int32_t units;                 // R Hkv tiles
  UDiv div_units, div_tiles, div_hkv, div_g;
  float scale, softcap, bias, post_scale;
  float* part_o;   // [parts, T H, D]
  float* part_ml;  // [parts, T H, 2]: running max (log2), row sum
};

constexpr float kCLog2e = 1.4426950408889634f;
constexpr float kCLazy = 8.0f;

// The kernel's arguments where they are used seldom (a page lookup, a masked step,
// the end): read again from the argument segment there, rather than held in scalar
// registers, and spilled, through the walk.
using ColdArgs = const __attribute__((address_space(4))) CacheAttnParams*;
__device__ __forceinline__ ColdArgs cold_args() {
  ColdArgs p = (ColdArgs)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(p));
  return p;
}

// What a workgroup computes for one (request, K/V head): the request's span.
struct CacheSpan {
  int32_t tok0, n, S;  // first query row, queries, tokens (clamped to what the buffers hold)
};

__device__ __forceinline__ CacheSpan cache_span(const CacheAttnParams& p, int r) {
  CacheSpan s;
  if (p.cu) {
    const int32_t a = imin32(imax32(p.cu[r], 0), p.T), b = imin32(imax32(p.cu[r + 1], 0), p.T);
    s.tok0 = a;
    s.n = imax32(b - a, 0);
  } else {
    s.tok0 = r;
    s.n = 1;
  }
  s.S = imin32(imax32(p.lens[r], 0), p.width << p.bshift);
  return s;
}

__device__ __forceinline__ UDiv cold_div(const __attribute__((address_space(4))) UDiv& d) { return {d.m, d.l}; }
__device__ __forceinline__ CacheMask cold_mask(ColdArgs a) {
  return {a->mask.causal, a->mask.window, a->mask.dil, a->mask.blk, a->mask.prefix, cold_div(a->mask.div_blk), cold_div(a->mask.div_dil),
          a->mask.comb};
}

// Positions of the queries of row tile rt (ROWS rows) and its walk.
template <int ROWS>
__device__ __forceinline__ TileWalk cache_walk_of(const CacheMask& m, UDiv div_g, const CacheSpan& s, int rt) {
  const int t0 = udiv(rt * ROWS, div_g), t1 = imin32(udiv(rt * ROWS + ROWS - 1, div_g), s.n - 1);
  const int32_t at = s.S - s.n;
  return cache_tile_walk(m, at + t0, at + t1, s.S, ROWS == 128 ? 64 : 32);
}

template <int FMT, bool HI>
__device__ __forceinline__ uint32_t cvt2(uint32_t w, float scale) {
  if constexpr (FMT == 0)
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, HI));
  else
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8(w, scale, HI));
}

// A nonzero bit for each byte of w that is an infinity or NaN.
template <int FMT>
__device__ __forceinline__ uint32_t nonfinite(uint32_t w) {
  if constexpr (FMT == 0) return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
  else return ((w & 0x7c7c7c7cu) + 0x04040404u) & 0x80808080u;
}

__device__ __forceinline__ uint32_t cpack(float a, float b) {
  cbf16x2_t r;
  r[0] = (__bf16)a;
  r[1] = (__bf16)b;
  return __builtin_bit_cast(uint32_t, r);
}

__device__ __forceinline__ float lo_f(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float hi_f(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }

// K or V codes of a 32-key step as loaded, and what belongs to its two 16-key
// halves (each inside one page).
template <int D>
struct CacheKeys {
  cu32x4_t w[2][D / 64];
  int32_t key;     // first key
  int32_t at[2];   // lane that holds the half's page
  bool ok[2];      // the page is inside the cache
};

template <int D>
struct CacheValues {
  uint32_t w[8][D / 64];
};

template <int D, int FMT, int SCORE, int NT, int NW>
__global__ __launch_bounds__(64 * NW, NT == 1 ? 3 : 2) void cache_attn_kernel(const CacheAttnParams p) {
  constexpr int KS = D / 32;            // k-steps of the first product
  constexpr int DC = D / 16;            // 16-row blocks of O^T; columns per lane of V
  constexpr int W64 = D / 64;
  constexpr int ROWS = 16 * NT;
  constexpr bool SOFTMAX = SCORE == CACHE_SOFTMAX || SCORE == CACHE_SOFTMAX_MOD;
  constexpr int LP = D + 4;             // LDS row pitch: rows start in other banks
  __shared__ __attribute__((aligned(16))) float lds[NW * ROWS * LP + NW * ROWS * 2];

  const int lane = threadIdx.x & 63, n16 = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // Parts in the slowest place: workgroups next to each other, which go to the XCDs
  // in turn, then are of different requests and heads.  (With parts next to each
  // other and 4 or 8 of them, some XCDs got only first parts and some only last
  // ones, which short requests do not have: 64 requests of 97 .. 8192 tokens in 4
  // parts, H32/8 D128, 137 us.)
  const int z = udiv((int)blockIdx.x, p.div_units), u = (int)blockIdx.x - z * p.units;
  const int rh = udiv(u, p.div_tiles), rt0 = u - rh * p.tiles;
  const int r = udiv(rh, p.div_hkv), hk = rh - r * p.Hkv;
  const int bs_mask = (1 << p.bshift) - 1;
  const int32_t* table = p.table + (int64_t)r * p.table_stride;
  // The chain lengths -> table -> scales, keys is what a short request waits for.
  // Without a window the first pages follow from the launch alone, so they are
  // asked for before the length is there (a wrong guess is only asked again).
  int32_t pg0 = 1 << 30, pg_id = -1;
  float pg_ks = 0.f, pg_vs = 0.f;
  if (p.mask.window == 0 && p.mask.blk == 0) {
    int first = z * p.chunk;
    if (((p.chunk * 32) >> p.bshift) > 63) first += wave * ((p.chunk + NW - 1) / NW);
    pg0 = (first * 32) >> p.bshift;
    const int at = pg0 + lane;
    pg_id = at < p.width ? cache_page(table[at], p.num_blocks) : -1;
    const int64_t id = imax32(pg_id, 0);
    pg_ks = p.ks[id * p.ks_sb + hk * p.ks_sh];
    pg_vs = p.vs[id * p.vs_sb + hk * p.vs_sh];
  }
  const CacheSpan sp = cache_span(p, r);
  const int n_rows = sp.n * p.G;

  for (int rt = rt0; rt * ROWS < n_rows; rt += p.tiles) {
    const ColdArgs ta = cold_args();
    const CacheMask mask = cold_mask(ta);
    const UDiv div_g = cold_div(ta->div_g);
    const TileWalk tw = cache_walk_of<ROWS>(mask, div_g, sp, rt);
    const int chunk = walk_chunk(tw.n, ta->parts, ta->chunk);
    const int used = (tw.n + chunk - 1) / chunk;  // parts that have steps
    if (z > 0 && z >= used) continue;             // part 0 writes the rows that see nothing
    int s0 = z * chunk, s1 = imin32(s0 + chunk, tw.n);
    const int row0 = rt * ROWS, per = (s1 - s0 + NW - 1) / NW;
    s0 = imin32(s0 + wave * per, s1);
    s1 = imin32(s0 + per, s1);

    // this lane's rows (one per 16-row block): keys, score constants, Q
    RowKeys rk[NT];
    int32_t ipos[NT];
    float c1[NT], sl[NT];
    cbf16x8_t qf[NT][KS];
    int32_t otok[NT], ohead[NT];
    bool rok[NT];
#pragma unroll
    for (int b = 0; b < NT; ++b) {
      const int row = row0 + 16 * b + n16;
      rok[b] = row < n_rows;
      const int t = rok[b] ? udiv(row, div_g) : 0, h = hk * ta->G + (rok[b] ? row - t * ta->G : 0);
      ipos[b] = sp.S - sp.n + t;
      rk[b] = rok[b] ? cache_row_keys(mask, ipos[b], sp.S) : RowKeys{0, 0, 0};
      c1[b] = ta->scale * (ta->head_scale ? ta->head_scale[h] : 1.f);
      sl[b] = ta->alibi ? ta->alibi[h] : 0.f;
      if constexpr (SCORE == CACHE_SOFTMAX) c1[b] *= kCLog2e;
      const uint16_t* qp = ta->q + (int64_t)(sp.tok0 + t) * ta->q_st + (int64_t)h * ta->q_sh;
      otok[b] = sp.tok0 + t;
      ohead[b] = h;
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        const cu32x4_t w = *(const cu32x4_t*)(qp + 64 * (s >> 1) + 16 * g + 8 * (s & 1));
        qf[b][s] = __builtin_bit_cast(cbf16x8_t, rok[b] ? w : cu32x4_t{0, 0, 0, 0});
      }
    }

    f32x4_t acc[NT][DC];
    float m_run[NT], l_run[NT];
#pragma unroll
    for (int b = 0; b < NT; ++b) {
      m_run[b] = -INFINITY;
      l_run[b] = 0.f;
#pragma unroll
      for (int c = 0; c < DC; ++c) acc[b][c] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    }

    // Page numbers and scales of 64 pages from pg0 on, one per lane; a step's two
    // halves are always among them.
    auto pages_from = [&](int pg) __attribute__((always_inline)) {
      const ColdArgs a = cold_args();
      pg0 = pg;
      const int at = pg + lane;
      pg_id = at < a->width ? cache_page(a->table[(int64_t)r * a->table_stride + at], a->num_blocks) : -1;
      const int64_t id = imax32(pg_id, 0);
      pg_ks = a->ks[id * a->ks_sb + hk * a->ks_sh];
      pg_vs = a->vs[id * a->vs_sb + hk * a->vs_sh];
    };
    const uint32_t k_off = (uint32_t)(n16 * (int32_t)p.k_st + 16 * g);
    const uint32_t v_off = (uint32_t)(4 * g * (int32_t)p.v_st + n16 * DC);
    auto pages_of = [&](int key) __attribute__((always_inline)) {
      const int pg = key >> p.bshift, last = (key + 16) >> p.bshift;
      if (pg < pg0 || last - pg0 > 63) pages_from(pg);
    };
    CacheKeys<D> kk;
    CacheValues<D> vv;
    auto issue_k = [&](int s) __attribute__((always_inline)) {
      kk.key = walk_key(tw, s);
      pages_of(kk.key);
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const int j = kk.key + 16 * t, at = (j >> p.bshift) - pg0;
        const int id = __builtin_amdgcn_readlane(pg_id, at);
        kk.at[t] = at;
        kk.ok[t] = id >= 0;
        const uint8_t* kp = p.k + (int64_t)imax32(id, 0) * p.k_sb + hk * p.k_sh + (int64_t)(j & bs_mask) * p.k_st;
#pragma unroll
        for (int c = 0; c < W64; ++c) kk.w[t][c] = *(const cu32x4_t*)(kp + k_off + 64 * c);
      }
    };
    auto issue_v = [&](int s) __attribute__((always_inline)) {  // after issue_k of the same step
      const int key = walk_key(tw, s);
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const int j = key + 16 * t, at = (j >> p.bshift) - pg0;
        const int id = __builtin_amdgcn_readlane(pg_id, at);
        const uint8_t* vp = p.v + (int64_t)imax32(id, 0) * p.v_sb + hk * p.v_sh + (int64_t)(j & bs_mask) * p.v_st;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint8_t* a = vp + v_off + (uint32_t)(e * (int32_t)p.v_st);
          if constexpr (W64 == 2) {
            const cu32x2_t w = *(const cu32x2_t*)a;
            vv.w[4 * t + e][0] = w[0];
            vv.w[4 * t + e][1] = w[1];
          } else {
            vv.w[4 * t + e][0] = *(const uint32_t*)a;
          }
        }
      }
    };

    // 0 x NaN: a code that is no number must not meet the zero weight of a row that
    // does not see its key.  Such codes are taken out of V, and what they do to the
    // rows that see them is added first: NaN where a row sees a NaN (a product of
    // 1 at those codes with 1 at the keys that it sees), and an infinity of e5m2,
    // as 2^120, by the row's weights, grown until it is one.
    auto clean = [&](const uint32_t (&vis)[NT], const uint32_t (&pw)[NT][4], const float (&vs)[2], float (&v2)[2]) __attribute__((always_inline)) {
      uint32_t bad = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e)
#pragma unroll
        for (int w = 0; w < W64; ++w) bad |= nonfinite<FMT>(vv.w[e][w]);
      const bool bs2[2] = {!(fabsf(vs[0]) < INFINITY), !(fabsf(vs[1]) < INFINITY)};
      if (!__any(bad != 0) && !bs2[0] && !bs2[1]) return;
      cbf16x8_t sees[NT];
#pragma unroll
      for (int b = 0; b < NT; ++b) {
        cu32x4_t w;
#pragma unroll
        for (int i = 0; i < 4; ++i)
          w[i] = ((vis[b] >> (2 * i)) & 1 ? 0x3f80u : 0u) | ((vis[b] >> (2 * i + 1)) & 1 ? 0x3f800000u : 0u);
        sees[b] = __builtin_bit_cast(cbf16x8_t, w);
      }
#pragma unroll
      for (int w = 0; w < W64; ++w)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          cu32x4_t nan_w, inf_w;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            nan_w[e] = inf_w[e] = 0;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const uint32_t x = (vv.w[2 * e + i][w] >> (8 * c)) & 0xffu, m = x & 0x7fu;
              const bool nan = bs2[e >> 1] || (FMT == 0 ? m == 0x7fu : m > 0x7cu);
              nan_w[e] |= (nan ? 0x3f80u : 0u) << (16 * i);
              if (FMT == 1 && m == 0x7cu) inf_w[e] |= (0x7b80u | (x & 0x80u) << 8) << (16 * i);
            }
          }
#pragma unroll
          for (int b = 0; b < NT; ++b) {
            f32x4_t& a = acc[b][4 * w + c];
            const f32x4_t zero = {0.f, 0.f, 0.f, 0.f};
            const f32x4_t k = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(cbf16x8_t, nan_w), sees[b], zero, 0, 0, 0);
#pragma unroll
            for (int e = 0; e < 4; ++e) a[e] = k[e] > 0.f ? NAN : a[e];
            if constexpr (FMT == 1) {
              const cbf16x8_t pf = __builtin_bit_cast(cbf16x8_t, cu32x4_t{pw[b][0], pw[b][1], pw[b][2], pw[b][3]});
              const f32x4_t y = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(cbf16x8_t, inf_w), pf, zero, 0, 0, 0);
#pragma unroll
              for (int e = 0; e < 4; ++e) a[e] += y[e] * 0x1p127f * 0x1p127f;
            }
          }
          __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
      for (int t = 0; t < 2; ++t)
        if (bs2[t]) v2[t] = 1.f;
#pragma unroll
      for (int e = 0; e < 8; ++e)
#pragma unroll
        for (int w = 0; w < W64; ++w) {
          const uint32_t t = nonfinite<FMT>(vv.w[e][w]);
          vv.w[e][w] &= ~((t >> 7) * 0xffu);
        }
    };

    // One step: its scores from K (whose registers then take the next step's),
    // weights, and the second product from V.
    auto compute = [&](int s) __attribute__((always_inline)) {
      f32x4_t sc[NT][2];  // lane: row n16 of each block, keys key + 16 t + 4 g + e
      const int key = kk.key;
      float ks[2], vs[2];  // before the next step's pages take their place
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        ks[t] = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(pg_ks), kk.at[t]));
        vs[t] = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(pg_vs), kk.at[t]));
      }
      const bool pok[2] = {kk.ok[0], kk.ok[1]};
#pragma unroll
      for (int t = 0; t < 2; ++t) {
#pragma unroll
        for (int b = 0; b < NT; ++b) sc[b][t] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < KS; ++i) {
          const uint32_t w0 = kk.w[t][i >> 1][2 * (i & 1)], w1 = kk.w[t][i >> 1][2 * (i & 1) + 1];
          const cbf16x8_t kf = __builtin_bit_cast(cbf16x8_t, cu32x4_t{cvt2<FMT, false>(w0, 1.f), cvt2<FMT, true>(w0, 1.f),
                                                                     cvt2<FMT, false>(w1, 1.f), cvt2<FMT, true>(w1, 1.f)});
#pragma unroll
          for (int b = 0; b < NT; ++b) sc[b][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf, qf[b][i], sc[b][t], 0, 0, 0);
        }
      }
      if (s + 1 < s1) issue_k(s + 1);
      const bool full = walk_full(tw, key, 32) && pok[0] && pok[1];
            // vs = 2^e mant: the power goes to V's conversion, mant (1 for a power of two) to P
      float v2[2], mant[2], inv[2];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const uint32_t bits = __float_as_uint(vs[t]);
        v2[t] = __uint_as_float(bits & 0x7f800000u);
        mant[t] = __uint_as_float((bits & 0x807fffffu) | 0x3f800000u);
      }
      const bool frac = mant[0] != 1.f || mant[1] != 1.f;
      inv[0] = inv[1] = 1.f;
      if (frac) {
        inv[0] = 1.f / mant[0];
        inv[1] = 1.f / mant[1];
      }
      uint32_t vis[NT];  // bit 4 t + e: the row sees the key
      uint32_t pw[NT][4];
#pragma unroll
      for (int b = 0; b < NT; ++b) {
        vis[b] = 0xffu;
        if (!full) {
          const uint32_t bits = cache_seen(cold_mask(cold_args()), rk[b], ipos[b], key) &
                                ((pok[0] ? 0xffffu : 0u) | (pok[1] ? 0xffff0000u : 0u));
          vis[b] = ((bits >> (4 * g)) & 0xfu) | ((bits >> (4 * g + 12)) & 0xf0u);
        }
        float x[2][4];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const float ck = c1[b] * ks[t];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float v = sc[b][t][e] * ck;
            if constexpr (SCORE != CACHE_SOFTMAX) {
              v = __builtin_fmaf(sl[b], (float)(key + 16 * t + 4 * g + e - ipos[b]), v);
              if (p.softcap > 0.f) {  // cap tanh(v / cap) = cap (1 - 2 / (1 + 2^(2 v log2e / cap)))
                const float ex = __builtin_amdgcn_exp2f(v * (2.f * kCLog2e / p.softcap));
                v = p.softcap * (1.f - 2.f * __builtin_amdgcn_rcpf(1.f + ex));
              }
              if constexpr (SCORE == CACHE_SOFTMAX_MOD) v *= kCLog2e;
            }
            x[t][e] = v;
          }
        }
        if constexpr (SOFTMAX) {
          if (!full)
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
              for (int e = 0; e < 4; ++e) x[t][e] = (vis[b] >> (4 * t + e)) & 1 ? x[t][e] : -INFINITY;
          float mx = fmaxf(fmaxf(fmaxf(x[0][0], x[0][1]), fmaxf(x[0][2], x[0][3])),
                           fmaxf(fmaxf(x[1][0], x[1][1]), fmaxf(x[1][2], x[1][3])));
          if (__any(mx > m_run[b] + kCLazy)) {
            mx = fmaxf(mx, __shfl_xor(mx, 16));
            mx = fmaxf(mx, __shfl_xor(mx, 32));
            mx = fmaxf(mx, m_run[b]);
            const float f = m_run[b] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m_run[b] - mx);
            l_run[b] *= f;
#pragma unroll
            for (int c = 0; c < DC; ++c) acc[b][c] *= f;
            m_run[b] = mx;
          }
          const float mr = m_run[b] == -INFINITY ? 0.f : m_run[b];
#pragma unroll
          for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) x[t][e] = __builtin_amdgcn_exp2f(x[t][e] - mr);
        } else {
#pragma unroll
          for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              float v = x[t][e];
              if constexpr (SCORE == CACHE_SIGMOID)
                v = __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-kCLog2e * (v + p.bias)));
              else
                v = v < 0.f ? 0.f : v;
              x[t][e] = full || ((vis[b] >> (4 * t + e)) & 1) ? v : 0.f;
            }
        }
        if (frac)
#pragma unroll
          for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) x[t][e] = (vis[b] >> (4 * t + e)) & 1 ? x[t][e] * mant[t] : 0.f;
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int e = 0; e < 2; ++e) pw[b][2 * t + e] = cpack(x[t][2 * e], x[t][2 * e + 1]);
        if constexpr (SOFTMAX)
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            const float add = (lo_f(pw[b][2 * t]) + hi_f(pw[b][2 * t])) + (lo_f(pw[b][2 * t + 1]) + hi_f(pw[b][2 * t + 1]));
            l_run[b] = __builtin_fmaf(add, inv[t], l_run[b]);
          }
      }
      if (!full) clean(vis, pw, vs, v2);
#pragma unroll
      for (int w = 0; w < W64; ++w) {
        cu32x4_t va[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {  // keys 2 e, 2 e + 1 of the lane's eight
          const uint32_t x = vv.w[2 * e][w], y = vv.w[2 * e + 1][w];
          const uint32_t lo = __builtin_amdgcn_perm(y, x, 0x05010400u), hi = __builtin_amdgcn_perm(y, x, 0x07030602u);
          const float f = v2[e >> 1];
          va[0][e] = cvt2<FMT, false>(lo, f);
          va[1][e] = cvt2<FMT, true>(lo, f);
          va[2][e] = cvt2<FMT, false>(hi, f);
          va[3][e] = cvt2<FMT, true>(hi, f);
        }
#pragma unroll
        for (int b = 0; b < NT; ++b) {
          const cbf16x8_t pf = __builtin_bit_cast(cbf16x8_t, cu32x4_t{pw[b][0], pw[b][1], pw[b][2], pw[b][3]});
#pragma unroll
          for (int c = 0; c < 4; ++c)
            acc[b][4 * w + c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(cbf16x8_t, va[c]), pf, acc[b][4 * w + c], 0, 0, 0);
        }
      }
      if (s + 1 < s1) issue_v(s + 1);
    };

    if (s0 < s1) {
      issue_k(s0);
      issue_v(s0);
      for (int s = s0; s < s1; ++s) compute(s);
    }

    // row sums over the four lanes of a row
    if constexpr (SOFTMAX)
#pragma unroll
      for (int b = 0; b < NT; ++b) {
        l_run[b] += __shfl_xor(l_run[b], 16);
        l_run[b] += __shfl_xor(l_run[b], 32);
      }

    const ColdArgs ca = cold_args();
    const bool whole = used <= 1;  // this workgroup has all the keys of its rows
    // merge the wavefronts' keys
    float* ml = lds + NW * ROWS * LP;  // [NW][ROWS][2]
    if constexpr (SOFTMAX) {
      if (g == 0)
#pragma unroll
        for (int b = 0; b < NT; ++b) {
          ml[(wave * ROWS + 16 * b + n16) * 2] = m_run[b];
          ml[(wave * ROWS + 16 * b + n16) * 2 + 1] = l_run[b];
        }
    }
    __syncthreads();
    float m_all[NT], l_all[NT];
#pragma unroll
    for (int b = 0; b < NT; ++b) {
      m_all[b] = -INFINITY;
      l_all[b] = 0.f;
      if constexpr (SOFTMAX) {
        float mw[NW], lw[NW];
#pragma unroll
        for (int w = 0; w < NW; ++w) {
          mw[w] = ml[(w * ROWS + 16 * b + n16) * 2];
          lw[w] = ml[(w * ROWS + 16 * b + n16) * 2 + 1];
          m_all[b] = fmaxf(m_all[b], mw[w]);
        }
#pragma unroll
        for (int w = 0; w < NW; ++w)
          l_all[b] += mw[w] == -INFINITY ? 0.f : lw[w] * __builtin_amdgcn_exp2f(mw[w] - m_all[b]);
        const float f = m_run[b] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m_run[b] - m_all[b]);
#pragma unroll
        for (int c = 0; c < DC; ++c) acc[b][c] *= f;
      }
      // [wave][row][d], the pieces of a lane 16 bytes each
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int c = 0; c < DC; c += 4)
          *(f32x4_t*)(lds + (wave * ROWS + 16 * b + n16) * LP + DC * (4 * g + e) + c) =
              f32x4_t{acc[b][c][e], acc[b][c + 1][e], acc[b][c + 2][e], acc[b][c + 3][e]};
    }
    __syncthreads();
    // wavefront w < 4 stores the pieces e = w of every lane's rows
#pragma unroll
    for (int b = 0; b < NT; ++b) {
      f32x4_t sum[DC / 4];
#pragma unroll
      for (int c = 0; c < DC / 4; ++c) {
        sum[c] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < NW; ++w)
          sum[c] += *(const f32x4_t*)(lds + (w * ROWS + 16 * b + n16) * LP + DC * (4 * g + wave) + 4 * c);
      }
      if (!rok[b] || wave >= 4) continue;
      const int at = DC * (4 * g + wave);
      if (whole) {
        const float f = SOFTMAX ? (l_all[b] != 0.f ? 1.f / l_all[b] : 0.f) : ca->post_scale;
        uint16_t* op = ca->o + (int64_t)otok[b] * ca->o_st + (int64_t)ohead[b] * ca->o_sh + at;
        if constexpr (DC == 8)
          *(cu32x4_t*)op = cu32x4_t{cpack(sum[0][0] * f, sum[0][1] * f), cpack(sum[0][2] * f, sum[0][3] * f),
                                    cpack(sum[1][0] * f, sum[1][1] * f), cpack(sum[1][2] * f, sum[1][3] * f)};
        else
          *(cu32x2_t*)op = cu32x2_t{cpack(sum[0][0] * f, sum[0][1] * f), cpack(sum[0][2] * f, sum[0][3] * f)};
      } else {
        const int64_t row = ((int64_t)z * ca->T + otok[b]) * ca->H + ohead[b];
#pragma unroll
        for (int c = 0; c < DC / 4; ++c) *(f32x4_t*)(ca->part_o + row * D + at + 4 * c) = sum[c];
        if (SOFTMAX && g == 0 && wave == 0) {
          ca->part_ml[2 * row] = m_all[b];
          ca->part_ml[2 * row + 1] = l_all[b];
        }
      }
    }
    __syncthreads();  // the next tile writes the same LDS
  }
}

using CacheAttnFn = void (*)(CacheAttnParams);

// The row tiles: 16 or 32 rows whose keys the wavefronts split (this file), 128 rows (cache_prompt_kernel.h).
enum CacheTile : int { CACHE_ROWS16 = 0, CACHE_ROWS32 = 1, CACHE_ROWS128 = 2 };
constexpr int kCacheRows[3] = {16, 32, 128}, kCacheStep[3] = {32, 32, 64};

CacheAttnFn select_cache_kernel_d64(int format, int score, int tile, int waves);
CacheAttnFn select_cache_kernel_d128(int format, int score, int tile, int waves);
CacheAttnFn select_cache_prompt_kernel(int head_dim, int format, int score);

template <int D>
CacheAttnFn pick_cache_kernel(int format, int score, int tile, int waves) {
#define CHIA_CACHE(F, S)                                                                          \
  if (format == F && score == S)                                                                  \
    return tile == CACHE_ROWS32 ? cache_attn_kernel<D, F, S, 2, 4>                                \
           : waves == 8         ? cache_attn_kernel<D, F, S, 1, 8> : cache_attn_kernel<D, F, S, 1, 4>;
#define CHIA_CACHE_FMT(F) \
  CHIA_CACHE(F, CACHE_SOFTMAX) CHIA_CACHE(F, CACHE_SOFTMAX_MOD) CHIA_CACHE(F, CACHE_SIGMOID) CHIA_CACHE(F, CACHE_RELU)
  CHIA_CACHE_FMT(0)
  CHIA_CACHE_FMT(1)
#undef CHIA_CACHE_FMT
#undef CHIA_CACHE
  return nullptr;
}

}  // namespace chia
