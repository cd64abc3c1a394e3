// cache_prompt_kernel.h -- attention of many queries over the paged 8-bit cache (gfx950).
//
// The function of cache_attn_kernel.h for prompts and chunks of them: with a
// hundred rows and more to a K/V head the matrix products bind, not the codes'
// bytes, so a workgroup converts each 64-key tile of K and V to bf16 once, in
// LDS, for its 128 rows.
//   S^T[key, row] = K Q^T, O^T[d, row] += V^T P^T on v_mfma_f32_32x32x16_bf16 with
//   the operand layouts and LDS swizzle of the one-block forward core
//   (attn_fwd_q1_kernel.h): a lane has one row and 16 keys of a 32-key block.
// A thread loads 16 codes of one key per 256 chunks of the tile, one tile ahead of
// the one computed, and stores them as 32 bytes of bf16 behind the current tile's
// work (two LDS stages, one barrier per tile).  The power of two of a key's scale
// is applied by the conversion; the fraction of a scale that is no power of two,
// which a branch finds out, multiplies the scores (K) or the weights (V).
//
// Two prompts' chunks of 1000 tokens over 9001 .. 16000, H32/8, D = 128 (408 GFLOP): 553 to 559 us,
// 735 TFLOP/s, matrix cores busy 30 % of the time and vector units 44 %: the chain products ->
// maximum -> exponentials -> products of a step at two wavefronts per SIMD.  A 64-row
// form (half the keys to each of two wavefronts) was not faster per row: a step takes
// as long.
#pragma once
#include "attn_fwd_kernel.h"
#include "cache_attn_kernel.h"

namespace chia {

template <int FMT>
__device__ __forceinline__ cu32x4_t cvt8(uint32_t lo, uint32_t hi, float scale) {
  return cu32x4_t{cvt2<FMT, false>(lo, scale), cvt2<FMT, true>(lo, scale), cvt2<FMT, false>(hi, scale), cvt2<FMT, true>(hi, scale)};
}

__device__ __forceinline__ float pow2_of(float s) { return __uint_as_float(__float_as_uint(s) & 0x7f800000u); }
__device__ __forceinline__ float fraction_of(float s) { return __uint_as_float((__float_as_uint(s) & 0x807fffffu) | 0x3f800000u); }

// One of two values (by value: chosen by reference they would have to lie in memory).
template <class T>
__device__ __forceinline__ T sel(int second, T a, T b) {
  return second ? b : a;
}

// x, hidden from the compiler: what is made from it stays where it is used
// rather than in registers through the walk.
template <class T>
__device__ __forceinline__ T here(T x) {
  asm volatile("" : "+v"(x));
  return x;
}

template <int D, int FMT, int SCORE>
__global__ __launch_bounds__(256, 2) void cache_prompt_kernel(const CacheAttnParams p) {
  constexpr int BN = 64, ROWS = 128;
  constexpr int DK = D / 16, DB = D / 32;
  constexpr int RP = 2 * D;                      // LDS row pitch (bytes)
  constexpr int K_BYTES = BN * RP, STAGE = 2 * K_BYTES;
  constexpr int CH = D / 16;                     // 16-code chunks per key
  constexpr int NL = BN * CH / 256;              // chunks per thread (of K, and of V)
  constexpr bool SOFTMAX = SCORE == CACHE_SOFTMAX || SCORE == CACHE_SOFTMAX_MOD;
  typedef short i16x8_t __attribute__((ext_vector_type(8)));
  __shared__ __attribute__((aligned(1024))) char lds[2 * STAGE];
  __shared__ int poison_s;                       // some tile's V had codes that are no numbers

  const int tid = threadIdx.x, lane = tid & 63, lq = lane & 31, lh = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  // parts in the slowest place, row tiles in the fastest (cache_attn_kernel.h says why; with each
  // K/V head's tiles on one XCD, whose L2 would hold its keys, a chunk of two prompts took a third longer)
  const int L = (int)blockIdx.x;
  const int z = udiv(L, p.div_units), u = L - z * p.units;
  const int rh = udiv(u, p.div_tiles), rt0 = u - rh * p.tiles;
  const int r = udiv(rh, p.div_hkv), hk = rh - r * p.Hkv;
  const CacheSpan sp = cache_span(p, r);
  const int n_rows = sp.n * p.G;
  const int bs_mask = (1 << p.bshift) - 1;
  const uint8_t* kbase = p.k + hk * p.k_sh;
  const uint8_t* vbase = p.v + hk * p.v_sh;

  // This lane's key among the 8 (D = 128) or 16 that its wavefront loads together, its
  // 16 codes of it, and its offset from the first.  Four lanes take 64 bytes of a key, the
  // next four those of the key whose swizzle differs in the lowest bit: a lane's codes
  // become an even and an odd 16-byte piece, and eight lanes' even pieces then lie in
  // eight different slots.
  const int q = lane >> 2, in_row = D == 128 ? (q >> 2) | ((q & 1) << 2) : (q >> 1) | ((q & 1) << 3);
  const int in_c = D == 128 ? (lane & 3) | ((q & 2) << 1) : lane & 3;
  const uint32_t k_off = (uint32_t)(in_row * (int32_t)p.k_st + 16 * in_c);
  const uint32_t v_off = (uint32_t)(in_row * (int32_t)p.v_st + 16 * in_c);
  // LDS byte offsets of this lane: K rows (A operand), V transposed reads
  const int k_lane = lq * RP + 16 * k_slot<D>(lq, lh);
  const int g16 = lane >> 4, s16 = lane & 15;
  const int v_row = 4 * (g16 >> 1) + (s16 >> 2);
  const int v_lane = K_BYTES + v_row * RP + 16 * k_slot<D>(v_row, 2 * (g16 & 1) + ((s16 & 3) >> 1)) + 8 * (s16 & 1);

  constexpr int SW8 = D == 128 ? 32 : 16;  // 16 row_swz(8): rows 8 further on flip this bit of the slot

  for (int rt = rt0; rt * ROWS < n_rows; rt += p.tiles) {
    const ColdArgs ta = cold_args();
    const CacheMask mask = cold_mask(ta);
    const UDiv div_g = cold_div(ta->div_g);
    const TileWalk tw = cache_walk_of<ROWS>(mask, div_g, sp, rt);
    const int chunk = walk_chunk(tw.n, ta->parts, ta->chunk);
    const int used = (tw.n + chunk - 1) / chunk;
    if (z > 0 && z >= used) continue;  // part 0 writes the rows that see nothing
    const int s0 = z * chunk, s1 = imin32(s0 + chunk, tw.n);

    const int row = rt * ROWS + 32 * wave + lq;
    const bool rok = row < n_rows;
    const int t = rok ? udiv(row, div_g) : 0, h = hk * ta->G + (rok ? row - t * ta->G : 0);
    const int ipos = sp.S - sp.n + t;
    const RowKeys rk = rok ? cache_row_keys(mask, ipos, sp.S) : RowKeys{0, 0, 0};
    float c1 = ta->scale * (ta->head_scale ? ta->head_scale[h] : 1.f);
    const float sl = ta->alibi ? ta->alibi[h] : 0.f;
    if constexpr (SCORE == CACHE_SOFTMAX) c1 *= kCLog2e;
    bf16x8_t qf[DK];
    {
      const uint16_t* qp = ta->q + (int64_t)(sp.tok0 + t) * ta->q_st + (int64_t)h * ta->q_sh + 8 * here(lh);
#pragma unroll
      for (int kk = 0; kk < DK; ++kk) {
        const u32x4_t w = *(const u32x4_t*)(qp + 16 * kk);
        qf[kk] = __builtin_bit_cast(bf16x8_t, rok ? w : u32x4_t{0, 0, 0, 0});
      }
    }

    // pages: numbers and scales of 64 from pg0 on, one per lane (every wavefront its own)
    int32_t pg0 = 1 << 30, pg_id = -1;
    float pg_ks = 0.f, pg_vs = 0.f;
    auto pages_of = [&](int key) __attribute__((always_inline)) {
      const int pg = key >> p.bshift, last = (key + BN - 16) >> p.bshift;
      if (pg >= pg0 && last - pg0 <= 63) return;
      const ColdArgs a = cold_args();
      pg0 = pg;
      const int at = pg + here(lane);
      pg_id = at < a->width ? cache_page(a->table[(int64_t)r * a->table_stride + at], a->num_blocks) : -1;
      const int64_t id = imax32(pg_id, 0);
      pg_ks = a->ks[id * a->ks_sb + hk * a->ks_sh];
      pg_vs = a->vs[id * a->vs_sb + hk * a->vs_sh];
    };
    // what belongs to the four 16-key groups of a tile: of the one in the
    // registers (next) and of the one in LDS that is computed (cur)
    struct Groups {
      int key;
      float ks[4], vs[4];
      bool full;  // every row of the workgroup's tile sees every key, every page is there
      bool frac;  // some scale is no power of two
      bool ok[4];
    };
    Groups next, cur;
    cu32x4_t kr[NL], vr[NL];
    auto load = [&](int s) __attribute__((always_inline)) {
      next.key = walk_key(tw, s);
      pages_of(next.key);
#pragma unroll
      for (int n = 0; n < NL; ++n) {
        // chunk c of the tile: key c / CH; the 64 lanes of a wavefront stay inside one group of 16 keys
        const int c0 = n * 256 + wave * 64, grp = c0 / CH / 16;
        const int key = next.key + 16 * grp, id = __builtin_amdgcn_readlane(pg_id, (key >> p.bshift) - pg0);
        const int64_t page = imax32(id, 0), place = (key & bs_mask) + (c0 / CH) % 16;
        kr[n] = *(const cu32x4_t*)(kbase + page * p.k_sb + place * p.k_st + k_off);
        vr[n] = *(const cu32x4_t*)(vbase + page * p.v_sb + place * p.v_st + v_off);
      }
    };
    auto scales = [&]() __attribute__((always_inline)) {  // of the tile that load() has asked for
      next.full = walk_full(tw, next.key, BN);
      if (p.bshift >= 6) {  // one page
        const int at = (next.key >> p.bshift) - pg0;
        const bool ok = __builtin_amdgcn_readlane(pg_id, at) >= 0;
        const float ks = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(pg_ks), at));
        const float vs = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(pg_vs), at));
#pragma unroll
        for (int q = 0; q < 4; ++q) next.ok[q] = ok, next.ks[q] = ks, next.vs[q] = vs;
        next.full = next.full && ok;
        next.frac = fraction_of(ks) != 1.f || fraction_of(vs) != 1.f;
        return;
      }
      next.frac = false;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int at = ((next.key + 16 * q) >> p.bshift) - pg0;
        next.ok[q] = __builtin_amdgcn_readlane(pg_id, at) >= 0;
        next.ks[q] = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(pg_ks), at));
        next.vs[q] = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(pg_vs), at));
        next.full = next.full && next.ok[q];
        next.frac = next.frac || fraction_of(next.ks[q]) != 1.f || fraction_of(next.vs[q]) != 1.f;
      }
    };
    // The tile in the registers to LDS.  Where not every row sees every key, values
    // that are no numbers are left out (0 x NaN must not reach the rows that do not
    // see them) and noted; RAW, after the walk, stores them as they are.
    auto store = [&](int stage, auto raw) __attribute__((always_inline)) {
      constexpr bool RAW = decltype(raw)::value;
      char* st = lds + stage * STAGE;
      bool bad = false;
#pragma unroll
      for (int n = 0; n < NL; ++n) {
        const int c0 = n * 256 + wave * 64, grp = c0 / CH / 16;
        const int row = (c0 / CH) + in_row, c = in_c;
        const float ks = pow2_of(sel(grp >> 1, sel(grp & 1, next.ks[0], next.ks[1]), sel(grp & 1, next.ks[2], next.ks[3])));
        const float vs = pow2_of(sel(grp >> 1, sel(grp & 1, next.vs[0], next.vs[1]), sel(grp & 1, next.vs[2], next.vs[3])));
        cu32x4_t vw = vr[n];
        if (!next.full) {
          const bool there = next.key + row < sp.S && sel(grp >> 1, sel(grp & 1, next.ok[0], next.ok[1]), sel(grp & 1, next.ok[2], next.ok[3]));
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t x = there ? vr[n][i] : 0u, odd = vs < INFINITY ? nonfinite<FMT>(x) : 0x80808080u;
            if constexpr (RAW) {
              vw[i] = vs < INFINITY || !there ? x : 0x7f7f7f7fu;
            } else {
              vw[i] = x & ~((odd >> 7) * 0xffu);
              bad = bad || (there && odd != 0);
            }
          }
        }
        const float f = RAW || !(next.full || vs < INFINITY) ? 1.f : vs;  // 0 times such a scale is no 0
        char* at = st + row * RP;
        const int slot0 = 16 * k_slot<D>(row, 2 * c), slot1 = 16 * k_slot<D>(row, 2 * c + 1);
        if constexpr (!RAW) {
          *(cu32x4_t*)(at + slot0) = cvt8<FMT>(kr[n][0], kr[n][1], ks);
          *(cu32x4_t*)(at + slot1) = cvt8<FMT>(kr[n][2], kr[n][3], ks);
        }
        *(cu32x4_t*)(at + K_BYTES + slot0) = cvt8<FMT>(vw[0], vw[1], f);
        *(cu32x4_t*)(at + K_BYTES + slot1) = cvt8<FMT>(vw[2], vw[3], f);
      }
      if (!RAW && !next.full && bad) poison_s = 1;
    };
    // bit e: the row sees key jb + 4 lh + 8 (e / 4) + e % 4
    auto seen = [&](int jb, bool ok0, bool ok1) __attribute__((always_inline)) {
      const uint32_t bits = (cache_seen(cold_mask(cold_args()), rk, here(ipos), jb) &
                             ((ok0 ? 0xffffu : 0u) | (ok1 ? 0xffff0000u : 0u))) >> (4 * here(lh));
      return (bits & 0xfu) | ((bits >> 4) & 0xf0u) | ((bits >> 8) & 0xf00u) | ((bits >> 12) & 0xf000u);
    };

    f32x16_t acc[DB];
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[db][e] = 0.f;
    float m_run = -INFINITY, l_run = 0.f;

    // The 16 scores of a 32-key block as the matrix cores give them.
    auto products = [&](const char* Kb) __attribute__((always_inline)) {
      f32x16_t s;
#pragma unroll
      for (int e = 0; e < 16; ++e) s[e] = 0.f;
      bf16x8_t kf[DK];
      const int kl = here(k_lane);
#pragma unroll
      for (int kk = 0; kk < DK; ++kk) kf[kk] = *(const bf16x8_t*)(Kb + (kl ^ (32 * kk)));
#pragma unroll
      for (int kk = 0; kk < DK; ++kk) s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf[kk], qf[kk], s, 0, 0, 0);
      return s;
    };
    // Score modifiers, in place; softmax in log2 units over kq.
    auto modify = [&](f32x16_t& s, int jb) __attribute__((always_inline)) {
      if constexpr (SCORE != CACHE_SOFTMAX) {
        const float x0 = (float)(jb + 4 * here(lh) - ipos);
        if (p.softcap > 0.f) {
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            float v = __builtin_fmaf(sl, x0 + (float)(8 * (e >> 2) + (e & 3)), s[e] * c1);
            const float ex = __builtin_amdgcn_exp2f(v * (2.f * kCLog2e / p.softcap));
            v = p.softcap * (1.f - 2.f * __builtin_amdgcn_rcpf(1.f + ex));
            s[e] = SCORE == CACHE_SOFTMAX_MOD ? v * kCLog2e : v;
          }
        } else {
          constexpr float unit = SCORE == CACHE_SOFTMAX_MOD ? kCLog2e : 1.f;
          const float c = here(c1) * unit, slope = here(sl) * unit;
#pragma unroll
          for (int e = 0; e < 16; ++e) s[e] = __builtin_fmaf(slope, x0 + (float)(8 * (e >> 2) + (e & 3)), s[e] * c);
        }
      }
    };
    const float kq = SCORE == CACHE_SOFTMAX ? c1 : 1.f;  // s kq: the score in log2 units (softmax)
    auto weight = [&](float v) __attribute__((always_inline)) {  // sigmoid, ReLU
      if constexpr (SCORE == CACHE_SIGMOID)
        return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-kCLog2e * (v + p.bias)));
      else
        return v < 0.f ? 0.f : v;
    };
    // raises the running maximum if `mx`, of this lane's scores, exceeds it by more than 8
    auto raise = [&](float mx) __attribute__((always_inline)) {
      mx = xhalf_max(mx) * kq;
      const float m_new = mx > m_run + kCLazy ? mx : m_run;
      if (__any(m_new != m_run)) {
        const float a = m_run == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m_run - m_new);
        l_run *= a;
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
          for (int e = 0; e < 16; ++e) acc[db][e] *= a;
        m_run = m_new;
      }
    };
    // V^T of 16 keys
    auto read_v = [&](const char* Vb, int vl, bf16x8_t (&vf)[DB]) __attribute__((always_inline)) {
#pragma unroll
      for (int db = 0; db < DB; ++db) {
        const i16x4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4_t*)(Vb + (vl ^ (64 * db))));
        const i16x4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4_t*)(Vb + 8 * RP + (vl ^ (64 * db) ^ SW8)));
        vf[db] = __builtin_bit_cast(bf16x8_t, (i16x8_t)__builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
      }
    };
    auto add_pv = [&](const bf16x8_t (&vf)[DB], const uint32_t* pk) __attribute__((always_inline)) {
      const bf16x8_t pf = __builtin_bit_cast(bf16x8_t, u32x4_t{pk[0], pk[1], pk[2], pk[3]});
#pragma unroll
      for (int db = 0; db < DB; ++db) acc[db] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf[db], pf, acc[db], 0, 0, 0);
    };

    // A tile that every row sees whole, of scales that are powers of two: both blocks
    // together, so that the second block's products run beside the first one's weights
    // and the first one's second product beside the second's weights.
    auto whole_tile = [&](const char* st) __attribute__((always_inline)) {
      f32x16_t s[2];
      s[0] = products(st);
      s[1] = products(st + 32 * RP);
      modify(s[0], cur.key);
      modify(s[1], cur.key + 32);
      float mo = 0.f;
      if constexpr (SOFTMAX) {
        float mx = fmaxf(s[0][0], s[1][0]);
#pragma unroll
        for (int e = 1; e < 16; ++e) mx = fmaxf(mx, fmaxf(s[0][e], s[1][e]));
        raise(mx);
        mo = m_run == -INFINITY ? 0.f : -m_run;
      }
      const int vl = here(v_lane);
      bf16x8_t vf[2][DB];
      read_v(st, vl, vf[0]);
      float ls[2] = {0.f, 0.f};
      uint32_t pk[2][8];
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) {
#pragma unroll
        for (int w = 0; w < 8; ++w) {
          float a = s[kb][2 * w], b = s[kb][2 * w + 1];
          if constexpr (SOFTMAX) {
            a = __builtin_amdgcn_exp2f(__builtin_fmaf(a, kq, mo));
            b = __builtin_amdgcn_exp2f(__builtin_fmaf(b, kq, mo));
          } else {
            a = weight(a);
            b = weight(b);
          }
          const bf16x2_t pb = pack2(a, b);
          if constexpr (SOFTMAX) ls[kb] = __builtin_amdgcn_fdot2_f32_bf16(pb, kOnes2, ls[kb], false);
          pk[kb][w] = __builtin_bit_cast(uint32_t, pb);
        }
        read_v(st + (32 * kb + 16) * RP, vl, vf[1]);
        add_pv(vf[0], &pk[kb][0]);
        if (kb == 0) read_v(st + 32 * RP, vl, vf[0]);
        add_pv(vf[1], &pk[kb][4]);
      }
      if constexpr (SOFTMAX) l_run += ls[0] + ls[1];
    };

    // One 32-key block of any other tile.
    auto block = [&](const char* st, int kb) __attribute__((always_inline)) {
      const float ks2[2] = {sel(kb, cur.ks[0], cur.ks[2]), sel(kb, cur.ks[1], cur.ks[3])};
      const float vs2[2] = {sel(kb, cur.vs[0], cur.vs[2]), sel(kb, cur.vs[1], cur.vs[3])};
      const bool ok2[2] = {sel(kb, cur.ok[0], cur.ok[2]), sel(kb, cur.ok[1], cur.ok[3])};
      const int jb = cur.key + 32 * kb;
      const char* Kb = st + 32 * kb * RP;
      f32x16_t s = products(Kb);
      // key of register e: jb + 4 lh + 8 (e / 4) + e % 4; e < 8: the block's first group of 16
      if (cur.frac)
#pragma unroll
        for (int e = 0; e < 16; ++e) s[e] *= fraction_of(ks2[e >> 3]);
      uint32_t vis = 0xffffu;
      if (!cur.full) vis = seen(jb, ok2[0], ok2[1]);
      asm("" : "+v"(vis));  // one register, not sixteen
      modify(s, jb);
      uint32_t pk[8];
      if constexpr (SOFTMAX) {
        if (!cur.full)
#pragma unroll
          for (int e = 0; e < 16; ++e) s[e] = (vis >> e) & 1 ? s[e] : -INFINITY;
        float mx = s[0];
#pragma unroll
        for (int e = 1; e < 16; ++e) mx = fmaxf(mx, s[e]);
        raise(mx);
        const float mo = m_run == -INFINITY ? 0.f : -m_run;
#pragma unroll
        for (int e = 0; e < 16; ++e) s[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[e], kq, mo));
      } else {
#pragma unroll
        for (int e = 0; e < 16; ++e) s[e] = cur.full || ((vis >> e) & 1) ? weight(s[e]) : 0.f;
      }
      float inv[2] = {1.f, 1.f};
      if (cur.frac) {
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          const float f = fraction_of(vs2[q]);
          inv[q] = 1.f / f;
#pragma unroll
          for (int e = 8 * q; e < 8 * q + 8; ++e) s[e] = (vis >> e) & 1 ? s[e] * f : 0.f;
        }
      }
      float ls[2] = {0.f, 0.f};
#pragma unroll
      for (int w = 0; w < 8; ++w) {
        const bf16x2_t pb = pack2(s[2 * w], s[2 * w + 1]);
        if constexpr (SOFTMAX) ls[w >> 2] = __builtin_amdgcn_fdot2_f32_bf16(pb, kOnes2, ls[w >> 2], false);
        pk[w] = __builtin_bit_cast(uint32_t, pb);
      }
      if constexpr (SOFTMAX) l_run = __builtin_fmaf(ls[0], inv[0], __builtin_fmaf(ls[1], inv[1], l_run));
      const int vl = here(v_lane);
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        bf16x8_t vf[DB];
        read_v(Kb + 16 * half * RP, vl, vf);
        add_pv(vf, &pk[4 * half]);
      }
    };

    if (s0 < s1) {
      __syncthreads();  // the tile before has been looked at
      if (tid == 0) poison_s = 0;
      load(s0);
      scales();
      __syncthreads();
      store(0, BoolTag<false>());
      __syncthreads();
      for (int s = s0; s < s1; ++s) {
        cur = next;
        const bool more = s + 1 < s1;
        if (more) load(s + 1);
        const int stage = (s - s0) & 1;
        if (cur.full && !cur.frac) {
          whole_tile(lds + stage * STAGE);
        } else {
#pragma unroll 1
          for (int kb = 0; kb < 2; ++kb) block(lds + stage * STAGE, kb);
        }
        if (more) {
          scales();
          store(stage ^ 1, BoolTag<false>());
        }
        __syncthreads();
      }
      if (poison_s != 0) {
        // The rows that see a value that is no number: its NaN, or its infinity (NaN for
        // ReLU, whose weight may be 0), by products of 1 at such values with 1 at the
        // keys that a row sees.
        for (int s = s0; s < s1; ++s) {
          load(s);
          scales();
          if (next.full) continue;
          __syncthreads();
          store(0, BoolTag<true>());
          __syncthreads();
#pragma unroll 1
          for (int hb = 0; hb < 4; ++hb) {
            const uint32_t vis = seen(next.key + 32 * (hb >> 1), sel(hb >> 1, next.ok[0], next.ok[2]), sel(hb >> 1, next.ok[1], next.ok[3])) >> (8 * (hb & 1));
            u32x4_t sees;
#pragma unroll
            for (int i = 0; i < 4; ++i)
              sees[i] = ((vis >> (2 * i)) & 1 ? 0x3f80u : 0u) | ((vis >> (2 * i + 1)) & 1 ? 0x3f800000u : 0u);
            const bf16x8_t sf = __builtin_bit_cast(bf16x8_t, sees);
            const int vl = here(v_lane);
#pragma unroll
            for (int db = 0; db < DB; ++db) {
              const char* pa = lds + 16 * hb * RP;
              const i16x4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4_t*)(pa + (vl ^ (64 * db))));
              const i16x4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4_t*)(pa + 8 * RP + (vl ^ (64 * db) ^ SW8)));
              const i16x8_t a = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
              i16x8_t nan, up, down;
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                const int m = a[i] & 0x7fff;
                const bool inf = SCORE != CACHE_RELU && m == 0x7f80;
                nan[i] = m >= 0x7f80 && !inf ? (short)0x3f80 : (short)0;
                up[i] = inf && a[i] >= 0 ? (short)0x3f80 : (short)0;
                down[i] = inf && a[i] < 0 ? (short)0x3f80 : (short)0;
              }
              f32x16_t zero;
#pragma unroll
              for (int e = 0; e < 16; ++e) zero[e] = 0.f;
              const f32x16_t n = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, nan), sf, zero, 0, 0, 0);
#pragma unroll
              for (int e = 0; e < 16; ++e) acc[db][e] = n[e] > 0.f ? NAN : acc[db][e];
              if constexpr (FMT == 1) {
                const f32x16_t u = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, up), sf, zero, 0, 0, 0);
#pragma unroll
                for (int e = 0; e < 16; ++e) acc[db][e] += u[e] > 0.f ? INFINITY : 0.f;
                const f32x16_t v = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, down), sf, zero, 0, 0, 0);
#pragma unroll
                for (int e = 0; e < 16; ++e) acc[db][e] -= v[e] > 0.f ? INFINITY : 0.f;
              }
            }
          }
        }
        __syncthreads();
      }
    }

    if constexpr (SOFTMAX) l_run = xhalf_sum(l_run);
    if (rok) {
      const ColdArgs a = cold_args();
      if (used <= 1) {
        const float f = SOFTMAX ? (l_run != 0.f ? 1.f / l_run : 0.f) : a->post_scale;
        uint16_t* op = a->o + (int64_t)(sp.tok0 + t) * a->o_st + (int64_t)h * a->o_sh + 4 * here(lh);
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
          for (int q = 0; q < 4; ++q)
            *(u32x2_t*)(op + 32 * db + 8 * q) = u32x2_t{pack_bf16x2(acc[db][4 * q] * f, acc[db][4 * q + 1] * f),
                                                       pack_bf16x2(acc[db][4 * q + 2] * f, acc[db][4 * q + 3] * f)};
      } else {
        const int64_t at = ((int64_t)z * a->T + sp.tok0 + t) * a->H + h;
        float* op = a->part_o + at * D + 4 * here(lh);
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
          for (int q = 0; q < 4; ++q)
            *(f32x4_t*)(op + 32 * db + 8 * q) = f32x4_t{acc[db][4 * q], acc[db][4 * q + 1], acc[db][4 * q + 2], acc[db][4 * q + 3]};
        if (SOFTMAX && lh == 0) {
          a->part_ml[2 * at] = m_run;
          a->part_ml[2 * at + 1] = l_run;
        }
      }
    }
  }
}

}  // namespace chia
