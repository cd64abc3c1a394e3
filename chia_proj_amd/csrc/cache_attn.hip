// cache_attn.hip -- chia_cache_attn: argument checks, the launch of the cache
// attention kernels (cache_attn_kernel.h) and the kernel that joins split keys.
#include <cmath>

#include "cache_attn_kernel.h"
#include "chia_cache.h"

namespace chia {
namespace {

// Joins the parts of rows whose keys were split: o = sum_z 2^(m_z - m) o_z / sum_z 2^(m_z - m) l_z.
// 32 (D = 128) or 16 lanes to a row, float4 each; ZG groups of them share a row's
// parts and meet in LDS, so that a few rows of many parts are not one lane's walk.
template <int D, bool SOFTMAX, int ROWS, int ZG>
__global__ __launch_bounds__(256) void cache_merge_kernel(const CacheAttnParams p) {
  constexpr int LPR = D / 4, SLOTS = 256 / LPR, RPW = SLOTS / ZG, SUBS = ROWS / RPW;
  __shared__ f32x4_t sum_s[ZG > 1 ? 256 : 1];
  __shared__ float ml_s[SLOTS][2];
  const int u = (int)blockIdx.x / SUBS, sub = (int)blockIdx.x % SUBS;
  const int rh = udiv(u, p.div_tiles), rt0 = u - rh * p.tiles;
  const int r = udiv(rh, p.div_hkv), hk = rh - r * p.Hkv;
  const CacheSpan sp = cache_span(p, r);
  const int n_rows = sp.n * p.G;
  const int slot = (int)threadIdx.x / LPR, d = 4 * ((int)threadIdx.x % LPR), zi = slot % ZG;
  const int64_t th = (int64_t)p.T * p.H;
  for (int rt = rt0; rt * ROWS + sub * RPW < n_rows; rt += p.tiles) {
    const TileWalk tw = cache_walk_of<ROWS>(p.mask, p.div_g, sp, rt);
    const int chunk = walk_chunk(tw.n, p.parts, p.chunk);
    const int used = (tw.n + chunk - 1) / chunk;
    if (used <= 1) continue;
    const int row = rt * ROWS + sub * RPW + slot / ZG;
    const bool ok = row < n_rows;
    const int t = ok ? udiv(row, p.div_g) : 0, h = hk * p.G + (ok ? row - t * p.G : 0);
    const int64_t at = (int64_t)(sp.tok0 + t) * p.H + h;
    f32x4_t sum = {0.f, 0.f, 0.f, 0.f};
    float m = -INFINITY, l = 0.f;
    if (ok) {
      // four parts' numbers on their way at a time
      for (int z0 = zi; z0 < used; z0 += 4 * ZG) {
        float mz[4], lz[4];
        f32x4_t oz[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int z = z0 + i * ZG;
          mz[i] = -INFINITY;
          lz[i] = 0.f;
          oz[i] = f32x4_t{0.f, 0.f, 0.f, 0.f};
          if (z < used) {
            oz[i] = *(const f32x4_t*)(p.part_o + (z * th + at) * D + d);
            if constexpr (SOFTMAX) {
              mz[i] = p.part_ml[2 * (z * th + at)];
              lz[i] = p.part_ml[2 * (z * th + at) + 1];
            }
          }
        }
        if constexpr (SOFTMAX) {
          const float all = fmaxf(fmaxf(fmaxf(mz[0], mz[1]), fmaxf(mz[2], mz[3])), m);
          const float f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - all);
          m = all;
          l *= f;
          sum *= f;
#pragma unroll
          for (int i = 0; i < 4; ++i) {  // a part that saw no key has zeros
            const float w = mz[i] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mz[i] - m);
            l = __builtin_fmaf(w, lz[i], l);
            sum += w * oz[i];
          }
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i) sum += oz[i];
        }
      }
    }
    if constexpr (ZG > 1) {
      sum_s[threadIdx.x] = sum;
      if (d == 0) {
        ml_s[slot][0] = m;
        ml_s[slot][1] = l;
      }
      __syncthreads();
      if (zi == 0) {
        float all = -INFINITY;
#pragma unroll
        for (int g = 0; g < ZG; ++g) all = fmaxf(all, ml_s[slot + g][0]);
        sum = f32x4_t{0.f, 0.f, 0.f, 0.f};
        l = 0.f;
#pragma unroll
        for (int g = 0; g < ZG; ++g) {
          const float mg = ml_s[slot + g][0];
          const float w = !SOFTMAX ? 1.f : mg == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mg - all);
          l = __builtin_fmaf(w, ml_s[slot + g][1], l);
          sum += w * sum_s[threadIdx.x + g * LPR];
        }
      }
      __syncthreads();
    }
    if (ok && zi == 0) {
      const float f = !SOFTMAX ? p.post_scale : l != 0.f ? 1.f / l : 0.f;
      *(cu32x2_t*)(p.o + (int64_t)(sp.tok0 + t) * p.o_st + (int64_t)h * p.o_sh + d) =
          cu32x2_t{cpack(sum[0] * f, sum[1] * f), cpack(sum[2] * f, sum[3] * f)};
    }
  }
}

constexpr int64_t kMaxSeq = (int64_t)1 << 28;
constexpr int kCUs = 256;  // MI355X compute units

int block_shift(int32_t bs) {
  for (int s = 4; s <= 8; ++s)
    if (bs == 1 << s) return s;
  return -1;
}

int validate(const chia_cache_attn_args* a) {
  if (!a || !a->attn) return CHIA_ATTN_ERR_NULL;
  if (a->struct_size != sizeof(chia_cache_attn_args) || a->reserved0 != 0) return CHIA_ATTN_ERR_STRUCT;
  for (int i = 0; i < 8; ++i)
    if (a->reserved[i] != 0) return CHIA_ATTN_ERR_STRUCT;
  const chia_attn_args* t = a->attn;
  if (t->struct_size != sizeof(chia_attn_args) || t->reserved0 != 0 || t->reserved[0] != 0 || t->reserved[1] != 0)
    return CHIA_ATTN_ERR_STRUCT;
  if (a->format > CHIA_ATTN_FP8_E5M2 || t->norm > CHIA_ATTN_NORM_RELU) return CHIA_ATTN_ERR_NORM;
  if (t->head_dim != 64 && t->head_dim != 128) return CHIA_ATTN_ERR_HEAD_DIM;
  const int shift = block_shift(a->block_size);
  if (shift < 0 || t->batch < 1 || t->batch > (1 << 24) || t->heads < 1 || t->heads > (1 << 16) || t->kv_heads < 0 ||
      (t->kv_heads > 0 && t->heads % t->kv_heads != 0) || t->seqlen < 1 || t->seqlen >= kMaxSeq || a->width < 1 ||
      a->table_stride < 0 || a->width > (kMaxSeq >> shift) || a->num_blocks < 1 ||
      a->num_blocks > (INT32_MAX >> shift) || a->queries < 0 || a->queries > kMaxSeq ||
      a->queries * t->heads > ((int64_t)1 << 30) || a->max_query < 1 ||
      (!t->cu_seqlens && a->queries != t->batch))
    return CHIA_ATTN_ERR_SHAPE;
  if (t->window < 0 || t->dilation < 1 || t->block < 0 || t->prefix < 0 || (t->dilation > 1 && t->prefix > 0))
    return CHIA_ATTN_ERR_MASK;
  if (!(t->scale > 0.f) || !std::isfinite(t->scale) || !(t->softcap >= 0.f) || !std::isfinite(t->softcap) ||
      !std::isfinite(t->bias) || !std::isfinite(t->post_scale))
    return CHIA_ATTN_ERR_SCALE;
  return CHIA_ATTN_OK;
}

// The launch: which row tile, how many of them per (request, K/V head), and how
// the steps of a tile's walk are split.
struct Shape {
  int tile, waves;
  int64_t tiles, parts, chunk;
};

Shape shape_of(const chia_cache_attn_args* a, const CacheMask& m) {
  const chia_attn_args* t = a->attn;
  const int64_t hkv = t->kv_heads > 0 ? t->kv_heads : t->heads, G = t->heads / hkv;
  const int64_t most = !t->cu_seqlens ? 1 : a->max_query < a->queries ? a->max_query : a->queries;
  const int64_t rows = G * (most < 1 ? 1 : most);
  Shape s;
  // 32 rows to a workgroup start and split better, 128 compute faster: about 870 and
  // 1700 (row x key)s per ns on a full chip, and 17 us more for the latter's longer steps
  // (H32/8 D128, us with 32 and 128: one prompt of 300 tokens 16, 25; 8 of 48 over 4000: 67, 60;
  // 32 of 32 over 4000: 130, 108; 64 of 10 over 4000, whose 40 rows fill 64 and 128: 139, 156).
  const double each = (double)(t->batch * hkv) * (double)(t->seqlen < a->width * a->block_size ? t->seqlen : a->width * a->block_size);
  const double us32 = each * (double)((rows + 31) / 32 * 32) / 0.87e6, us128 = each * (double)((rows + 127) / 128 * 128) / 1.7e6 + 17.0;
  s.tile = rows <= 16 ? CACHE_ROWS16 : us32 <= us128 ? CACHE_ROWS32 : CACHE_ROWS128;
  const int R = kCacheRows[s.tile];
  s.tiles = (rows + R - 1) / R;
  // A bound on the queries that is far too wide does not make millions of empty
  // workgroups: those there are walk more tiles.
  const int64_t tiles_most = ((int64_t)1 << 18) / (t->batch * hkv);
  if (s.tiles > tiles_most) s.tiles = tiles_most > 0 ? tiles_most : 1;
  // steps of the longest request's last tile
  const int64_t S = t->seqlen < (a->width * a->block_size) ? t->seqlen : a->width * a->block_size;
  const int64_t span = (R + G - 1) / G;
  const int32_t i0 = (int32_t)(S - (span < most ? span : most));
  const TileWalk w = cache_tile_walk(m, i0 < 0 ? 0 : i0, (int32_t)S - 1, (int32_t)S, kCacheStep[s.tile]);
  const int64_t steps = w.n > 0 ? w.n : 1;
  const int64_t groups = t->batch * hkv * s.tiles;
  // How many parts.  A part costs a workgroup's start and end (lengths, table, first
  // keys; merge) whatever it holds, the second kernel 3 to 5 us, and too few parts
  // leave CUs idle or waiting for the longest request.  us by workgroups asked for: 2
  // requests of 131072 tokens, H32/8 D128, 100 (512), 118 (576), 103 (768), 109 (1024); 11 of up to 32318,
  // H16/8 D64, 90 (440), 68 (704), 77 (1496); 16 of 33 .. 4096, 16 heads, D64, 38 (512), 33 (1024), 28 (1536),
  // 33 (2048); 64 of 97 .. 8192, H32/8 D128, 125 (1 part), 113 (4), 106 (5), 108 (6); 16 verifying 5 tokens over 4096,
  // 35 (512), 42 (768), 47 (1024); 2 of 2994, 2 heads, parts of 16 steps 13.1, of 8 11.6.
  const bool small = s.tile == CACHE_ROWS16;
  const int64_t most_wgs = small ? (t->head_dim == 64 ? 4 : 3) : 2;  // per CU at once
  int64_t least = 16, parts;
  if (s.tile == CACHE_ROWS128) least = 4;
  else if (small && groups * steps <= 2048 && steps > 32) least = 8;
  if (groups <= 128 || !small) {
    // Few (request, head, row tile)s: their parts are nearly equal, so that the CUs with
    // most of them set the time: the number whose 2, 3 or 4 per CU leave the fewest
    // places empty.
    parts = 1;
    double best = 0.0;
    for (int64_t k = 2; k <= most_wgs; ++k) {
      const int64_t n = k * kCUs / groups;
      const double used = (double)(n * groups) / (double)(k * kCUs);
      if (n >= 1 && used > best + 0.02) best = used, parts = n;
    }
  } else {
    // Many: their parts are of unequal length or not there at all, and half as many
    // again as the chip holds keep it full; but, for balance, no parts much beyond 48 steps.
    parts = most_wgs * kCUs * 3 / 2 / groups;
    int64_t balance = steps / 48;
    if (balance > 6 * most_wgs * kCUs / groups) balance = 6 * most_wgs * kCUs / groups;
    if (parts < balance) parts = balance;
  }
  if (parts > steps / least) parts = steps / least;
  if (parts < 1) parts = 1;
  // Eight wavefronts to a workgroup where the parts are few: the same wavefronts per
  // CU in one workgroup instead of two, with half the parts to join, or none (16-row tiles,
  // us with four and eight: 32 requests under a window of 1024, 8 heads D128, 20.3 (2 parts), 17.9 (1); 4 of
  // 17848, 16 heads D128, 54, 52; 11 of 32318, 8 heads D64, 69, 64; 56 of 397, 2 heads D64, 7.8, 7.1).
  s.waves = 4;
  if (small && steps > 8 && (groups <= 128 || (groups <= kCUs && parts <= 2))) {
    s.waves = 8;
    parts = (t->head_dim == 64 ? 2 : 1) * kCUs / groups;
    if (groups > 128) parts = 1;
    const int64_t most = steps / (groups * steps <= 2048 && steps > 32 ? 8 : 12);
    if (parts > most) parts = most;
    if (parts < 1) parts = 1;
  }
  s.chunk = (steps + parts - 1) / parts;
  s.parts = (steps + s.chunk - 1) / s.chunk;
  return s;
}

CacheMask mask_of(const chia_attn_args* t) {
  CacheMask m;
  // a reach past every length is none
  m.causal = t->causal ? 1 : 0;
  m.window = t->window < kMaxSeq ? t->window : 0;
  m.dil = t->dilation < kMaxSeq ? t->dilation : (int32_t)kMaxSeq;
  m.blk = t->block < kMaxSeq ? t->block : 0;
  m.prefix = t->prefix < kMaxSeq ? t->prefix : (int32_t)kMaxSeq;
  m.div_blk = make_udiv(m.blk > 0 ? m.blk : 1);
  m.div_dil = make_udiv(m.dil);
  m.comb = cache_comb(m.dil);
  return m;
}

struct Merge {
  CacheAttnFn fn;
  int subs;  // workgroups per row tile
};

template <int D, bool SOFTMAX, int ROWS>
Merge merge_of(bool many) {
  constexpr int slots = 1024 / D;
  return many ? Merge{cache_merge_kernel<D, SOFTMAX, ROWS, 8>, ROWS * 8 / slots}
              : Merge{cache_merge_kernel<D, SOFTMAX, ROWS, 1>, ROWS / slots};
}

template <int D, bool SOFTMAX>
Merge merge_of(int tile, bool many) {
  return tile == CACHE_ROWS16 ? merge_of<D, SOFTMAX, kCacheRows[CACHE_ROWS16]>(many)
         : tile == CACHE_ROWS32 ? merge_of<D, SOFTMAX, kCacheRows[CACHE_ROWS32]>(many)
                                : merge_of<D, SOFTMAX, kCacheRows[CACHE_ROWS128]>(many);
}

Merge merge_kernel(int head_dim, bool softmax, int tile, bool many) {
  return head_dim == 64 ? (softmax ? merge_of<64, true>(tile, many) : merge_of<64, false>(tile, many))
                        : (softmax ? merge_of<128, true>(tile, many) : merge_of<128, false>(tile, many));
}

int64_t workspace_of(const chia_cache_attn_args* a, const Shape& s) {
  return s.parts > 1 ? s.parts * a->queries * a->attn->heads * (a->attn->head_dim + 2) * (int64_t)sizeof(float) : 0;
}

}  // namespace
}  // namespace chia

using namespace chia;

extern "C" int64_t chia_cache_attn_workspace_size(const chia_cache_attn_args* a) {
  const int st = validate(a);
  if (st != CHIA_ATTN_OK) return st;
  return workspace_of(a, shape_of(a, mask_of(a->attn)));
}

extern "C" int chia_cache_attn(const chia_cache_attn_args* a, void* stream) {
  const int st = validate(a);
  if (st != CHIA_ATTN_OK) return st;
  if (a->queries == 0) return CHIA_ATTN_OK;
  const chia_attn_args* t = a->attn;
  if (!t->q || !t->k || !t->v || !t->o || !a->k_scale || !a->v_scale || !a->block_tables || !a->seq_lens)
    return CHIA_ATTN_ERR_NULL;
  for (const void* ptr : {t->q, t->k, t->v, (const void*)t->o, (const void*)a->workspace})
    if ((uintptr_t)ptr & 15u) return CHIA_ATTN_ERR_ALIGN;
  for (const void* ptr : {(const void*)a->k_scale, (const void*)a->v_scale, (const void*)a->block_tables,
                          (const void*)a->seq_lens, (const void*)t->cu_seqlens, (const void*)t->head_scale,
                          (const void*)t->alibi_slopes})
    if ((uintptr_t)ptr & 3u) return CHIA_ATTN_ERR_ALIGN;
  for (int i = 0; i < 3; ++i)
    if ((i > 0 && (t->q_stride[i] % 8 || t->o_stride[i] % 8)) || t->k_stride[i] % 16 || t->v_stride[i] % 16)
      return CHIA_ATTN_ERR_ALIGN;
  // a lane reaches the 16 tokens of a load with 32-bit offsets
  for (const int64_t* sd : {t->k_stride, t->v_stride})
    if (sd[2] < 0 || sd[2] >= ((int64_t)1 << 26)) return CHIA_ATTN_ERR_SHAPE;

  CacheAttnParams p{};
  p.mask = mask_of(t);
  const Shape s = shape_of(a, p.mask);
  const int64_t bytes = workspace_of(a, s);
  if (bytes > 0 && (!a->workspace || a->workspace_bytes < bytes)) return CHIA_ATTN_ERR_WORKSPACE;
  p.q = (const uint16_t*)t->q;
  p.o = (uint16_t*)t->o;
  p.k = (const uint8_t*)t->k;
  p.v = (const uint8_t*)t->v;
  p.ks = a->k_scale;
  p.vs = a->v_scale;
  p.q_sh = t->q_stride[1], p.q_st = t->q_stride[2];
  p.o_sh = t->o_stride[1], p.o_st = t->o_stride[2];
  p.k_sb = t->k_stride[0], p.k_sh = t->k_stride[1], p.k_st = t->k_stride[2];
  p.v_sb = t->v_stride[0], p.v_sh = t->v_stride[1], p.v_st = t->v_stride[2];
  p.ks_sb = a->k_scale_stride[0], p.ks_sh = a->k_scale_stride[1];
  p.vs_sb = a->v_scale_stride[0], p.vs_sh = a->v_scale_stride[1];
  p.table = a->block_tables;
  p.table_stride = a->table_stride;
  p.lens = a->seq_lens;
  p.cu = t->cu_seqlens;
  p.head_scale = t->head_scale;
  p.alibi = t->alibi_slopes;
  p.R = (int32_t)t->batch;
  p.H = (int32_t)t->heads;
  p.Hkv = t->kv_heads > 0 ? t->kv_heads : p.H;
  p.G = p.H / p.Hkv;
  p.T = (int32_t)a->queries;
  p.width = (int32_t)a->width;
  p.num_blocks = (int32_t)a->num_blocks;
  p.bshift = block_shift(a->block_size);
  p.tiles = (int32_t)s.tiles;
  p.parts = (int32_t)s.parts;
  p.chunk = (int32_t)s.chunk;
  p.div_tiles = make_udiv(p.tiles);
  p.div_hkv = make_udiv(p.Hkv);
  p.div_g = make_udiv(p.G);
  p.scale = t->scale;
  p.softcap = t->softcap;
  p.bias = t->bias;
  p.post_scale = t->post_scale;
  p.part_o = (float*)a->workspace;
  p.part_ml = bytes > 0 ? p.part_o + s.parts * a->queries * t->heads * t->head_dim : nullptr;
  const int64_t units = t->batch * p.Hkv * s.tiles, wgs = units * s.parts;
  if (wgs > INT32_MAX / 4 || units > INT32_MAX / 64) return CHIA_ATTN_ERR_SHAPE;
  p.units = (int32_t)units;
  p.div_units = make_udiv(p.units);

  const int score = t->norm == CHIA_ATTN_NORM_SIGMOID ? CACHE_SIGMOID
                    : t->norm == CHIA_ATTN_NORM_RELU  ? CACHE_RELU
                    : t->alibi_slopes || t->softcap > 0.f ? CACHE_SOFTMAX_MOD : CACHE_SOFTMAX;
  const CacheAttnFn fn = s.tile == CACHE_ROWS128 ? select_cache_prompt_kernel((int)t->head_dim, (int)a->format, score)
                         : t->head_dim == 64     ? select_cache_kernel_d64((int)a->format, score, s.tile, s.waves)
                                                 : select_cache_kernel_d128((int)a->format, score, s.tile, s.waves);
  if (!fn) return CHIA_ATTN_ERR_NORM;
  void* kargs[] = {&p};
  hipError_t err = hipLaunchKernel(reinterpret_cast<const void*>(fn), dim3((unsigned)wgs), dim3(64 * (unsigned)s.waves), kargs, 0,
                                   (hipStream_t)stream);
  if (err == hipSuccess && s.parts > 1) {
    const Merge m = merge_kernel((int)t->head_dim, t->norm == CHIA_ATTN_NORM_SOFTMAX, s.tile, s.parts >= 8);
    err = hipLaunchKernel(reinterpret_cast<const void*>(m.fn), dim3((unsigned)(units * m.subs)), dim3(256), kargs, 0,
                          (hipStream_t)stream);
  }
  if (err != hipSuccess) return (int)err;
  err = hipGetLastError();
  return err == hipSuccess ? CHIA_ATTN_OK : (int)err;
}
