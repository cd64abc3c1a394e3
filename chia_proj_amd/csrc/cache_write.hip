// cache_write.hip -- rounding new K / V tokens into the paged 8-bit cache.
//
// A run is the consecutive new tokens of one page.  For each run and K/V head:
//   need  = least 2^e >= 2^-126 with max |finite value| <= 2^e top,
//           top = 1.75 2^8 (e4m3) or 1.75 2^15 (e5m2): from the exponent and the
//           fraction (<= or > 0.75) of the largest bf16 magnitude, as integers;
//   scale = the page had begun (the run starts behind its first place)
//           ? max(need, old scale) : need;
//   codes = rne(value / scale); kept codes *= old / scale, rounded, if that is not 1.
// A power of two costs a floating-point code no precision (only the exponent
// moves), makes the division and, but for codes that become subnormal, the
// rescaling of kept codes exact, and makes a page's scale independent of how its
// tokens were cut into calls.
//
// Bound by memory: 4 D bytes in and 2 D out per token and head.  A team of 1, 2
// or 4 wavefronts holds a whole run in registers (16-byte loads, 16 lanes a row
// at D = 128) between the maximum and the rounding, so K and V are read once.  20
// prompts of up to 4096 tokens, 8 heads, D = 128 (221 MB): 50 us, 4.4 TB/s; 128 single
// tokens: 4.8 us (the host call: 7.5).
#include <hip/hip_runtime.h>

#include "chia_cache.h"
#include "cache_geom.h"

namespace chia {
namespace {

typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));

struct WriteSide {
  const uint16_t* x;
  uint8_t* codes;
  float* scale;
  int64_t x_st, x_sh, c_sb, c_sh, c_st, s_sb, s_sh;
};

struct WriteParams {
  WriteSide side[2];  // K, V
  const int32_t* slots;
  int32_t T, H, n_slots, bshift, window;
  UDiv div_h;
};

// A scale that was there; 0 for what is none.
__device__ __forceinline__ float usable(float s) { return s > 0.f && s < INFINITY ? s : 0.f; }

template <int FMT>  // CHIA_ATTN_FP8_E4M3 / E5M2
__device__ __forceinline__ uint32_t pack4(float a, float b, float c, float d) {
  int r;
  if constexpr (FMT == 0) {
    r = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    r = __builtin_amdgcn_cvt_pk_fp8_f32(c, d, r, true);
  } else {
    r = __builtin_amdgcn_cvt_pk_bf8_f32(a, b, 0, false);
    r = __builtin_amdgcn_cvt_pk_bf8_f32(c, d, r, true);
  }
  return (uint32_t)r;
}

template <int FMT>
__device__ __forceinline__ float code_at(uint32_t w, int i) {
  if constexpr (FMT == 0)
    return i == 0 ? __builtin_amdgcn_cvt_f32_fp8(w, 0) : i == 1 ? __builtin_amdgcn_cvt_f32_fp8(w, 1)
         : i == 2 ? __builtin_amdgcn_cvt_f32_fp8(w, 2) : __builtin_amdgcn_cvt_f32_fp8(w, 3);
  else
    return i == 0 ? __builtin_amdgcn_cvt_f32_bf8(w, 0) : i == 1 ? __builtin_amdgcn_cvt_f32_bf8(w, 1)
         : i == 2 ? __builtin_amdgcn_cvt_f32_bf8(w, 2) : __builtin_amdgcn_cvt_f32_bf8(w, 3);
}

// Infinities to the largest value; NaN passes both comparisons.
template <int FMT>
__device__ __forceinline__ float bounded(float x) {
  constexpr float top = FMT == 0 ? 448.f : 57344.f;
  return x > top ? top : x < -top ? -top : x;
}

// p, an fp32 result whose exact value is p + err, rounded to odd instead: cut towards
// zero, the last bit 1 if anything was cut, so that the rounding to 8 bits that
// follows sees on which side of a tie the exact value lies.
__device__ __forceinline__ float to_odd(float p, float err) {
  if (!(err > 0.f || err < 0.f) || p == 0.f) return p;
  uint32_t b = __float_as_uint(p);
  if ((err < 0.f) != (p < 0.f)) b -= 1;
  return __uint_as_float(b | 1u);
}

// x / scale and code * ratio, as far as the rounding to 8 bits looks.  Powers of two
// (what this file makes) are exact; a page that somebody else rounded may have any scale.
__device__ __forceinline__ float over(float x, float scale, float inv, bool pow2) {
  if (pow2) return x * inv;
  const float q = x / scale;
  return to_odd(q, __builtin_fmaf(-q, scale, x));
}

__device__ __forceinline__ float times(float x, float ratio) {
  const float y = x * ratio;
  return to_odd(y, __builtin_fmaf(x, ratio, -y));
}

// Magnitude bits of a bf16, 0 for infinities and NaN; the order of the bits is that of the values.
__device__ __forceinline__ uint32_t finite_bits(uint32_t h) {
  const uint32_t b = h & 0x7fffu;
  return b < 0x7f80u ? b : 0u;
}

// The least 2^e >= 2^-126 with the bf16 magnitude `bits` <= 1.75 2^(e + SHIFT).
template <int FMT>
__device__ __forceinline__ float need_of(uint32_t bits) {
  constexpr int shift = FMT == 0 ? 8 : 15;
  const int e = (int)(bits >> 7) - 127 - shift + ((bits & 0x7fu) > 0x60u ? 1 : 0);
  return __uint_as_float((uint32_t)((e < -126 ? -126 : e) + 127) << 23);
}

// Eight bf16 values to codes.
template <int FMT>
__device__ __forceinline__ u32x2_t codes_of(u32x4_t x, float scale, float inv, bool pow2) {
  float f[8];
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    f[2 * w] = bounded<FMT>(over(__uint_as_float(x[w] << 16), scale, inv, pow2));
    f[2 * w + 1] = bounded<FMT>(over(__uint_as_float(x[w] & 0xffff0000u), scale, inv, pow2));
  }
  return u32x2_t{pack4<FMT>(f[0], f[1], f[2], f[3]), pack4<FMT>(f[4], f[5], f[6], f[7])};
}

// The first `rows` rows of a page to a scale that has grown: chunks first, first + step, ...
template <int D, int FMT>
__device__ __forceinline__ void rescale(uint8_t* page, int64_t row_stride, int rows, float ratio, int first, int step) {
  constexpr int LPR = D / 8;
  for (int c = first; c < rows * LPR; c += step) {
    u32x2_t* at = (u32x2_t*)(page + (int64_t)(c / LPR) * row_stride + (c % LPR) * 8);
    u32x2_t v = *at;
#pragma unroll
    for (int w = 0; w < 2; ++w)
      v[w] = pack4<FMT>(bounded<FMT>(times(code_at<FMT>(v[w], 0), ratio)), bounded<FMT>(times(code_at<FMT>(v[w], 1), ratio)),
                        bounded<FMT>(times(code_at<FMT>(v[w], 2), ratio)), bounded<FMT>(times(code_at<FMT>(v[w], 3), ratio)));
    *at = v;
  }
}

__device__ __forceinline__ uint32_t largest(u32x4_t x) {
  uint32_t m = 0;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    const uint32_t lo = finite_bits(x[w]), hi = finite_bits(x[w] >> 16), h = lo > hi ? lo : hi;
    m = m > h ? m : h;
  }
  return m;
}

// W wavefronts to a team; N 16-byte chunks of a run per lane.
template <int D, int FMT, int W, int N>
__global__ __launch_bounds__(256) void cache_write_kernel(const WriteParams p) {
  constexpr int LPR = D / 8;         // lanes per row
  constexpr int TEAMS = 4 / W;
  __shared__ uint32_t amax_s[4];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int tl = (wave % W) * 64 + lane;  // lane of the team
  const int bs = 1 << p.bshift;
  // unit = (window of tokens, side, head)
  const int unit = (int)blockIdx.x * TEAMS + wave / W;
  const int wh = udiv(unit, p.div_h), head = unit - wh * p.H;
  const int t0 = (wh >> 1) * p.window;
  if (W == 1 && t0 >= p.T) return;  // with larger teams the whole workgroup is one unit or two: below
  const WriteSide& s = p.side[wh & 1];
  const int t_end = imin32(t0 + p.window, p.T);

  auto slot_at = [&](int t) -> int32_t {  // -1 outside the cache or the tokens
    if (t < 0 || t >= p.T) return -1;
    return cache_slot(p.slots[t], p.n_slots);
  };

  for (int base = t0; base < t0 + p.window; base += 64) {
    // the runs that begin at tokens base .. base + 63 of this window
    const int t = base + lane;
    const int32_t mine = slot_at(t), before = slot_at(t - 1);
    const bool begins = mine >= 0 && (before < 0 || before + 1 != mine || (mine & (bs - 1)) == 0);
    uint64_t starts = __ballot(begins && t < t_end);
    const uint64_t goes_on = __ballot(mine >= 0 && !begins);  // continues the run of the token before
    // Runs of one token (decoding requests among prompts): a row's lanes to each,
    // several at a time, rather than the whole team to one after the other.
    const uint64_t single = starts & ~(goes_on >> 1) & ~(1ull << 63);
    if (single) {
      constexpr int PER = 64 / LPR, DEEP = 4;  // tokens at a time, rounds in flight
      const int count = __popcll(single);
      starts &= ~single;
      // lane i: the token of the i-th of them
      const bool is = (single >> lane) & 1;
      const int rank = __popcll(single & ((1ull << lane) - 1));
      const int order = __builtin_amdgcn_ds_permute((is ? rank : count + lane - rank) << 2, lane);
      for (int k0 = (wave % W) * DEEP * PER; k0 < count; k0 += W * DEEP * PER) {
        u32x4_t x[DEEP];
        int32_t slot[DEEP];
        float old[DEEP];
#pragma unroll
        for (int k = 0; k < DEEP; ++k) {
          const int i = k0 + k * PER + lane / LPR, at = __shfl(order, i & 63);
          const int32_t v = __shfl(mine, at);
          slot[k] = i < count ? v : -1;
          x[k] = u32x4_t{0, 0, 0, 0};
          old[k] = 0.f;
          if (slot[k] >= 0) {
            x[k] = *(const u32x4_t*)(s.x + (int64_t)(base + at) * s.x_st + head * s.x_sh + (lane % LPR) * 8);
            if (slot[k] & (bs - 1)) old[k] = s.scale[(int64_t)(slot[k] >> p.bshift) * s.s_sb + head * s.s_sh];
          }
        }
#pragma unroll
        for (int k = 0; k < DEEP; ++k) {
          uint32_t amax = largest(x[k]);
#pragma unroll
          for (int d = 1; d < LPR; d <<= 1) {
            const uint32_t o = (uint32_t)__shfl_xor((int)amax, d);
            amax = amax > o ? amax : o;
          }
          if (slot[k] < 0) continue;
          const int off = slot[k] & (bs - 1);
          const int64_t page = slot[k] >> p.bshift;
          old[k] = usable(old[k]);
          const float need = need_of<FMT>(amax), scale = need > old[k] ? need : old[k];
          const bool pow2 = (__float_as_uint(scale) & 0x7fffffu) == 0, grown = off > 0 && scale != old[k];
          if (lane % LPR == 0 && (off == 0 || grown)) s.scale[page * s.s_sb + head * s.s_sh] = scale;
          uint8_t* cp = s.codes + page * s.c_sb + head * s.c_sh;
          *(u32x2_t*)(cp + (int64_t)off * s.c_st + (lane % LPR) * 8) = codes_of<FMT>(x[k], scale, 1.f / scale, pow2);
          if (grown) rescale<D, FMT>(cp, s.c_st, off, old[k] / scale, lane % LPR, LPR);
        }
      }
    }
    while (true) {
      bool any = starts != 0;
      if constexpr (W == 2) {
        // two teams of one workgroup share its barriers: both go on while either has a run
        any = __syncthreads_or(any);
      }
      if (!any) break;
      const bool live = starts != 0;
      const int i = live ? __builtin_ctzll(starts) : 0;
      const int run_t = base + i;
      const int32_t slot = live ? __builtin_amdgcn_readlane(mine, i) : 0;
      const int off = slot & (bs - 1);
      int len = 0;  // tokens of the run
      if (live) {
        const uint64_t behind = i < 63 ? ~(goes_on >> (i + 1)) : ~0ull;  // its lowest bit: the first that does not go on
        len = i < 63 ? 1 + __builtin_ctzll(behind) : 1;
        if (len > 63 - i) {  // up to the last lane, and perhaps further
          len = 64 - i;
          const int most = bs - off;
          while (len < most) {
            const int k = len + lane;
            const uint64_t same = __ballot(k < most && slot_at(run_t + k) == slot + k);
            const int n = same == ~0ull ? 64 : __builtin_ctzll(~same);
            len += n;
            if (n < 64) break;
          }
        }
      }
      const int64_t page = slot >> p.bshift;
      float* sp = s.scale + page * s.s_sb + head * s.s_sh;
      float old = live && off > 0 ? *sp : 0.f;
      const uint16_t* xr = s.x + (int64_t)run_t * s.x_st + head * s.x_sh;
      u32x4_t x[N];
      uint32_t amax = 0;
#pragma unroll
      for (int n = 0; n < N; ++n) {
        const int c = n * (64 * W) + tl, row = c / LPR, col = c % LPR;
        x[n] = u32x4_t{0, 0, 0, 0};
        if (row < len) x[n] = *(const u32x4_t*)(xr + (int64_t)row * s.x_st + col * 8);
      }
#pragma unroll
      for (int n = 0; n < N; ++n) {
        const uint32_t m = largest(x[n]);
        amax = amax > m ? amax : m;
      }
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) {
        const uint32_t o = (uint32_t)__shfl_xor((int)amax, d);
        amax = amax > o ? amax : o;
      }
      if constexpr (W > 1) {
        if (lane == 0) amax_s[wave] = amax;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < W; ++w) {
          const uint32_t o = amax_s[wave / W * W + w];
          amax = amax > o ? amax : o;
        }
        __syncthreads();
      }
      if (live) {
        old = usable(old);
        const float need = need_of<FMT>(amax);
        const float scale = need > old ? need : old;
        const bool grown = off > 0 && scale != old;
        if (tl == 0 && (off == 0 || grown)) *sp = scale;
        uint8_t* cp = s.codes + page * s.c_sb + head * s.c_sh;
        const bool pow2 = (__float_as_uint(scale) & 0x7fffffu) == 0;
        const float inv = 1.f / scale;
#pragma unroll
        for (int n = 0; n < N; ++n) {
          const int c = n * (64 * W) + tl, row = c / LPR, col = c % LPR;
          if (row < len)
            *(u32x2_t*)(cp + (int64_t)(off + row) * s.c_st + col * 8) = codes_of<FMT>(x[n], scale, inv, pow2);
        }
        if (grown) rescale<D, FMT>(cp, s.c_st, off, old / scale, tl, 64 * W);
        starts &= starts - 1;
      }
    }
  }
}

using WriteFn = void (*)(WriteParams);

struct WriteKernel {
  WriteFn fn;
  int teams;  // per workgroup
};

// A lane holds 4 chunks of 16 bytes (8 and 16 for the largest pages): a page has
// bs D / 8 chunks for 64 lanes of 1, 2 or 4 wavefronts.
template <int D, int FMT>
WriteKernel pick(int bs) {
  switch (bs * D / 512) {  // chunks per lane of one wavefront
    case 2: return {cache_write_kernel<D, FMT, 1, 2>, 4};
    case 4: return {cache_write_kernel<D, FMT, 1, 4>, 4};
    case 8: return {cache_write_kernel<D, FMT, 1, 8>, 4};
    case 16: return {cache_write_kernel<D, FMT, 2, 8>, 2};
    case 32: return {cache_write_kernel<D, FMT, 4, 8>, 1};
    case 64: return {cache_write_kernel<D, FMT, 4, 16>, 1};
  }
  return {nullptr, 0};
}

}  // namespace
}  // namespace chia

using namespace chia;

extern "C" int chia_cache_write(const chia_cache_write_args* a, void* stream) {
  if (!a) return CHIA_ATTN_ERR_NULL;
  if (a->struct_size != sizeof(chia_cache_write_args)) return CHIA_ATTN_ERR_STRUCT;
  for (int i = 0; i < 7; ++i)
    if (a->reserved[i] != 0) return CHIA_ATTN_ERR_STRUCT;
  if (a->format > CHIA_ATTN_FP8_E5M2) return CHIA_ATTN_ERR_NORM;
  if (a->head_dim != 64 && a->head_dim != 128) return CHIA_ATTN_ERR_HEAD_DIM;
  int shift = -1;
  for (int s = 4; s <= 8; ++s)
    if (a->block_size == 1 << s) shift = s;
  if (shift < 0 || a->tokens < 0 || a->tokens > ((int64_t)1 << 28) || a->kv_heads < 1 || a->kv_heads > (1 << 16) ||
      a->num_blocks < 1 || a->num_blocks > (INT32_MAX >> shift))
    return CHIA_ATTN_ERR_SHAPE;
  if (a->tokens == 0) return CHIA_ATTN_OK;
  if (!a->k || !a->v || !a->k_cache || !a->v_cache || !a->k_scale || !a->v_scale || !a->slots) return CHIA_ATTN_ERR_NULL;
  for (const void* ptr : {a->k, a->v, (const void*)a->k_cache, (const void*)a->v_cache})
    if ((uintptr_t)ptr & 15u) return CHIA_ATTN_ERR_ALIGN;
  for (const void* ptr : {(const void*)a->k_scale, (const void*)a->v_scale, (const void*)a->slots})
    if ((uintptr_t)ptr & 3u) return CHIA_ATTN_ERR_ALIGN;
  for (int i = 0; i < 3; ++i)
    if ((i < 2 && (a->k_stride[i] % 8 || a->v_stride[i] % 8)) || a->k_cache_stride[i] % 16 || a->v_cache_stride[i] % 16)
      return CHIA_ATTN_ERR_ALIGN;
  WriteParams p{};
  p.side[0] = {(const uint16_t*)a->k, (uint8_t*)a->k_cache, a->k_scale, a->k_stride[0], a->k_stride[1],
               a->k_cache_stride[0], a->k_cache_stride[1], a->k_cache_stride[2], a->k_scale_stride[0], a->k_scale_stride[1]};
  p.side[1] = {(const uint16_t*)a->v, (uint8_t*)a->v_cache, a->v_scale, a->v_stride[0], a->v_stride[1],
               a->v_cache_stride[0], a->v_cache_stride[1], a->v_cache_stride[2], a->v_scale_stride[0], a->v_scale_stride[1]};
  p.slots = a->slots;
  p.T = (int32_t)a->tokens;
  p.H = (int32_t)a->kv_heads;
  p.n_slots = (int32_t)(a->num_blocks << shift);
  p.bshift = shift;
  p.div_h = make_udiv(p.H);
  const int fmt = (int)a->format, bs = a->block_size;
  const WriteKernel k = a->head_dim == 64 ? (fmt ? pick<64, 1>(bs) : pick<64, 0>(bs))
                                          : (fmt ? pick<128, 1>(bs) : pick<128, 0>(bs));
  if (!k.fn) return CHIA_ATTN_ERR_SHAPE;
  // A window of tokens per team: as many as a wavefront has rows' worth of lanes (4 or
  // 8), since each may be a run of its own (decoding), and more, up to a page, where
  // that many teams would mostly find that their tokens continue a run (prompts): as many as keep 2048 teams (8 thousand tokens of
  // 16 heads, D = 64, pages of 64: 33 us with 65536 teams, 24 with 16384, 16 with 4096; 16384 of 8,
  // D = 128, pages of 128: 37 with 4096, 25 with 2048).
  int64_t units = 2 * a->kv_heads * a->tokens;
  p.window = 512 / (int)a->head_dim;
  units = 2 * a->kv_heads * ((a->tokens + p.window - 1) / p.window);
  while (p.window < bs && units > 2048) {
    p.window *= 2;
    units = 2 * a->kv_heads * ((a->tokens + p.window - 1) / p.window);
  }
  const int64_t wgs = (units + k.teams - 1) / k.teams;
  if (wgs > INT32_MAX / 4) return CHIA_ATTN_ERR_SHAPE;
  void* kargs[] = {&p};
  hipError_t err = hipLaunchKernel(reinterpret_cast<const void*>(k.fn), dim3((unsigned)wgs), dim3(256), kargs, 0,
                                   (hipStream_t)stream);
  if (err != hipSuccess) return (int)err;
  err = hipGetLastError();
  return err == hipSuccess ? CHIA_ATTN_OK : (int)err;
}
