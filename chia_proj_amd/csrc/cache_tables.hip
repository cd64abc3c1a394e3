// cache_tables.hip -- block tables, slots and free list of the paged K/V cache.
//
// One step of a serving loop, per request r with ctx tokens in the cache and n
// new ones (bs: tokens per page):
//   have = ceil(ctx / bs), take = min(ceil((ctx + n) / bs), width) - have,
//   rank_r = sum of take over the requests before, cu_r = sum of n over them,
//   table[r][have + m] = free[count - 1 - (rank_r + m)],
//   slot of token cu_r + x = table[r][p / bs] bs + p % bs, p = ctx + x.
// Two prefix sums over the requests and a scatter.  It reads and writes a few
// bytes per request and token, so what bounds it is the launch and the chain
// lengths -> scan -> table entry -> slot; every workgroup scans all requests
// itself (1024 at a time, four bytes each) rather than wait for another one, and
// they share the tokens and pages by stride.  256 decoding requests take 5.8 us, 48
// prompts of up to 4096 tokens 6.3 (the host call: 10.4).
#include <hip/hip_runtime.h>

#include "chia_cache.h"
#include "mask.h"

namespace chia {
namespace {

constexpr int kThreads = 1024;
constexpr int kWaves = kThreads / 64;
constexpr uint32_t kMost = 1u << 30;     // sums stop here: more tokens or pages than any buffer holds
constexpr int32_t kMaxLen = 1 << 28;

struct TablesParams {
  int32_t* table;
  int64_t table_stride;
  int32_t R, width, bs, bshift;
  const int32_t *ctx, *fresh, *free_blocks, *free_count;
  int64_t capacity;
  int32_t T;
  int32_t *slots, *positions, *cu, *lens, *free_left, *missing;
};

__device__ __forceinline__ uint32_t sat(uint32_t a, uint32_t b) {
  const uint32_t s = a + b;  // both <= 2^30
  return s < kMost ? s : kMost;
}

struct Pair {
  uint32_t tok, page;
};

// Inclusive saturating scan over the workgroup's threads; total: the last value.
__device__ Pair scan(Pair x, Pair& total, Pair* part) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const uint32_t a = __shfl_up(x.tok, d), b = __shfl_up(x.page, d);
    if (lane >= d) x = {sat(x.tok, a), sat(x.page, b)};
  }
  if (lane == 63) part[wave] = x;
  __syncthreads();
  Pair before = {0, 0}, all = {0, 0};
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    const Pair y = part[w];
    if (w < wave) before = {sat(before.tok, y.tok), sat(before.page, y.page)};
    all = {sat(all.tok, y.tok), sat(all.page, y.page)};
  }
  __syncthreads();
  total = all;
  return {sat(x.tok, before.tok), sat(x.page, before.page)};
}

__device__ __forceinline__ int32_t length(int32_t n) { return n < 0 ? 0 : imin32(n, kMaxLen); }

// The last row of the chunk whose start is <= x (starts ascend; start[0] <= x).
__device__ __forceinline__ int row_of(const uint32_t* start, int rows, uint32_t x) {
  int lo = 0, n = rows;
  while (n > 1) {
    const int half = n >> 1;
    if (start[lo + half] <= x) lo += half;
    n -= half;
  }
  return lo;
}

__global__ __launch_bounds__(kThreads) void cache_tables_kernel(const TablesParams p) {
  __shared__ Pair part[kWaves];
  __shared__ uint32_t tok0[kThreads], page0[kThreads];
  __shared__ int32_t ctx_s[kThreads];
  const int tid = threadIdx.x, grid = (int)gridDim.x, wg = (int)blockIdx.x;
  const int64_t cnt = *p.free_count;
  const int32_t count = (int32_t)(cnt < 0 ? 0 : cnt < p.capacity ? cnt : p.capacity);
  Pair carry = {0, 0};
  uint32_t lacking = 0;  // workgroup 0: this thread's requests' tokens without a slot

  // the page of rank k, or -1; a page that no 31-bit slot reaches counts as none
  auto page_of_rank = [&](uint32_t k) -> int32_t {
    if (k >= (uint32_t)count) return -1;
    return p.free_blocks[count - 1 - (int32_t)k];
  };
  auto usable = [&](int32_t page) { return page >= 0 && page < (INT32_MAX >> p.bshift); };

  for (int r0 = 0; r0 < p.R; r0 += kThreads) {
    const int rows = imin32(kThreads, p.R - r0), r = r0 + tid;
    const bool mine = tid < rows;
    const int32_t ctx = mine ? length(p.ctx[r]) : 0, n = mine ? length(p.fresh[r]) : 0;
    const int32_t have = imin32((ctx + p.bs - 1) >> p.bshift, p.width);
    const int32_t need = imin32((ctx + n + p.bs - 1) >> p.bshift, p.width);
    const int32_t take = need - have;
    Pair total;
    const Pair incl = scan({(uint32_t)n, (uint32_t)take}, total, part);
    const uint32_t t_first = sat(carry.tok, incl.tok - (uint32_t)n);   // exact below the limit
    const uint32_t k_first = sat(carry.page, incl.page - (uint32_t)take);
    tok0[tid] = t_first;
    page0[tid] = k_first;
    ctx_s[tid] = ctx;
    __syncthreads();

    if (wg == 0 && mine) {
      p.cu[r] = (int32_t)t_first;
      p.lens[r] = ctx + n;
      // tokens inside max_tokens; of these, those in the page that had begun and in pages that were there to take
      const int32_t in = t_first >= (uint32_t)p.T ? 0 : imin32(n, p.T - (int32_t)t_first);
      const int32_t begun = imin32(n, imax32(0, (have << p.bshift) - ctx));
      const bool ok = begun > 0 && usable(p.table[(int64_t)r * p.table_stride + (ctx >> p.bshift)]);
      const int32_t avail = k_first >= (uint32_t)count ? 0 : imin32(take, count - (int32_t)k_first);
      const int32_t slotted = (ok ? imin32(begun, in) : 0) + imin32(imax32(0, in - begun), avail << p.bshift);
      lacking = sat(lacking, (uint32_t)(n - slotted));
    }

    // the pages taken: by rank
    const uint32_t k_end = sat(carry.page, total.page);
    for (uint32_t k = carry.page + wg * kThreads + tid; k < k_end; k += (uint32_t)grid * kThreads) {
      const int i = row_of(page0, rows, k);
      const int32_t col = imin32((ctx_s[i] + p.bs - 1) >> p.bshift, p.width) + (int32_t)(k - page0[i]);
      if (col < p.width) p.table[(int64_t)(r0 + i) * p.table_stride + col] = page_of_rank(k);
    }
    // the tokens: a slot each
    const uint32_t t_end = (uint32_t)imin32((int32_t)sat(carry.tok, total.tok), p.T);
    for (uint32_t t = carry.tok + wg * kThreads + tid; t < t_end; t += (uint32_t)grid * kThreads) {
      const int i = row_of(tok0, rows, t);
      const int32_t c = ctx_s[i], pos = c + (int32_t)(t - tok0[i]);
      const int32_t first = (c + p.bs - 1) >> p.bshift, at = pos >> p.bshift;
      int32_t page = -1;
      if (at < p.width)
        page = at < first ? p.table[(int64_t)(r0 + i) * p.table_stride + at] : page_of_rank(page0[i] + (uint32_t)(at - first));
      p.slots[t] = usable(page) ? (page << p.bshift) + (pos & (p.bs - 1)) : -1;
      p.positions[t] = pos;
    }
    carry = {sat(carry.tok, total.tok), k_end};
    __syncthreads();
  }

  for (uint32_t t = carry.tok + wg * kThreads + tid; t < (uint32_t)p.T; t += (uint32_t)grid * kThreads)
    p.slots[t] = p.positions[t] = -1;
  if (wg == 0) {
    Pair total;
    scan({lacking, 0}, total, part);
    if (tid == 0) {
      p.cu[p.R] = (int32_t)carry.tok;
      *p.missing = (int32_t)total.tok;
      *p.free_left = imax32(0, count - (int32_t)carry.page);
    }
  }
}

struct ReleaseParams {
  int32_t* table;
  int64_t table_stride;
  int32_t R, width, bs, bshift;
  const int32_t* ctx;
  const uint8_t* finished;
  int32_t* free_blocks;
  const int32_t* free_count;
  int64_t capacity;
  int32_t* free_left;
};

// One workgroup: pages are counted and pushed a request at a time per wavefront,
// the requests' places on the stack by a prefix sum of how many each gives back.
__global__ __launch_bounds__(kThreads) void cache_release_kernel(const ReleaseParams p) {
  __shared__ Pair part[kWaves];
  __shared__ uint32_t at_s[kThreads], n_s[kThreads];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t cnt = *p.free_count;
  const int32_t count = (int32_t)(cnt < 0 ? 0 : cnt < p.capacity ? cnt : p.capacity);
  uint32_t carry = (uint32_t)count;
  for (int r0 = 0; r0 < p.R; r0 += kThreads) {
    const int rows = imin32(kThreads, p.R - r0);
    for (int i = wave; i < rows; i += kWaves) {  // how many pages each row gives back
      const int r = r0 + i;
      int n = 0;
      if (p.finished[r]) {
        const int32_t have = imin32((length(p.ctx[r]) + p.bs - 1) >> p.bshift, p.width);
        for (int c = lane; c < have; c += 64) n += p.table[(int64_t)r * p.table_stride + c] >= 0;
      }
#pragma unroll
      for (int d = 32; d > 0; d >>= 1) n += __shfl_xor(n, d);
      if (lane == 0) n_s[i] = (uint32_t)n;
    }
    __syncthreads();
    Pair total;
    const uint32_t mine = tid < rows ? n_s[tid] : 0;
    const Pair incl = scan({0, mine}, total, part);
    at_s[tid] = sat(carry, incl.page - mine);
    __syncthreads();
    for (int i = wave; i < rows; i += kWaves) {
      const int r = r0 + i;
      if (!p.finished[r]) continue;
      const int32_t have = imin32((length(p.ctx[r]) + p.bs - 1) >> p.bshift, p.width);
      uint32_t at = at_s[i];
      for (int c0 = 0; c0 < p.width; c0 += 64) {
        const int c = c0 + lane;
        int32_t* e = p.table + (int64_t)r * p.table_stride + c;
        const int32_t page = c < have ? *e : -1;
        const uint64_t bits = __ballot(page >= 0);
        const uint32_t to = at + (uint32_t)__popcll(bits & ((1ull << lane) - 1));
        if (page >= 0 && (int64_t)to < p.capacity) p.free_blocks[to] = page;
        at += (uint32_t)__popcll(bits);
        if (c < p.width) *e = -1;
      }
    }
    carry = sat(carry, total.page);
    __syncthreads();
  }
  if (tid == 0) *p.free_left = (int32_t)((int64_t)carry < p.capacity ? (int64_t)carry : p.capacity);
}

bool aligned4(const void* ptr) { return ((uintptr_t)ptr & 3u) == 0; }

int block_shift(int32_t bs) {
  for (int s = 4; s <= 8; ++s)
    if (bs == 1 << s) return s;
  return -1;
}

int launched(hipError_t err) {
  if (err != hipSuccess) return (int)err;
  err = hipGetLastError();
  return err == hipSuccess ? CHIA_ATTN_OK : (int)err;
}

constexpr int64_t kMaxRows = (int64_t)1 << 24, kMaxEntries = (int64_t)1 << 28;

}  // namespace
}  // namespace chia

using namespace chia;

extern "C" int chia_cache_tables(const chia_cache_tables_args* a, void* stream) {
  if (!a) return CHIA_ATTN_ERR_NULL;
  if (a->struct_size != sizeof(chia_cache_tables_args)) return CHIA_ATTN_ERR_STRUCT;
  for (int i = 0; i < 8; ++i)
    if (a->reserved[i] != 0) return CHIA_ATTN_ERR_STRUCT;
  const int shift = block_shift(a->block_size);
  if (shift < 0 || a->requests < 1 || a->requests > kMaxRows || a->width < 1 || a->table_stride < a->width ||
      a->width > (kMaxEntries >> shift) || a->free_capacity < 0 || a->free_capacity > kMaxEntries ||
      a->max_tokens < 0 || a->max_tokens > kMaxEntries)
    return CHIA_ATTN_ERR_SHAPE;
  if (!a->block_tables || !a->context_lens || !a->new_lens || !a->free_count || (!a->free_blocks && a->free_capacity) ||
      ((!a->slots || !a->positions) && a->max_tokens) || !a->cu_seqlens || !a->seq_lens || !a->free_left || !a->missing)
    return CHIA_ATTN_ERR_NULL;
  for (const void* ptr : {(const void*)a->block_tables, (const void*)a->context_lens, (const void*)a->new_lens,
                          (const void*)a->free_blocks, (const void*)a->free_count, (const void*)a->slots,
                          (const void*)a->positions, (const void*)a->cu_seqlens, (const void*)a->seq_lens,
                          (const void*)a->free_left, (const void*)a->missing})
    if (!aligned4(ptr)) return CHIA_ATTN_ERR_ALIGN;
  TablesParams p{a->block_tables, a->table_stride, (int32_t)a->requests, (int32_t)a->width, a->block_size, shift,
                 a->context_lens, a->new_lens, a->free_blocks, a->free_count, a->free_capacity, (int32_t)a->max_tokens,
                 a->slots, a->positions, a->cu_seqlens, a->seq_lens, a->free_left, a->missing};
  const int64_t items = a->max_tokens > a->requests ? a->max_tokens : a->requests;
  const int64_t wgs = (items + kThreads - 1) / kThreads;
  cache_tables_kernel<<<dim3((unsigned)(wgs < 1 ? 1 : wgs < 256 ? wgs : 256)), dim3(kThreads), 0, (hipStream_t)stream>>>(p);
  return launched(hipSuccess);
}

extern "C" int chia_cache_release(const chia_cache_release_args* a, void* stream) {
  if (!a) return CHIA_ATTN_ERR_NULL;
  if (a->struct_size != sizeof(chia_cache_release_args)) return CHIA_ATTN_ERR_STRUCT;
  for (int i = 0; i < 8; ++i)
    if (a->reserved[i] != 0) return CHIA_ATTN_ERR_STRUCT;
  const int shift = block_shift(a->block_size);
  if (shift < 0 || a->requests < 1 || a->requests > kMaxRows || a->width < 1 || a->table_stride < a->width ||
      a->width > (kMaxEntries >> shift) || a->free_capacity < 1 || a->free_capacity > kMaxEntries)
    return CHIA_ATTN_ERR_SHAPE;
  if (!a->block_tables || !a->context_lens || !a->finished || !a->free_blocks || !a->free_count || !a->free_left)
    return CHIA_ATTN_ERR_NULL;
  for (const void* ptr : {(const void*)a->block_tables, (const void*)a->context_lens, (const void*)a->free_blocks,
                          (const void*)a->free_count, (const void*)a->free_left})
    if (!aligned4(ptr)) return CHIA_ATTN_ERR_ALIGN;
  ReleaseParams p{a->block_tables, a->table_stride, (int32_t)a->requests, (int32_t)a->width, a->block_size, shift,
                  a->context_lens, a->finished, a->free_blocks, a->free_count, a->free_capacity, a->free_left};
  cache_release_kernel<<<dim3(1), dim3(kThreads), 0, (hipStream_t)stream>>>(p);
  return launched(hipSuccess);
}
