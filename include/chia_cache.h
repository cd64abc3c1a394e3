/*
 * chia_cache.h -- C ABI of the paged 8-bit K/V cache of the MI355X (gfx950)
 * attention library: block tables built on the GPU, cache writes and attention
 * over the cache (libchia_attn.so).
 *
 * The cache holds K and V codes in OCP float8 (e4m3fn or e5m2) in pages of
 * block_size tokens, [num_blocks, kv_heads, block_size, head_dim] with
 * arbitrary strides and a unit head_dim stride, and float32 scales
 * [num_blocks, kv_heads]: a value is code * scale of its page and head.
 * block_tables[r][n] is the page of request r's tokens n * block_size and up;
 * the slot of a token is page * block_size + its place in the page.
 *
 * Every entry point only enqueues kernels on `stream`, allocates nothing, keeps
 * no state and returns enum chia_attn_status (chia_attn.h) or a hipError_t.
 * Lengths, tables, slots and scales are device memory that the host does not
 * read.  Whatever they hold, the kernels read and write inside the buffers they
 * are given: a slot or page outside the cache is skipped.
 *
 * No counterpart in the reference (JoshiP-commits/CHIA_proj), whose kernels take
 * one fixed shape with as many keys as queries.
 */
#ifndef CHIA_CACHE_H
#define CHIA_CACHE_H

#include <stdint.h>

#include "chia_attn.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Grow every request by new_lens[r] tokens.  With ctx = context_lens[r] and
 * have = ceil(ctx / block_size), the pages from `have` to
 * min(ceil((ctx + new) / block_size), width) - 1 come off the free list, a stack
 * whose last entry goes first: request 0's pages first, each request's in order.
 * Where it is empty the table gets -1.  The new tokens, packed request by
 * request, get their positions and slots (-1: none).  Calling it again with the
 * same inputs writes the same values. */
typedef struct chia_cache_tables_args {
  uint32_t struct_size;        /* sizeof(chia_cache_tables_args) */
  int32_t block_size;          /* tokens per page: a power of two, 16 .. 256 */
  int32_t* block_tables;       /* [requests, width], entries `have` and up written */
  int64_t table_stride;        /* elements between rows, >= width */
  int64_t requests, width;     /* >= 1 */
  const int32_t* context_lens; /* [requests]; negative counts as 0 (so does new_lens) */
  const int32_t* new_lens;     /* [requests] */
  const int32_t* free_blocks;  /* [free_capacity] pages; NULL only with capacity 0 */
  const int32_t* free_count;   /* [1] how many of them there are */
  int64_t free_capacity;
  int64_t max_tokens;          /* entries of slots and positions; those behind the new tokens get -1 */
  int32_t* slots;              /* [max_tokens] */
  int32_t* positions;          /* [max_tokens] */
  int32_t* cu_seqlens;         /* [requests + 1] offsets of the packed new tokens */
  int32_t* seq_lens;           /* [requests] ctx + new */
  int32_t* free_left;          /* [1] what is left of free_count; another buffer than that */
  int32_t* missing;            /* [1] new tokens without a slot: the free list was empty, the table too
                                  narrow or without the page that had begun, or max_tokens too few */
  int32_t reserved[8];         /* must be zero */
} chia_cache_tables_args;

int chia_cache_tables(const chia_cache_tables_args* args, void* stream);

/* Give back the pages of every request r with finished[r] != 0: those of its
 * first ceil(context_lens[r] / block_size) table entries that are >= 0 go onto
 * the stack, request by request, in order, as far as its capacity goes, and its
 * table row becomes -1. */
typedef struct chia_cache_release_args {
  uint32_t struct_size;        /* sizeof(chia_cache_release_args) */
  int32_t block_size;
  int32_t* block_tables;       /* [requests, width] */
  int64_t table_stride;
  int64_t requests, width;
  const int32_t* context_lens; /* [requests] */
  const uint8_t* finished;     /* [requests] */
  int32_t* free_blocks;        /* [free_capacity], written from free_count on */
  const int32_t* free_count;   /* [1] */
  int64_t free_capacity;
  int32_t* free_left;          /* [1] the new count; may be free_count itself */
  int32_t reserved[8];         /* must be zero */
} chia_cache_release_args;

int chia_cache_release(const chia_cache_release_args* args, void* stream);

/* Round K and V of `tokens` new tokens into their slots.  The tokens of one page
 * have to be consecutive, in slot order; a page written from a place > 0 on keeps
 * what lies before that place and one written from its first place starts anew.
 * The scale of a page and head becomes the least power of two 2^e >= 2^-126 with
 * which the largest finite |value| of the new tokens fits the format, or stays
 * what it was if that is more and the page had begun; codes kept from before are
 * then multiplied by old / new scale.  Rounding is to nearest, ties to even;
 * infinities become the largest value, NaN stays NaN.  Tokens whose slot is
 * outside [0, num_blocks * block_size) are skipped.  Two tokens with one slot, or
 * a page whose tokens are apart, leave that page's values unspecified. */
typedef struct chia_cache_write_args {
  uint32_t struct_size;        /* sizeof(chia_cache_write_args) */
  uint32_t format;             /* CHIA_ATTN_FP8_E4M3 or CHIA_ATTN_FP8_E5M2 */
  const void* k;               /* bf16 [tokens, kv_heads, head_dim] */
  const void* v;
  void* k_cache;               /* float8 [num_blocks, kv_heads, block_size, head_dim] */
  void* v_cache;
  float* k_scale;              /* [num_blocks, kv_heads] */
  float* v_scale;
  const int32_t* slots;        /* [tokens] */
  int64_t tokens, kv_heads, head_dim, num_blocks;
  int64_t k_stride[2], v_stride[2];               /* token, head, in elements (multiples of 8) */
  int64_t k_cache_stride[3], v_cache_stride[3];   /* block, head, token (multiples of 16) */
  int64_t k_scale_stride[2], v_scale_stride[2];   /* block, head */
  int32_t block_size;
  int32_t reserved[7];         /* must be zero */
} chia_cache_write_args;

int chia_cache_write(const chia_cache_write_args* args, void* stream);

/* Attention of each request's newest tokens over its cached ones.  `attn`
 * describes the call as for chia_attn_fwd: q and o are packed bf16 [T, heads,
 * head_dim] (stride[1] head, stride[2] token, stride[0] unused), k and v the
 * caches (strides block, head, token, multiples of 16), batch the requests,
 * kv_heads, the mask, the score and the normaliser.  cu_seqlens NULL: one query
 * per request, T = batch; otherwise request r's queries are cu_seqlens[r] ..
 * cu_seqlens[r + 1] - 1 and lie at the last positions of its seq_lens[r] tokens.
 * seqlen is the longest request (a hint: it sizes the launch, longer ones are
 * computed all the same).  seq_order is ignored.
 * Key j of a request is seen if the mask has it and j < seq_lens[r], its page is
 * in the cache and the query's position is not negative; a query that sees no
 * key gives 0.  Rows of o behind the last query stay as they are.  An infinity or
 * NaN in a key or value that a query does not see does not reach it. */
typedef struct chia_cache_attn_args {
  uint32_t struct_size;        /* sizeof(chia_cache_attn_args) */
  uint32_t format;             /* of both caches */
  const chia_attn_args* attn;
  const float* k_scale;        /* [num_blocks, kv_heads] */
  const float* v_scale;
  int64_t k_scale_stride[2], v_scale_stride[2];   /* block, head */
  const int32_t* block_tables; /* [batch, width] */
  int64_t table_stride, width; /* table_stride 0: one row for all */
  const int32_t* seq_lens;     /* [batch] */
  int64_t num_blocks;
  int64_t queries;             /* T: rows of q and o */
  int64_t max_query;           /* most queries of one request (a hint, as seqlen) */
  int32_t block_size;
  int32_t reserved0;           /* must be zero */
  void* workspace;             /* chia_cache_attn_workspace_size bytes, 16-byte aligned */
  int64_t workspace_bytes;
  int32_t reserved[8];         /* must be zero */
} chia_cache_attn_args;

/* Bytes of workspace chia_cache_attn needs (0 where no request's keys are
 * split); negative: an argument error.  Reads sizes only. */
int64_t chia_cache_attn_workspace_size(const chia_cache_attn_args* args);

int chia_cache_attn(const chia_cache_attn_args* args, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* CHIA_CACHE_H */
