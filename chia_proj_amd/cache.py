"""Serving over a paged 8-bit K/V cache.

A serving step calls, in this order,

    step = extend_block_tables(tables, lens, new_lens, free_blocks, free_count, block_size=64, max_tokens=T)
    write_cache(k, v, k_cache, v_cache, k_scale, v_scale, step.slots)
    o = attention_cache(q, k_cache, v_cache, k_scale, v_scale, tables, step.seq_lens, step.cu_seqlens)

and release_block_tables() for requests that have ended.  Lengths, tables and
slots stay on the GPU: no call waits for it or copies from it, so a step can be
captured into a HIP graph.  The cache is ordinary tensors that the caller owns:

    k_cache, v_cache   torch.float8_e4m3fn or torch.float8_e5m2 [pages, H_kv, block_size, D]
    k_scale, v_scale   float32 [pages, H_kv]; a value is code * scale
    tables             int32 [requests, width], the page of each block_size tokens

The reference has no counterpart: its kernels take one fixed shape with as many
keys as queries (extra_bench.py:8-22).
"""
from __future__ import annotations

import ctypes
from typing import NamedTuple, Optional

import torch

from . import _lib
from .attention import (FP8_FORMATS, PerHead, _args_cache, _ARGS_CACHE_MAX, _check_params, _current_stream, _head_key,
                        _layout_ok_packed, _per_head_vector, make_args)

BLOCK_SIZES = (16, 32, 64, 128, 256)


class CacheStep(NamedTuple):
    """What extend_block_tables() returns: int32 tensors on the GPU."""

    slots: torch.Tensor       # [max_tokens] each new token's page * block_size + place; -1: none
    positions: torch.Tensor   # [max_tokens] its position in its request; -1 behind the last token
    cu_seqlens: torch.Tensor  # [requests + 1] offsets of the packed new tokens
    seq_lens: torch.Tensor    # [requests] lengths with the new tokens
    free_count: torch.Tensor  # [1] pages left on the free list
    missing: torch.Tensor     # [1] new tokens without a slot


def _vector(name: str, t, device, shape, dtype=torch.int32) -> torch.Tensor:
    if not isinstance(t, torch.Tensor) or t.dtype != dtype:
        raise TypeError(f"{name} must be a {dtype} tensor, got {getattr(t, 'dtype', type(t).__name__)}")
    if t.dim() != len(shape) or any(s is not None and s != n for s, n in zip(shape, t.shape)):
        raise ValueError(f"{name} must have shape {tuple('*' if s is None else s for s in shape)}, got {tuple(t.shape)}")
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, expected {device}")
    return t


def _contiguous(name: str, t: torch.Tensor) -> torch.Tensor:
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    return t


def _check_table(block_tables, block_size) -> torch.device:
    if not isinstance(block_tables, torch.Tensor) or block_tables.dtype != torch.int32:
        raise TypeError(f"block_tables must be an int32 tensor, got "
                        f"{getattr(block_tables, 'dtype', type(block_tables).__name__)}")
    if block_tables.dim() != 2 or block_tables.shape[1] < 1 or (block_tables.shape[0] > 0 and block_tables.stride(1) != 1):
        raise ValueError(f"block_tables must be [requests, width] with unit last stride, got {tuple(block_tables.shape)}")
    if block_tables.device.type != "cuda":
        raise ValueError(f"block_tables must be on a GPU device, got {block_tables.device}")
    if block_size not in BLOCK_SIZES:
        raise ValueError(f"block_size must be one of {BLOCK_SIZES}, got {block_size}")
    return block_tables.device


def _row_stride(t: torch.Tensor) -> int:
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def extend_block_tables(block_tables: torch.Tensor, context_lens: torch.Tensor, new_lens: torch.Tensor,
                        free_blocks: torch.Tensor, free_count: torch.Tensor, *, block_size: int,
                        max_tokens: int) -> CacheStep:
    """Grow every request by its new tokens: the pages that it lacks come off the free list.

    block_tables int32 [requests, width] is written in place: request r, with
    context_lens[r] tokens in the cache, gets pages for new_lens[r] more (int32
    [requests]; negative counts as 0).  free_blocks int32 [n] is a stack of page
    numbers with free_count int32 [1] of them; its last page goes first.  It is not
    changed: pass the result's free_count to the next call.  Where it runs out, or
    the table is too narrow, table entries and slots are -1 and `missing` counts the
    tokens without a slot.  The new tokens are numbered request by request;
    max_tokens is the size of slots and positions, -1 behind the last token.
    """
    if torch.compiler.is_compiling():
        return CacheStep(*torch.ops.chia_attn.extend_block_tables(block_tables, context_lens, new_lens, free_blocks,
                                                                  free_count, block_size, max_tokens))
    # as in attention(): a call with the shapes and layouts of an earlier one reuses
    # its validated argument struct; only the pointers are new
    try:
        key = ("cache_tables", block_size, max_tokens) + _meta(block_tables, context_lens, new_lens, free_blocks,
                                                               free_count)
        cache = _args_cache()
        entry = cache.get(key)
    except (AttributeError, TypeError):
        entry = key = None
    if entry is None:
        device = _check_table(block_tables, block_size)
        R = block_tables.shape[0]
        for name, t, n in (("context_lens", context_lens, R), ("new_lens", new_lens, R),
                           ("free_blocks", free_blocks, None), ("free_count", free_count, 1)):
            _contiguous(name, _vector(name, t, device, (n,)))
        if max_tokens < 0:
            raise ValueError(f"max_tokens must be >= 0, got {max_tokens}")
        T = int(max_tokens)
        a = _lib.CacheTablesArgs(block_size=block_size, table_stride=_row_stride(block_tables), requests=R,
                                 width=block_tables.shape[1], free_capacity=free_blocks.shape[0], max_tokens=T)
        entry = (a, device, T, R, (T, T, R + 1, R, 1, 1))
        if key is not None and R > 0:
            _remember(cache, key, entry)
    a, device, T, R, sizes = entry
    # one allocation: slots, positions, offsets, lengths, the two counts
    flat = torch.empty(2 * T + 2 * R + 3, dtype=torch.int32, device=device)
    step = CacheStep._make(flat.split_with_sizes(sizes))
    if R == 0:
        flat.fill_(-1)
        step.cu_seqlens.zero_()
        step.missing.zero_()
        step.free_count.copy_(free_count.clamp(0, free_blocks.shape[0]))
        return step
    at = flat.data_ptr()
    a.block_tables, a.context_lens, a.new_lens = block_tables.data_ptr(), context_lens.data_ptr(), new_lens.data_ptr()
    a.free_blocks, a.free_count = free_blocks.data_ptr(), free_count.data_ptr()
    a.slots, a.positions, a.cu_seqlens = at, at + 4 * T, at + 8 * T
    at += 8 * T + 4 * (R + 1)
    a.seq_lens, a.free_left, a.missing = at, at + 4 * R, at + 4 * R + 4
    _launch(_lib.cache_tables, a, block_tables)
    return step


def release_block_tables(block_tables: torch.Tensor, context_lens: torch.Tensor, finished: torch.Tensor,
                         free_blocks: torch.Tensor, free_count: torch.Tensor, *, block_size: int) -> torch.Tensor:
    """Give back the pages of the requests that `finished` (bool [requests]) marks.

    The pages of such a request's first context_lens[r] tokens go onto the stack
    free_blocks (in place, from free_count on, as far as it has room), its table row
    becomes -1.  Returns the new count, int32 [1].
    """
    if torch.compiler.is_compiling():
        return torch.ops.chia_attn.release_block_tables(block_tables, context_lens, finished, free_blocks, free_count,
                                                        block_size)
    device = _check_table(block_tables, block_size)
    R = block_tables.shape[0]
    for name, t, n in (("context_lens", context_lens, R), ("free_blocks", free_blocks, None), ("free_count", free_count, 1)):
        _contiguous(name, _vector(name, t, device, (n,)))
    _contiguous("finished", _vector("finished", finished, device, (R,), torch.bool))
    if R == 0 or free_blocks.shape[0] == 0:
        return free_count.clamp(0, free_blocks.shape[0])
    left = torch.empty(1, dtype=torch.int32, device=device)
    a = _lib.CacheReleaseArgs(block_size=block_size, block_tables=block_tables.data_ptr(),
                              table_stride=_row_stride(block_tables), requests=R, width=block_tables.shape[1],
                              context_lens=context_lens.data_ptr(), finished=finished.data_ptr(),
                              free_blocks=free_blocks.data_ptr(), free_count=free_count.data_ptr(),
                              free_capacity=free_blocks.shape[0], free_left=left.data_ptr())
    _launch(_lib.cache_release, a, block_tables)
    return left


def _check_cache(k_cache, v_cache, k_scale, v_scale):
    """Host checks of the cache's tensors; (pages, H_kv, block_size, D)."""
    for name, t in (("k_cache", k_cache), ("v_cache", v_cache)):
        if not isinstance(t, torch.Tensor) or t.dtype not in FP8_FORMATS:
            raise TypeError(f"{name} must be a torch.float8_e4m3fn or torch.float8_e5m2 tensor, got "
                            f"{getattr(t, 'dtype', type(t).__name__)}")
        if t.dim() != 4 or t.shape != k_cache.shape or t.dtype != k_cache.dtype or t.device != k_cache.device:
            raise ValueError(f"k_cache and v_cache must be [pages, H_kv, block_size, D] tensors of one shape, type and "
                             f"device, got {tuple(k_cache.shape)}, {tuple(t.shape)}")
        if t.stride(3) != 1 or any(s % 16 for s in t.stride()[:3]) or t.data_ptr() % 16:
            raise ValueError(f"{name} must have unit last stride, strides that are multiples of 16 and 16-byte alignment")
        if min(t.stride()[:3]) < 0 or t.stride(2) >= 1 << 26:
            raise ValueError(f"{name}'s token stride must be below 2^26 elements, got {t.stride(2)}")
    pages, heads, bs, D = k_cache.shape
    if pages < 1 or heads < 1 or bs not in BLOCK_SIZES or D not in (64, 128):
        raise ValueError(f"k_cache must be [pages, H_kv, block_size, D] with block_size in {BLOCK_SIZES} and D 64 or "
                         f"128, got {tuple(k_cache.shape)}")
    if pages * bs >= 1 << 31:
        raise ValueError("at most 2^31 - 1 slots")
    if k_cache.device.type != "cuda":
        raise ValueError(f"the cache must be on a GPU device, got {k_cache.device}")
    for name, t in (("k_scale", k_scale), ("v_scale", v_scale)):
        _vector(name, t, k_cache.device, (pages, heads), torch.float32)
    return pages, heads, bs, D


def _meta(*tensors):
    """What a cached call is recognised by: shapes, types, devices and layouts."""
    return tuple([(t.shape, t.dtype, t.device, t.stride()) for t in tensors])


def _laid_out(t: torch.Tensor) -> torch.Tensor:
    """t, or a contiguous and aligned copy where the kernels cannot read it as it lies."""
    return t if _layout_ok_packed(t) else t.clone(memory_format=torch.contiguous_format)


_get_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)


def _launch(call, args, t: torch.Tensor) -> None:
    """call(args, stream) on t's device and its current stream."""
    if _get_device() == t.get_device():
        call(args, _current_stream(t))
    else:
        with torch.cuda.device(t.device):
            call(args, _current_stream(t))


def _remember(cache, key, entry) -> None:
    cache[key] = entry
    if len(cache) > _ARGS_CACHE_MAX:
        cache.popitem(last=False)


def write_cache(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor,
                v_scale: torch.Tensor, slots: torch.Tensor) -> None:
    """Round new tokens' k and v (bf16 [T, H_kv, D]) into their slots (int32 [T]), in place.

    The scale of a page and head is the least power of two 2^e >= 2^-126 with which
    the largest finite magnitude written since the page's first slot fits the format
    (448 for e4m3, 57344 for e5m2): writing from a place > 0 on keeps what lies
    before it, rescaled where the scale grows, and writing the first place starts
    the page anew.  Rounding is to nearest, ties to even; infinities become the
    largest value, NaN stays.  Slots outside the cache (-1) are skipped.

    The tokens of one page must be consecutive in k, v and slots, in slot order, as
    extend_block_tables() numbers them; a slot that occurs twice, or a page whose
    tokens are apart, leaves that page's values unspecified.
    """
    if torch.compiler.is_compiling():
        torch.ops.chia_attn.write_cache(k, v, k_cache, v_cache, k_scale, v_scale, slots)
        return
    if torch.is_grad_enabled() and any(isinstance(t, torch.Tensor) and t.requires_grad for t in (k, v)):
        raise ValueError("write_cache is forward only: k and v must not require grad")
    try:
        key = ("cache_write",) + _meta(k, v, k_cache, v_cache, k_scale, v_scale, slots)
        args = _args_cache()
        a = args.get(key)
    except (AttributeError, TypeError):
        a = key = None
    if a is not None:
        ptrs = (k.data_ptr(), v.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr())
        if not (ptrs[0] | ptrs[1] | ptrs[2] | ptrs[3]) & 15:
            a.k, a.v, a.k_cache, a.v_cache = ptrs
            a.k_scale, a.v_scale, a.slots = k_scale.data_ptr(), v_scale.data_ptr(), slots.data_ptr()
            _launch(_lib.cache_write, a, k_cache)
            return
    pages, heads, bs, D = _check_cache(k_cache, v_cache, k_scale, v_scale)
    _contiguous("slots", _vector("slots", slots, k_cache.device, (None,)))
    T = slots.shape[0]
    for name, t in (("k", k), ("v", v)):
        if not isinstance(t, torch.Tensor) or t.dtype != torch.bfloat16:
            raise TypeError(f"{name} must be a bfloat16 tensor, got {getattr(t, 'dtype', type(t).__name__)}")
        if tuple(t.shape) != (T, heads, D):
            raise ValueError(f"{name} must be [T, H_kv, D] = {(T, heads, D)}, got {tuple(t.shape)}")
        if t.device != k_cache.device:
            raise ValueError(f"{name} is on {t.device}, the cache on {k_cache.device}")
    if T == 0:
        return
    k_, v_ = _laid_out(k), _laid_out(v)
    a = _lib.CacheWriteArgs(format=FP8_FORMATS[k_cache.dtype][0], k=k_.data_ptr(), v=v_.data_ptr(),
                            k_cache=k_cache.data_ptr(), v_cache=v_cache.data_ptr(), k_scale=k_scale.data_ptr(),
                            v_scale=v_scale.data_ptr(), slots=slots.data_ptr(), tokens=T, kv_heads=heads, head_dim=D,
                            num_blocks=pages, block_size=bs)
    a.k_stride[:], a.v_stride[:] = k_.stride()[:2], v_.stride()[:2]
    a.k_cache_stride[:], a.v_cache_stride[:] = k_cache.stride()[:3], v_cache.stride()[:3]
    a.k_scale_stride[:], a.v_scale_stride[:] = k_scale.stride(), v_scale.stride()
    _launch(_lib.cache_write, a, k_cache)
    if key is not None and k_ is k and v_ is v:
        _remember(args, key, a)


def attention_cache(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor,
                    v_scale: torch.Tensor, block_tables: torch.Tensor, seq_lens: torch.Tensor,
                    cu_seqlens: Optional[torch.Tensor] = None, *, max_query: Optional[int] = None,
                    max_seqlen: Optional[int] = None, norm: str = "softmax", causal: bool = True, window: int = 0,
                    dilation: int = 1, block: int = 0, prefix: int = 0, scale: Optional[float] = None,
                    head_scale: PerHead = None, alibi_slopes: PerHead = None, softcap: float = 0.0, bias: float = 0.0,
                    post_scale: float = 1.0, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """attention() of each request's newest tokens over its tokens in the cache.

    q bf16 [T, H, D], H_kv dividing H; seq_lens int32 [requests] counts each
    request's tokens in the cache, the newest included (write_cache() first).
    Without cu_seqlens every request has one query, T = requests.  With cu_seqlens
    (int32 [requests + 1]) request r's queries are q[cu_seqlens[r]:cu_seqlens[r + 1]],
    its last tokens in order; rows behind the last are left as they are in `out`
    (without `out`: unset).  Mask, score and normaliser are attention()'s, with each
    token's position in its request; keys >= seq_lens[r] and pages outside the cache
    are not seen, and a query that sees no key gives 0.

    max_query (default T) and max_seqlen (default the table's width) bound a request's
    queries and tokens; they size the launch, and exceeding them costs time, not
    results.  Returns o bf16 [T, H, D].  Forward only.
    """
    if isinstance(q, torch.Tensor) and q.requires_grad and torch.is_grad_enabled():
        raise ValueError("attention_cache is forward only: q must not require grad")
    if torch.compiler.is_compiling():
        if out is not None:
            raise ValueError("out= is not supported under torch.compile")
        from .library import call_cache_attn

        p = dict(norm=norm, causal=causal, window=window, dilation=dilation, block=block, prefix=prefix, scale=scale,
                 head_scale=head_scale, alibi_slopes=alibi_slopes, softcap=softcap, bias=bias, post_scale=post_scale)
        for name, positive in (("head_scale", True), ("alibi_slopes", False)):
            p[name] = _per_head_vector(p[name], q.shape[1], q.device, name, positive=positive, cache=False)
        return call_cache_attn(q, k_cache, v_cache, k_scale, v_scale, block_tables, seq_lens, cu_seqlens, max_query,
                               max_seqlen, p)
    # as in attention(): a call with the shapes, layouts and parameters of an
    # earlier one reuses its validated argument structs; only the pointers are new
    try:
        key = ("cache_attn", None if cu_seqlens is None else (cu_seqlens.shape, cu_seqlens.dtype, cu_seqlens.device,
                                                              cu_seqlens.stride()),
               None if out is None else (out.shape, out.dtype, out.device, out.stride()), max_query, max_seqlen, norm,
               causal, window, dilation, block, prefix, scale, softcap, bias, post_scale, _head_key(head_scale),
               _head_key(alibi_slopes)) + _meta(q, k_cache, v_cache, k_scale, v_scale, block_tables, seq_lens)
        cache = _args_cache()
        entry = cache.get(key)
    except (AttributeError, TypeError):
        entry = key = None
    if entry is not None:
        c, a, nbytes, hs, sl = entry
        o = torch.empty(q.shape, dtype=torch.bfloat16, device=q.device) if out is None else out
        ptrs = (q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), o.data_ptr())
        if not (ptrs[0] | ptrs[1] | ptrs[2] | ptrs[3]) & 15:
            a.q, a.k, a.v, a.o = ptrs
            if hs is not None:
                a.head_scale = (head_scale if isinstance(head_scale, torch.Tensor) and head_scale.is_cuda
                                else hs).data_ptr()
            if sl is not None:
                a.alibi_slopes = (alibi_slopes if isinstance(alibi_slopes, torch.Tensor) and alibi_slopes.is_cuda
                                  else sl).data_ptr()
            if cu_seqlens is not None:
                a.cu_seqlens = cu_seqlens.data_ptr()
            c.k_scale, c.v_scale = k_scale.data_ptr(), v_scale.data_ptr()
            c.block_tables, c.seq_lens = block_tables.data_ptr(), seq_lens.data_ptr()
            if nbytes:
                ws = torch.empty(nbytes, dtype=torch.uint8, device=q.device)
                c.workspace = ws.data_ptr()
            _launch(_lib.cache_attn, c, q)
            return o

    pages, hkv, bs, D = _check_cache(k_cache, v_cache, k_scale, v_scale)
    device = _check_table(block_tables, bs)
    if device != k_cache.device:
        raise ValueError(f"block_tables is on {device}, the cache on {k_cache.device}")
    R, width = block_tables.shape
    if not isinstance(q, torch.Tensor) or q.dtype != torch.bfloat16:
        raise TypeError(f"q must be a bfloat16 tensor, got {getattr(q, 'dtype', type(q).__name__)}")
    if q.dim() != 3 or q.shape[2] != D or q.shape[1] < 1 or q.shape[1] % hkv != 0:
        raise ValueError(f"q must be [T, H, D] with H_kv = {hkv} dividing H and D = {D}, got {tuple(q.shape)}")
    if q.device != device:
        raise ValueError(f"q is on {q.device}, the cache on {device}")
    T, H, _ = q.shape
    _contiguous("seq_lens", _vector("seq_lens", seq_lens, device, (R,)))
    if cu_seqlens is not None:
        _contiguous("cu_seqlens", _vector("cu_seqlens", cu_seqlens, device, (R + 1,)))
    elif T != R:
        raise ValueError(f"without cu_seqlens every request has one query: q has {T} rows for {R} requests")
    sc = _check_params(D, norm, window, dilation, block, prefix, scale, softcap)
    most_q = T if max_query is None else int(max_query)
    most_s = width * bs if max_seqlen is None else int(max_seqlen)
    if (T > 0 and most_q < 1) or most_s < 1:
        raise ValueError(f"max_query and max_seqlen must be >= 1, got {max_query}, {max_seqlen}")
    if out is not None and (out.shape != q.shape or out.dtype != torch.bfloat16 or out.device != device
                            or not _layout_ok_packed(out)):
        raise ValueError("out must be a bf16 tensor of q's shape on q's device with unit last stride, strides that are "
                         "multiples of 8 and 16-byte alignment")
    hs = _per_head_vector(head_scale, H, device, "head_scale", positive=True)
    sl = _per_head_vector(alibi_slopes, H, device, "alibi_slopes", positive=False)
    o = torch.empty(q.shape, dtype=torch.bfloat16, device=device) if out is None else out
    if T == 0 or R == 0:
        return o
    q_ = _laid_out(q)
    a = make_args(batch=R, heads=H, seqlen=min(most_s, width * bs), head_dim=D, norm=norm, causal=causal, window=window,
                  dilation=dilation, block=block, prefix=prefix, scale=sc, softcap=softcap, bias=bias,
                  post_scale=post_scale)
    a.q, a.k, a.v, a.o = q_.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), o.data_ptr()
    a.kv_heads = hkv
    a.q_stride[:], a.o_stride[:] = (0, q_.stride(1), q_.stride(0)), (0, o.stride(1), o.stride(0))
    a.k_stride[:], a.v_stride[:] = k_cache.stride()[:3], v_cache.stride()[:3]
    a.head_scale = hs.data_ptr() if hs is not None else None
    a.alibi_slopes = sl.data_ptr() if sl is not None else None
    a.cu_seqlens = cu_seqlens.data_ptr() if cu_seqlens is not None else None
    c = _lib.CacheAttnArgs(format=FP8_FORMATS[k_cache.dtype][0], attn=ctypes.pointer(a), k_scale=k_scale.data_ptr(),
                           v_scale=v_scale.data_ptr(), block_tables=block_tables.data_ptr(),
                           table_stride=_row_stride(block_tables), width=width, seq_lens=seq_lens.data_ptr(),
                           num_blocks=pages, queries=T, max_query=min(most_q, T), block_size=bs)
    c.k_scale_stride[:], c.v_scale_stride[:] = k_scale.stride(), v_scale.stride()
    c.workspace_bytes = nbytes = _lib.cache_attn_workspace_size(c)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None
    c.workspace = ws.data_ptr() if nbytes else None
    _launch(_lib.cache_attn, c, q)
    if key is not None and q_ is q:
        _remember(cache, key, (c, a, nbytes, hs, sl))
    return o
