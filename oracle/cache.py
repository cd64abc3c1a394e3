"""The paged 8-bit K/V cache in plain loops and float64 (CPU).  TEST INFRASTRUCTURE ONLY.

The reference has no cache; these restate the operators' definitions:

  tables_ref   page tables, slots and positions of one serving step
  write_ref    new tokens rounded into their slots, one power-of-two scale per page and head
  attend_ref   attention of each request's newest tokens over its pages, and for each
               output the quantities from which a test derives its tolerance
"""
from __future__ import annotations

import math

import torch

TOP = {torch.float8_e4m3fn: 448.0, torch.float8_e5m2: 57344.0}
_FORMAT = {torch.float8_e4m3fn: (-6, 3), torch.float8_e5m2: (-14, 2)}  # least normal exponent, fraction bits


def tables_ref(table, ctx, new, free, count, bs, max_tokens):
    """(table, slots, positions, cu, lens, left, missing) as lists."""
    width = len(table[0])
    table, stack = [list(r) for r in table], list(free[:max(0, min(count, len(free)))])
    slots, positions, cu, lens, missing = [], [], [0], [], 0
    for row, c, n in zip(table, ctx, new):
        c, n = max(c, 0), max(n, 0)
        for p in range(-(-c // bs), min(-(-(c + n) // bs), width)):
            row[p] = stack.pop() if stack else -1
        for p in range(c, c + n):
            page = row[p // bs] if p // bs < width else -1
            slots.append(page * bs + p % bs if page >= 0 else -1)
            positions.append(p)
            missing += page < 0 or len(slots) > max_tokens
        cu.append(cu[-1] + n)
        lens.append(c + n)
    pad = [-1] * max_tokens
    return table, (slots + pad)[:max_tokens], (positions + pad)[:max_tokens], cu, lens, len(stack), missing


def need_scale(amax: float, dtype) -> float:
    """The least 2^e >= 2^-126 with amax <= 2^e times the format's largest value."""
    e = -126
    if amax > 0:
        e = max(e, math.ceil(math.log2(amax / TOP[dtype])))
        while e > -126 and amax <= 2.0 ** (e - 1) * TOP[dtype]:  # log2's own rounding
            e -= 1
        while amax > 2.0 ** e * TOP[dtype]:
            e += 1
    return 2.0 ** e


def round_code(x: torch.Tensor, dtype) -> torch.Tensor:
    """float64 to the nearest value of the format, ties to even, infinities to the largest."""
    least, bits = _FORMAT[dtype]
    y = x.double()
    exponent = (torch.frexp(y)[1] - 1).clamp(min=least).double()
    step = torch.exp2(exponent - bits)
    r = (torch.round(y / step) * step).clamp(-TOP[dtype], TOP[dtype])
    return torch.where(torch.isnan(y), y, torch.where(torch.isinf(y), torch.sign(y) * TOP[dtype], r))


def write_ref(x, codes, scale, slots):
    """codes (float64 values) and scale (float64) after writing x [T, H, D] into `slots`;
    codes [pages, H, bs, D] float8, scale [pages, H] float32, all on the CPU."""
    dtype, (pages, H, bs, _) = codes.dtype, codes.shape
    out, sc = codes.float().double(), scale.double().clone()
    x = x.double()
    slots = [s if 0 <= s < pages * bs else -1 for s in slots]
    t = 0
    while t < len(slots):
        if slots[t] < 0:
            t += 1
            continue
        u = t + 1
        while u < len(slots) and slots[u] == slots[u - 1] + 1 and slots[u] % bs:
            u += 1
        page, off = divmod(slots[t], bs)
        for h in range(H):
            a = x[t:u, h].abs()
            need = need_scale(float(torch.where(torch.isfinite(a), a, 0.0).max()), dtype)
            old = float(sc[page, h]) if off else 0.0
            new = max(need, old)
            if off and new != old:
                out[page, h, :off] = round_code(out[page, h, :off] * (old / new), dtype)
            out[page, h, off:off + u - t] = round_code(x[t:u, h] / new, dtype)
            sc[page, h] = new
        t = u
    return out, sc


def row_mask(S, i, *, causal, window, dilation, block, prefix):
    """Keys 0 .. S - 1 that a query at position i sees, by the mask's definition."""
    if i < 0:
        return torch.zeros(S, dtype=torch.bool)
    j = torch.arange(S)
    d = i - j
    ok = (d >= 0) if causal else torch.ones(S, dtype=torch.bool)
    if window:
        ok = ok & ((d < window) if causal else (d.abs() < window))
    if dilation > 1:
        ok = ok & (d % dilation == 0)
    if block:
        ok = ok & (j // block == i // block)
    if prefix:
        ok = ok | (j < prefix)
    return ok


def attend_ref(q, k_codes, v_codes, k_scale, v_scale, table, lens, cu, *, norm="softmax", causal=True, window=0,
               dilation=1, block=0, prefix=0, scale=None, head_scale=None, alibi_slopes=None, softcap=0.0, bias=0.0,
               post_scale=1.0):
    """(o, size, slack) float64 [T, H, D] for q [T, H, D] (NaN rows where no request has a query).

    size = sum_j p_j |v_j| (over sum_j p_j for softmax): what a relative error of every
    weight moves an output by.  slack: what the fp32 arithmetic of the scores may move it
    by; with s_j off by at most e_j, softmax and sigmoid weights move by e_j relative, ReLU
    weights by e_j.
    """
    T, H, D = q.shape
    pages, hkv, bs, _ = k_codes.shape
    kc, vc, qd = k_codes.float().double(), v_codes.float().double(), q.double()
    o = torch.full((T, H, D), float("nan"), dtype=torch.float64)
    size, slack = torch.zeros_like(o), torch.zeros_like(o)
    sc = 1 / math.sqrt(D) if scale is None else scale
    for r, S in enumerate(lens):
        S = max(0, min(S, table.shape[1] * bs))
        n = cu[r + 1] - cu[r]
        ids = table[r, :-(-S // bs)].long()
        there = (ids >= 0) & (ids < pages)
        at = torch.where(there, ids, 0)
        exists = there.repeat_interleave(bs)[:S]
        for h in range(H):
            g = h // (H // hkv)
            k = (kc[at, g] * k_scale.double()[at, g][:, None, None]).reshape(-1, D)[:S]
            v = (vc[at, g] * v_scale.double()[at, g][:, None, None]).reshape(-1, D)[:S]
            for x in range(n):
                i = S - n + x
                see = row_mask(S, i, causal=causal, window=window, dilation=dilation, block=block, prefix=prefix) & exists
                t = cu[r] + x
                kv, vv = k[see], v[see]
                o[t, h] = 0
                if kv.shape[0] == 0:
                    continue
                c = sc * (1.0 if head_scale is None else float(head_scale[h]))
                s = kv @ qd[t, h] * c
                # fp32 sums of D exact products, then a handful of roundings of the score
                e = c * (kv.abs() @ qd[t, h].abs()) * (D + 8) * 2.0 ** -24
                if alibi_slopes is not None:
                    rel = float(alibi_slopes[h]) * (torch.arange(S)[see] - i).double()
                    s, e = s + rel, e + rel.abs() * 2.0 ** -23
                if softcap:
                    s = torch.tanh(s / softcap) * softcap
                    e = e + softcap * 2.0 ** -20  # one approximate exponential and reciprocal, times the cap
                e = e + (s.abs() + abs(bias)) * 2.0 ** -21 + 2.0 ** -20
                if norm == "softmax":
                    p = torch.exp(s - s.max())
                    p = p / p.sum()
                    f = 1.0
                elif norm == "sigmoid":
                    p, f = torch.sigmoid(s + bias), post_scale
                else:
                    p, f = torch.relu(s), post_scale
                o[t, h] = p @ vv * f
                size[t, h] = p @ vv.abs() * abs(f)
                w = p * e if norm != "relu" else e
                slack[t, h] = (2 if norm == "softmax" else 1) * ((w @ vv.abs()) * abs(f))
                if norm == "softmax":
                    slack[t, h] += float((p * e).sum()) * size[t, h]
    return o, size, slack
