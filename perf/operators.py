"""Timed cases of the paged 8-bit K/V cache: what a serving loop does with it, step by step.

Three operators, in the order in which a step calls them:

  tables   extend_block_tables: every request grows by some tokens; the pages that it
           lacks come off the free list, and each new token gets its slot
  write    write_cache: the new tokens' K and V are rounded to float8 into their slots,
           with one scale for each page and head
  attend   attention_cache: each request's newest tokens attend over its pages

The cache: codes [pages, heads, page size, D] in float8 e4m3 or e5m2 and scales float32
[pages, heads], for K and for V; a value is code * scale.  A scale that write_cache sets
is the least power of two 2^e >= 2^-126 with which the largest value ever written to the
page since its first slot fits the format.

Lengths go from one token to 131072, page sizes from 16 to 128, heads and channels are
those of the attention cases (4 to 32 heads, 64 and 128 channels).
"""
from __future__ import annotations

import math
import random

import torch

own = False

_DEV = "cuda"
_TYPES = {"e4m3": (torch.float8_e4m3fn, 448.0, 9), "e5m2": (torch.float8_e5m2, 57344.0, 16)}  # largest = 0.875 2^x


def listed():
    return [
        # one decoding step's bookkeeping for a full batch: latency of a single launch
        dict(name="tables_decode_r256", op="tables", R=256, lo=1, hi=8192, new=1, bs=64, lens_seed=1),
        # admission of a batch of long prompts: a hundred thousand slots
        dict(name="tables_prefill_r48", op="tables", R=48, lo=0, hi=1500, new=4096, bs=16, lens_seed=2),
        # one decoding step's K and V: every token ends in a page that others began
        dict(name="write_decode_r128", op="write", R=128, lo=1, hi=4096, new=1, bs=64, Hkv=8, D=128, fmt="e4m3",
             lens_seed=3),
        # prompts of a mid-size batch, heads of 64 channels
        dict(name="write_prefill_r7_d64", op="write", R=7, lo=0, hi=900, new=2600, bs=64, Hkv=16, D=64, fmt="e4m3",
             lens_seed=4),
        # long prompts in small pages, the wider range of e5m2
        dict(name="write_prefill_r20_e5m2", op="write", R=20, lo=0, hi=5000, new=4096, bs=16, Hkv=8, D=128,
             fmt="e5m2", lens_seed=5),
        # one user's short chat, one token: latency of a layer
        dict(name="decode_r1_s512", op="attend", R=1, lo=512, hi=512, n=1, bs=16, H=8, Hkv=8, D=64, fmt="e4m3",
             lens_seed=6),
        # an ordinary batch of decoding requests of unequal length, grouped heads
        dict(name="decode_r64_gqa", op="attend", R=64, lo=97, hi=8192, n=1, bs=64, H=32, Hkv=8, D=128, fmt="e4m3",
             lens_seed=7),
        # two very long documents: few rows, the keys split over the chip
        dict(name="decode_r2_s131072", op="attend", R=2, lo=100003, hi=131072, n=1, bs=128, H=32, Hkv=8, D=128,
             fmt="e4m3", lens_seed=8),
        # a sliding-window layer with capped scores over long requests
        dict(name="decode_r32_window_softcap", op="attend", R=32, lo=700, hi=32768, n=1, bs=64, H=16, Hkv=8, D=128,
             fmt="e4m3", window=1024, softcap=50.0, lens_seed=9),
        # one K/V head per query head, ALiBi, e5m2, small pages
        dict(name="decode_r16_mha_alibi_e5m2", op="attend", R=16, lo=33, hi=4096, n=1, bs=16, H=16, Hkv=16, D=64,
             fmt="e5m2", alibi=True, lens_seed=10),
        # five drafted tokens of each request are verified in one pass
        dict(name="verify_r16_n5", op="attend", R=16, lo=300, hi=4096, n=5, bs=64, H=32, Hkv=8, D=128, fmt="e4m3",
             lens_seed=11),
        # a chunk of two long prompts behind what is in the cache: bound by the products
        dict(name="chunk_r2_n1000", op="attend", R=2, lo=9001, hi=16000, n=1000, bs=64, H=32, Hkv=8, D=128,
             fmt="e4m3", lens_seed=12),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of the listed ones' ranges."""
    op = rng.choice(("tables", "write", "attend", "attend", "attend"))
    case = dict(op=op, bs=rng.choice((16, 32, 64, 128)), lens_seed=rng.randrange(1 << 30))
    if op == "tables":
        case.update(R=_log_int(rng, 1, 512), lo=0, hi=_log_int(rng, 1, 16384), new=_log_int(rng, 1, 4096))
        case["new"] = max(1, min(case["new"], 131072 // case["R"]))
        return case
    case.update(D=rng.choice((64, 128)), Hkv=rng.choice((1, 2, 4, 8, 16)), fmt=rng.choice(("e4m3", "e4m3", "e5m2")))
    if op == "write":
        case.update(R=_log_int(rng, 1, 256), lo=0, hi=_log_int(rng, 1, 8192), new=_log_int(rng, 1, 4096))
        while case["R"] * case["new"] * case["Hkv"] * case["D"] > 40_000_000:
            case["new"] = case["new"] * 4 // 5 + 1 if case["new"] > 4 else 1
            case["R"] = max(1, case["R"] * 4 // 5)
        while case["R"] * (case["hi"] + case["new"]) * case["Hkv"] * case["D"] > 400_000_000:
            case["hi"] = max(1, case["hi"] * 4 // 5)
            case["R"] = max(1, case["R"] * 4 // 5)
        return case
    case["H"] = case["Hkv"] * rng.choice((1, 2, 4, 8)) if case["Hkv"] <= 4 else case["Hkv"] * rng.choice((1, 2, 4))
    case["n"] = rng.choice((1, 1, 1, rng.randint(2, 8), _log_int(rng, 16, 1000)))
    case["R"], case["hi"] = _log_int(rng, 1, 128), _log_int(rng, 16, 65536)
    case["lo"] = max(1, case["hi"] // rng.choice((1, 2, 16)))
    kind = rng.choice(("causal", "causal", "window", "softcap", "alibi", "prefix", "sigmoid", "block", "dilation"))
    if kind == "window":
        case["window"] = rng.choice((129, 256, 1024))
    elif kind == "softcap":
        case["softcap"] = rng.choice((30.0, 50.0))
    elif kind == "alibi":
        case["alibi"] = True
    elif kind == "prefix":
        case["prefix"], case["window"] = rng.choice((100, 256)), 512
    elif kind == "sigmoid":
        case["norm"] = "sigmoid"
    elif kind == "block":
        case["block"] = rng.choice((200, 256, 512))
    elif kind == "dilation":
        case["dilation"] = rng.choice((2, 4))
    while True:  # no dearer than the listed ones, and the plain form's memory stays small
        tokens = case["R"] * (case["hi"] + case["n"])
        if (tokens * case["Hkv"] * case["D"] <= 200_000_000 and tokens * case["n"] * case["H"] <= 500_000_000):
            return case
        if case["R"] > 1:
            case["R"] = max(1, case["R"] * 4 // 5)
        elif case["n"] > 8:
            case["n"] = case["n"] * 4 // 5
        else:
            case["hi"] = case["hi"] * 4 // 5
            case["lo"] = min(case["lo"], case["hi"])


# ---- what a case is -----------------------------------------------------------

def _lens(case):
    """Tokens in the cache before the step, and new ones, of every request (attend: the
    length with the newest tokens, and how many those are)."""
    rng = random.Random(case["lens_seed"])
    R, lo, hi = case["R"], case["lo"], case["hi"]
    old = [hi if r == 0 else rng.randint(lo, hi) for r in range(R)]
    if case["op"] == "attend":
        n = [case["n"] if r == 0 or case["n"] < 8 else rng.randint(case["n"] // 2, case["n"]) for r in range(R)]
        return [x + m for x, m in zip(old, n)], n
    n = [case["new"] if r == 0 or case["new"] < 8 else rng.randint(0, case["new"]) for r in range(R)]
    return old, n


def _pages(tokens, bs):
    return -(-tokens // bs)


def _mask(case):
    return dict(window=case.get("window", 0), block=case.get("block", 0), prefix=case.get("prefix", 0),
                dilation=case.get("dilation", 1))


def _seen(case, i):
    """Keys that a token at position i sees."""
    m = _mask(case)
    lo = max(0, i - m["window"] + 1) if m["window"] else 0
    if m["block"]:
        lo = max(lo, i // m["block"] * m["block"])
    n = (i - lo) // m["dilation"] + 1
    if m["prefix"]:
        p = min(m["prefix"], i + 1)
        n = p + max(0, i - max(lo, p) + 1)
    return n


def work(case):
    """Every input read once and every output written once."""
    old, new = _lens(case)
    bs, R = case["bs"], case["R"]
    if case["op"] == "tables":
        T = sum(new)
        taken = sum(_pages(o + n, bs) - _pages(o, bs) for o, n in zip(old, new))
        # lengths in; offsets and lengths out; the pages taken in and out; a slot and a position of each token
        return {"bytes": 4 * (2 * R + 2 * R + 2 * taken + 2 * T), "flops": 0}
    Hkv, D = case["Hkv"], case["D"]
    if case["op"] == "write":
        T = sum(new)
        runs = sum(_pages(o + n, bs) - o // bs for o, n in zip(old, new) if n)
        return {"bytes": T * (2 * Hkv * D * (2 + 1) + 4) + 2 * 4 * runs * Hkv, "flops": 4 * T * Hkv * D}
    H = case["H"]
    keys = rows = flops = 0
    for length, n in zip(old, new):
        # K and V rows that some row of the request sees, each once
        first, last = length - n, length - 1
        m = _mask(case)
        if n == 1:
            keys += _seen(case, last)
        else:
            lo = max(0, first - m["window"] + 1) if m["window"] else 0
            if m["block"]:
                lo = max(lo, first // m["block"] * m["block"])
            keys += length - lo + min(m["prefix"], lo)
        rows += n
        flops += 4 * H * D * sum(_seen(case, i) for i in range(first, length))
    return {"bytes": 2 * keys * Hkv * D + 2 * 4 * Hkv * (keys // bs) + 4 * (keys // bs) + 2 * 2 * rows * H * D,
            "flops": flops}


# ---- inputs -------------------------------------------------------------------

def _need(amax, fmt):
    """The least 2^e >= 2^-126 with amax <= 2^e * (largest value of the format)."""
    m, e = torch.frexp(amax)
    x = (e - _TYPES[fmt][2] + (m > 0.875)).clamp(min=-126)
    return torch.ldexp(torch.ones((), device=amax.device), x)


def _values(g, tokens, Hkv, D, spread):
    """K- or V-like rows: heads of unequal size, some channels several times the others
    (`spread`: K has such channels), now and then a token that stands out."""
    x = torch.randn(tokens, Hkv, D, generator=g, device=_DEV)
    head = torch.exp(0.4 * torch.randn(1, Hkv, 1, generator=g, device=_DEV))
    chan = torch.exp(spread * torch.randn(1, Hkv, D, generator=g, device=_DEV))
    tok = 1 + 3 * (torch.rand(tokens, 1, 1, generator=g, device=_DEV) > 0.98)
    return (x * head * chan * tok).to(torch.bfloat16)


def _filled(g, pages, bs, Hkv, D, fmt, spread):
    """Codes [pages, Hkv, bs, D] and scales [pages, Hkv] of a cache that is in use."""
    dt, top, _ = _TYPES[fmt]
    x = _values(g, pages * bs, Hkv, D, spread).view(pages, bs, Hkv, D).transpose(1, 2)
    scale = _need(x.abs().amax((2, 3)).float(), fmt)
    return (x / scale[:, :, None, None]).to(dt).contiguous(), scale


def _tables(rng_seed, old, bs, width, pages):
    """[R, width] page numbers in no order, -1 behind each request's last, and the pages left."""
    free = list(range(pages))
    random.Random(rng_seed).shuffle(free)
    rows = []
    for n in old:
        have = _pages(n, bs)
        rows.append(free[:have] + [-1] * (width - have))
        del free[:have]
    return torch.tensor(rows, dtype=torch.int32).to(_DEV), free


def prepare(case, seed):
    g = torch.Generator(_DEV).manual_seed(seed)
    old, new = _lens(case)
    bs, R, op = case["bs"], case["R"], case["op"]
    i32 = lambda x: torch.tensor(x, dtype=torch.int32).to(_DEV)  # noqa: E731
    if op == "attend":
        width = max(_pages(n, bs) for n in old)
        pages = sum(_pages(n, bs) for n in old) + 3
        table, _ = _tables(seed, old, bs, width, pages)
        H, Hkv, D = case["H"], case["Hkv"], case["D"]
        kc, ks = _filled(g, pages, bs, Hkv, D, case["fmt"], 0.5)
        vc, vs = _filled(g, pages, bs, Hkv, D, case["fmt"], 0.1)
        T = sum(new)
        q = torch.randn(T, H, D, generator=g, device=_DEV).to(torch.bfloat16)
        cu = [0]
        for n in new:
            cu.append(cu[-1] + n)
        slopes = None
        if case.get("alibi"):
            slopes = torch.tensor([2.0 ** (-8.0 * (h + 1) / H) for h in range(H)]).to(_DEV)
        return dict(case=case, q=q, kc=kc, vc=vc, ks=ks, vs=vs, table=table, lens=i32(old), cu=i32(cu),
                    max_n=max(new), max_len=max(old), slopes=slopes, bias=-math.log(max(old)))
    width = max(_pages(o + n, bs) for o, n in zip(old, new)) + 1
    pages = sum(_pages(o + n, bs) for o, n in zip(old, new)) + 5
    table, free = _tables(seed, old, bs, width, pages)
    T = sum(new)
    if op == "tables":
        return dict(case=case, table=table, old=i32(old), new=i32(new), free=i32(free), count=i32([len(free)]),
                    max_tokens=T + 16)  # the step's tensors are a little larger than its tokens
    slots = []
    at = 0
    for r, row in enumerate(table.tolist()):
        have = _pages(old[r], bs)
        more = _pages(old[r] + new[r], bs) - have
        row = row[:have] + free[at:at + more]
        at += more
        slots.extend(row[p // bs] * bs + p % bs for p in range(old[r], old[r] + new[r]))
    Hkv, D = case["Hkv"], case["D"]
    kc, ks = _filled(g, pages, bs, Hkv, D, case["fmt"], 0.5)
    vc, vs = _filled(g, pages, bs, Hkv, D, case["fmt"], 0.1)
    return dict(case=case, k=_values(g, T, Hkv, D, 0.5), v=_values(g, T, Hkv, D, 0.1), kc=kc, vc=vc, ks=ks, vs=vs,
                slots=i32(slots))


# ---- one pass -----------------------------------------------------------------

def run(state):
    op = state["case"]["op"]
    if op == "tables":
        return _run_tables(state)
    if op == "write":
        return _run_write(state)
    return _run_attend(state)


def _run_tables(s):
    bs = s["case"]["bs"]
    if own:
        import chia_proj_amd as lib

        step = lib.extend_block_tables(s["table"], s["old"], s["new"], s["free"], s["count"], block_size=bs,
                                       max_tokens=s["max_tokens"])
        return dict(table=s["table"], slots=step.slots, positions=step.positions, cu=step.cu_seqlens,
                    lens=step.seq_lens, count=step.free_count, missing=step.missing)
    old, new, table, free = s["old"].long(), s["new"].long(), s["table"].long(), s["free"].long()
    R, width = table.shape
    have = (old + bs - 1) // bs
    take = (old + new + bs - 1) // bs - have
    start = torch.cumsum(take, 0) - take  # pages taken by the requests before
    col = torch.arange(width, device=_DEV)[None]
    k = start[:, None] + col - have[:, None]  # this entry's rank among the pages taken
    fresh = (col >= have[:, None]) & (col < (have + take)[:, None])
    at = s["count"].long() - 1 - k  # the free list is a stack: its last entry goes first
    page = torch.where(at >= 0, free[at.clamp(0, free.numel() - 1)], -1)
    table = torch.where(fresh, page, table)
    cu = torch.zeros(R + 1, dtype=torch.int64, device=_DEV)
    cu[1:] = torch.cumsum(new, 0)
    t = torch.arange(s["max_tokens"], device=_DEV)
    row = torch.searchsorted(cu[1:], t, right=True)
    inside = row < R
    row = row.clamp(max=R - 1)
    pos = old[row] + t - cu[row]
    page = table[row, torch.where(inside, pos // bs, 0)]
    slots = torch.where(inside & (page >= 0), page * bs + pos % bs, -1)
    i32 = torch.int32
    return dict(table=table.to(i32), slots=slots.to(i32), positions=torch.where(inside, pos, -1).to(i32), cu=cu.to(i32),
                lens=(old + new).to(i32), count=(s["count"].long() - take.sum()).clamp(min=0).to(i32),
                missing=(inside & (slots < 0)).sum().reshape(1).to(i32))


def _write_plain(x, codes, scale, slots, fmt):
    dt, top, _ = _TYPES[fmt]
    _, Hkv, bs, D = codes.shape
    x = x.float()
    pages, at = torch.unique(slots.long() // bs, return_inverse=True)  # the pages written to, and each token's
    off, n = slots.long() % bs, pages.numel()
    a = torch.where(torch.isfinite(x), x.abs(), 0.0).amax(-1)
    first = torch.full((n,), bs, device=_DEV).scatter_reduce(0, at, off, "amin")
    need = torch.zeros(n, Hkv, device=_DEV).scatter_reduce(0, at[:, None].expand(-1, Hkv), _need(a, fmt), "amax")
    begun = (first > 0)[:, None]
    old = scale[pages]
    new = torch.maximum(need, torch.where(begun, old, 0.0))
    ratio = torch.where(begun, old / new, 1.0)[:, :, None, None]
    kept = (torch.arange(bs, device=_DEV)[None] < first[:, None])[:, None, :, None]
    held = codes.view(torch.uint8)[pages].view(dt).float()
    held = torch.where(kept, held * ratio, held).to(dt)
    mine = (x / new[at][:, :, None]).clamp(-top, top).to(dt)
    held.view(torch.uint8).transpose(1, 2)[at, off] = mine.view(torch.uint8)
    codes.view(torch.uint8)[pages] = held.view(torch.uint8)
    scale[pages] = new
    return codes, scale


def _run_write(s):
    if own:
        import chia_proj_amd as lib

        lib.write_cache(s["k"], s["v"], s["kc"], s["vc"], s["ks"], s["vs"], s["slots"])
        return dict(k=s["kc"], v=s["vc"], k_scale=s["ks"], v_scale=s["vs"])
    kc, ks = _write_plain(s["k"], s["kc"], s["ks"], s["slots"], s["case"]["fmt"])
    vc, vs = _write_plain(s["v"], s["vc"], s["vs"], s["slots"], s["case"]["fmt"])
    return dict(k=kc, v=vc, k_scale=ks, v_scale=vs)


def _gathered(codes, scale, table):
    """[R, Hkv, keys, D] float32 values of every request's pages."""
    t = table.long().clamp(min=0)
    x = codes.view(torch.uint8)[t].view(codes.dtype).float() * scale[t][..., None, None]
    R, P, Hkv, bs, D = x.shape
    return x.transpose(1, 2).reshape(R, Hkv, P * bs, D)


def _run_attend(s):
    c = s["case"]
    if own:
        import chia_proj_amd as lib

        return lib.attention_cache(s["q"], s["kc"], s["vc"], s["ks"], s["vs"], s["table"], s["lens"],
                                   None if c["n"] == 1 else s["cu"], max_query=s["max_n"], max_seqlen=s["max_len"],
                                   norm=c.get("norm", "softmax"), causal=True, softcap=c.get("softcap", 0.0),
                                   alibi_slopes=s["slopes"], bias=s["bias"] if c.get("norm") == "sigmoid" else 0.0,
                                   **_mask(c))
    m = _mask(c)
    H, Hkv, D = c["H"], c["Hkv"], c["D"]
    G, lens, cu = H // Hkv, s["lens"].long(), s["cu"].long()
    n = cu[1:] - cu[:-1]
    k, v = _gathered(s["kc"], s["ks"], s["table"]), _gathered(s["vc"], s["vs"], s["table"])
    R, _, L, _ = k.shape
    N = s["max_n"]
    t = torch.arange(N, device=_DEV)[None]  # [R, N]: the request's t-th new token
    there = t < n[:, None]
    row = (cu[:-1, None] + t).clamp(max=s["q"].shape[0] - 1)
    q = s["q"].float()[row]  # [R, N, H, D]
    q = q.view(R, N, Hkv, G, D).permute(0, 2, 3, 1, 4).reshape(R, Hkv, G * N, D)
    x = (torch.matmul(q, k.transpose(-1, -2)) / math.sqrt(D)).view(R, Hkv, G, N, L)
    i = (lens - n)[:, None] + t  # positions
    j = torch.arange(L, device=_DEV)
    d = i[:, :, None] - j
    if s["slopes"] is not None:
        x = x - s["slopes"].view(1, Hkv, G, 1, 1) * d[:, None, None].float()
    if c.get("softcap"):
        x = c["softcap"] * torch.tanh(x / c["softcap"])
    ok = d >= 0
    if m["window"]:
        ok = ok & (d < m["window"])
    if m["dilation"] > 1:
        ok = ok & (d % m["dilation"] == 0)
    if m["block"]:
        ok = ok & (i[:, :, None] // m["block"] == j // m["block"])
    if m["prefix"]:
        ok = ok | (j < m["prefix"])
    ok = (ok & (j < lens[:, None, None]))[:, None, None]  # [R, 1, 1, N, L]
    if c.get("norm") == "sigmoid":
        p = torch.where(ok, 1 / (1 + torch.exp(-(x + s["bias"]))), 0.0)
    else:
        x = torch.where(ok, x, -torch.inf)
        p = torch.exp(x - x.amax(-1, keepdim=True))
        p = p / p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(R, Hkv, G * N, L), v).view(R, Hkv, G, N, D).permute(0, 3, 1, 2, 4).reshape(R, N, H, D)
    return o[there].to(torch.bfloat16)


# ---- the definition in 64 bits --------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    return {"tables": _exact_tables, "write": _exact_write, "attend": _exact_attend}[case["op"]](case, s)


def _exact_tables(case, s):
    bs = case["bs"]
    table, free = s["table"].tolist(), s["free"].tolist()[:int(s["count"])]
    slots, positions, cu = [], [], [0]
    missing = 0
    for row, o, n in zip(table, s["old"].tolist(), s["new"].tolist()):
        for p in range(o, o + n):
            if p % bs == 0:
                row[p // bs] = free.pop() if free else -1
            page = row[p // bs]
            slots.append(page * bs + p % bs if page >= 0 else -1)
            positions.append(p)
            missing += page < 0
        cu.append(cu[-1] + n)
    pad = [-1] * (s["max_tokens"] - len(slots))
    t = lambda x: torch.tensor(x)  # noqa: E731
    return dict(table=t(table), slots=t(slots + pad), positions=t(positions + pad), cu=t(cu),
                lens=s["old"].cpu() + s["new"].cpu(), count=t([len(free)]), missing=t([missing]))


def _rounded(x, fmt):
    """float64 values to the format's nearest (least normal 2^-6 with 3 bits of fraction, 2^-14 with 2)."""
    least, bits = {"e4m3": (-6, 3), "e5m2": (-14, 2)}[fmt]
    exponent = (torch.frexp(x)[1] - 1).clamp(min=least).double()
    step = torch.exp2(exponent - bits)
    top = _TYPES[fmt][1]
    return (torch.round(x / step) * step).clamp(-top, top)


def _exact_write(case, s):
    """The rounding to 8 bits is part of the definition: to nearest, ties to even."""
    bs, top = case["bs"], _TYPES[case["fmt"]][1]
    slots = s["slots"].tolist()
    runs, t = [], 0
    while t < len(slots):
        u = t + 1
        while u < len(slots) and slots[u] == slots[u - 1] + 1 and slots[u] % bs:
            u += 1
        runs.append((t, u, slots[t] // bs, slots[t] % bs))
        t = u
    out = {}
    for name, x, codes, scale in (("k", s["k"], s["kc"], s["ks"]), ("v", s["v"], s["vc"], s["vs"])):
        x, codes, scale = x.double().cpu(), codes.float().cpu().double(), scale.double().cpu()
        for a, b, page, off in runs:
            old = scale[page].clone()
            largest = x[a:b].abs().amax((0, 2))
            new = torch.tensor([2.0 ** max(-126, math.ceil(math.log2(m / top))) if m else 2.0 ** -126
                                for m in largest.tolist()], dtype=torch.float64)
            new = torch.maximum(new, old) if off else new
            codes[page, :, :off] = _rounded(codes[page, :, :off] * (old / new)[:, None, None], case["fmt"])
            codes[page, :, off:off + b - a] = _rounded(x[a:b].transpose(0, 1) / new[:, None, None], case["fmt"])
            scale[page] = new
        out[name], out[name + "_scale"] = codes, scale
    return out


def _exact_attend(case, s):
    m, H, Hkv, D = _mask(case), case["H"], case["Hkv"], case["D"]
    lens, cu, out = s["lens"].tolist(), s["cu"].tolist(), []
    bs = case["bs"]
    for r, length in enumerate(lens):
        pages = s["table"][r, :_pages(length, bs)].long()
        k, v = ((c[pages].double() if c.dtype.itemsize > 1 else c.view(torch.uint8)[pages].view(c.dtype).double())
                * sc[pages].double()[..., None, None] for c, sc in ((s["kc"], s["ks"]), (s["vc"], s["vs"])))
        k, v = (y.transpose(0, 1).reshape(Hkv, -1, D)[:, :length] for y in (k, v))
        q = s["q"][cu[r]:cu[r + 1]].double()
        n = q.shape[0]
        i = torch.arange(length - n, length, device=_DEV)[:, None]
        j = torch.arange(length, device=_DEV)[None]
        seen = i >= j
        if m["window"]:
            seen &= i - j < m["window"]
        if m["dilation"] > 1:
            seen &= (i - j) % m["dilation"] == 0
        if m["block"]:
            seen &= torch.div(i, m["block"], rounding_mode="floor") == torch.div(j, m["block"], rounding_mode="floor")
        if m["prefix"]:
            seen |= j < m["prefix"]
        o = torch.empty(n, H, D, dtype=torch.float64, device=_DEV)
        for h in range(H):
            x = q[:, h] @ k[h * Hkv // H].t() / math.sqrt(D)
            if s["slopes"] is not None:
                x = x + s["slopes"][h].double() * (j - i)
            if case.get("softcap"):
                x = torch.tanh(x / case["softcap"]) * case["softcap"]
            if case.get("norm") == "sigmoid":
                p = torch.sigmoid(x + s["bias"]) * seen
            else:
                p = torch.softmax(x.masked_fill(~seen, float("-inf")), -1)
            o[:, h] = p @ v[h * Hkv // H]
        out.append(o)
    return torch.cat(out)
