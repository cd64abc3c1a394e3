"""Every row tile and workgroup shape of the cache attention, against the float64 oracle.

The launch takes 16 rows of a K/V head with four or eight wavefronts, tiles of 32 rows,
or, for prompts of much work, 128 rows (another kernel).  What it takes follows from
bounds that the host knows; here they are chosen (a wide table, bounds that are not
tight) so that small problems, which the oracle can compute, reach every one.
test_which_kernel_runs checks that they do.
"""
import pytest
import torch

import chia_proj_amd as lib
from test_gpu_cache import DEV, E4, E5, VARIANTS, Case, _i32, _say, oc

pytestmark = pytest.mark.gpu
WIDE = 1 << 14  # table columns: the host then reckons with requests of that many pages


def _wide(c):
    """The same requests in a wide table, pages behind their last not in the cache."""
    t = torch.full((c.table.shape[0], WIDE), -1, dtype=torch.int32)
    t[:, :c.table.shape[1]] = c.table
    dev = c.device()
    dev[5] = t.to(DEV)
    return dev


def _prompt(c, **kw):
    return lib.attention_cache(*_wide(c), _i32(c.cu).to(DEV), max_query=4096, **kw)


def _kernels(fn):
    fn()
    torch.cuda.synchronize()
    with torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CUDA]) as prof:
        fn()
        torch.cuda.synchronize()
    return " ".join(e.key for e in prof.key_averages())


def test_which_kernel_runs():
    """cache_attn_kernel<D, format, score, blocks of 16 rows, wavefronts>"""
    _say("[kernels]")
    many = Case([200] * 3, n=[40, 7, 33], H=8, Hkv=2, D=128, bs=64, seed=1)
    assert "cache_prompt_kernel<128, 0, 0>" in _kernels(lambda: _prompt(many))
    assert "cache_attn_kernel<128, 0, 0, 2, 4>" in _kernels(lambda: many.call(max_query=40, max_seqlen=200))
    few = Case([700, 300], H=8, Hkv=2, D=64, bs=64, seed=1)
    assert "cache_attn_kernel<64, 0, 0, 1, 8>" in _kernels(lambda: few.call(max_seqlen=700))
    assert "cache_attn_kernel<64, 0, 0, 1, 4>" in _kernels(lambda: few.call(max_seqlen=200))
    batch = Case([100] * 40, H=8, Hkv=8, D=64, bs=64, seed=1)
    assert "cache_attn_kernel<64, 0, 0, 1, 4>" in _kernels(lambda: batch.call(max_seqlen=4000))


@pytest.mark.parametrize("kw", VARIANTS, ids=lambda kw: "-".join(f"{k}" for k in kw) or "plain")
def test_prompt_tiles(kw):
    """Every mask, score modifier and normaliser on the 128-row kernel, both channel counts and formats."""
    _say(f"[prompt] {kw}")
    for n, D, dtype, bs in (([1, 3, 0, 7, 5, 2, 4], 64, E4, 16), ([60, 17, 0, 1, 33, 90, 64], 128, E5, 64),
                            ([60, 17, 0, 1, 33, 90, 64], 64, E5, 128), ([130, 20, 64, 0, 65, 1, 2], 128, E4, 16)):
        lens = [max(a, b) for a, b in zip([1, 40, 64, 100, 33, 300, 517], n)]
        c = Case(lens, n=n, D=D, dtype=dtype, bs=bs, seed=5)
        c.check(_prompt(c, **kw), **kw)


@pytest.mark.parametrize("bs", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("H,Hkv", [(2, 2), (12, 4), (17, 1), (32, 2)])
def test_prompt_pages_and_heads(bs, H, Hkv):
    _say(f"[prompt] pages {bs} {H}/{Hkv}")
    c = Case([129, 63, 64, 65, 400, 31], n=[129, 40, 1, 65, 30, 0], H=H, Hkv=Hkv, D=128, bs=bs, seed=bs)
    c.check(_prompt(c))
    c = Case([129, 63, 64, 65, 400, 31], n=[129, 40, 1, 65, 30, 0], H=H, Hkv=Hkv, D=64, bs=bs, seed=bs + 1)
    c.check(_prompt(c))


def test_prompt_split_and_wrong_bounds():
    """Keys split between workgroups, a bound on the queries that most requests exceed, far too wide ones."""
    _say("[prompt] split")
    c = Case([3001, 2000], n=[90, 40], H=4, Hkv=1, D=128, bs=32, seed=3)
    dev, cu = _wide(c), _i32(c.cu).to(DEV)
    for norm in ("softmax", "relu"):
        for bounds in (dict(max_query=4096), dict(max_query=1 << 20), dict(max_query=200, max_seqlen=1 << 18), dict()):
            c.check(lib.attention_cache(*dev, cu, norm=norm, **bounds), norm=norm)
    a, b = (lib.attention_cache(*dev, cu, max_query=4096) for _ in range(2))
    assert torch.equal(a, b)
    # few workgroups for many tiles: each walks several
    c = Case([900] * 4, n=[700, 20, 0, 300], H=4, Hkv=1, D=64, bs=64, seed=4)
    c.check(lib.attention_cache(*_wide(c), _i32(c.cu).to(DEV), max_query=100))


@pytest.mark.parametrize("dtype", [E4, E5])
def test_prompt_numbers_that_are_none(dtype):
    """As on the other tiles: NaN reaches the queries that see it and no other."""
    _say(f"[prompt] nan {dtype}")
    bad = 0x7F if dtype == E4 else 0x7E
    for D in (64, 128):
        c = Case([200, 90, 150], n=[80, 40, 33], bs=16, dtype=dtype, D=D, seed=11)
        for pos in (20, 199, 160):
            p = c.table[0, pos // 16].long()
            c.vc.view(torch.uint8)[p, :, pos % 16, ::3] = bad
            c.kc.view(torch.uint8)[p, 1, pos % 16, 0] = bad
        p = c.table[1, 1].long()
        c.vc.view(torch.uint8)[p] = bad
        c.ks[p], c.vs[p] = float("nan"), float("inf")
        c.table[2, 3] = -1
        for kw in (dict(window=48), dict(window=48, norm="sigmoid"), dict(block=64)):
            want, _, _ = oc.attend_ref(c.q, c.kc, c.vc, c.ks, c.vs, c.table, c.lens, c.cu, **{**dict(causal=True), **kw})
            got = _prompt(c, **kw).double().cpu()
            assert torch.equal(torch.isnan(got), torch.isnan(want)), kw
            fine = ~torch.isnan(want)
            assert float((got - want)[fine].abs().max()) < 0.05 * float(want[fine].abs().max())


def test_prompt_infinities_of_e5m2():
    _say("[prompt] inf")
    c = Case([70], n=40, bs=16, dtype=E5, seed=13)
    p = c.table[0, 4].long()
    c.vc.view(torch.uint8)[p, 0, 4, 0] = 0x7C  # position 68
    c.vc.view(torch.uint8)[p, 1, 5, 1] = 0xFC  # position 69
    got = _prompt(c).float().cpu()
    assert [float(got[t, 0, 0]) for t in (38, 39)] == [float("inf")] * 2 and float(got[39, 2, 1]) == float("-inf")
    got[38:, :2, 0] = 0
    got[39, 2:, 1] = 0
    assert bool(torch.isfinite(got).all())


def test_prompt_scales_and_rising_scores():
    """Scales that are no powers of two; scores that rise along the keys."""
    _say("[prompt] scales")
    for norm in ("softmax", "sigmoid", "relu"):
        c = Case([200, 77], n=[70, 77], bs=32, D=128, seed=15)
        c.ks *= 1.37
        c.vs *= torch.linspace(0.6, 1.9, c.vs.numel()).reshape(c.vs.shape)
        c.check(_prompt(c, norm=norm), norm=norm)
    c = Case([900], n=100, H=4, Hkv=2, D=64, bs=64, seed=17, spread=0.0)
    c.ks *= torch.exp2(torch.arange(c.ks.shape[0]) % 7).float()[:, None]
    for kw in (dict(scale=1.0), dict(scale=1e-4), dict(alibi_slopes=[3.0, 1.0, 0.5, 0.1]), dict(alibi_slopes=[-3.0, -1.0, -0.5, -0.1])):
        c.check(_prompt(c, **kw), **kw)


@pytest.mark.parametrize("R,Hkv,hi", [(70, 8, 700), (300, 2, 90), (24, 8, 3000), (40, 4, 1500)])
def test_batches_of_many_groups(R, Hkv, hi):
    """Four wavefronts to a workgroup, whole requests and parts of them, many requests that have few of the parts."""
    _say(f"[batch] {R} {Hkv} {hi}")
    g = torch.Generator().manual_seed(R)
    lens = [hi] + [int(x) for x in torch.randint(0, hi // 3, (R - 1,), generator=g)]
    Case(lens, H=Hkv, Hkv=Hkv, D=64, bs=64, seed=R).check()


def test_captured_prompt_follows_its_inputs():
    """Two graphs of prompt calls, replayed in turn with eager work between: each has its own workspace."""
    _say("[prompt] graphs")
    cases = [Case([3001, 2000], n=[90, 40], H=4, Hkv=1, D=64, bs=32, seed=s) for s in (21, 22)]
    devs, cu = [_wide(c) for c in cases], _i32(cases[0].cu).to(DEV)
    call = lambda d: lib.attention_cache(*d, cu, max_query=4096)  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for d in devs:
            call(d)
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for d in devs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(call(d))
        graphs.append(g)
    for i in range(4):
        for d in devs:
            d[0].copy_(torch.randn(d[0].shape, generator=torch.Generator().manual_seed(i)).to(torch.bfloat16))
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        got = [o.clone() for o in outs]
        for d, o in zip(devs, got):
            assert torch.equal(call(d), o)


def test_gradients_are_refused():
    c = Case([20], n=1, seed=1)
    q, kc, vc, ks, vs, table, lens = c.device()
    k = torch.zeros(1, 2, 64, dtype=torch.bfloat16, device=DEV, requires_grad=True)
    with pytest.raises(ValueError, match="forward only"):
        lib.write_cache(k, k, kc, vc, ks, vs, lens)
    with pytest.raises(ValueError, match="forward only"):
        lib.attention_cache(q.requires_grad_(), kc, vc, ks, vs, table, lens)
    with torch.no_grad():
        lib.attention_cache(q, kc, vc, ks, vs, table, lens)


@pytest.mark.parametrize("dilation", [2, 31, 32, 33, 100, 1 << 20])
@pytest.mark.parametrize("causal", [True, False])
def test_dilations_around_a_word(dilation, causal):
    """The keys a row sees of 32 are one word: dilations below, at and past its width, on every row tile."""
    _say(f"[dilation] {dilation} {causal}")
    kw = dict(dilation=dilation, causal=causal)
    c = Case([33, 700, 64, 301], H=8, Hkv=2, D=128, bs=16, seed=dilation)
    c.check(c.call(**kw), **kw)
    c = Case([33, 700, 64, 301], n=[20, 1, 0, 33], H=4, Hkv=2, D=64, dtype=E5, bs=32, seed=dilation + 1)
    c.check(c.call(max_query=33, max_seqlen=700, **kw), **kw)
    c.check(_prompt(c, **kw), **kw)
