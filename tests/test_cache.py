"""CPU tests of the paged 8-bit cache: its oracle against closed forms and the generic
attention oracle, the walk geometry (a host program), the C ABI's layout and refusals,
and the Python layer's refusals and fake shapes."""
import ctypes
import re
import shutil
import subprocess
from pathlib import Path

import pytest
import torch

import chia_proj_amd as lib
from chia_proj_amd import _lib
from oracle import cache as oc
from oracle import generic

ROOT = Path(__file__).resolve().parent.parent
HEADER = ROOT / "include" / "chia_cache.h"
FP8 = (torch.float8_e4m3fn, torch.float8_e5m2)


# ---- the oracle -----------------------------------------------------------------

@pytest.mark.parametrize("dtype", FP8)
def test_rounding_is_the_formats(dtype):
    codes = torch.arange(256, dtype=torch.uint8).view(dtype).float()
    codes = codes[torch.isfinite(codes)]
    assert torch.equal(oc.round_code(codes, dtype), codes.double())
    g = torch.Generator().manual_seed(1)
    x = torch.cat([torch.randn(4000, generator=g) * s for s in (1e-7, 1e-3, 1.0, 100.0)])
    x = x.clamp(-oc.TOP[dtype], oc.TOP[dtype])
    assert torch.equal(oc.round_code(x, dtype), x.to(dtype).double())
    mid = (codes.sort().values[:-1] + codes.sort().values[1:]) / 2  # ties
    assert torch.equal(oc.round_code(mid, dtype), mid.to(dtype).double())


@pytest.mark.parametrize("dtype", FP8)
def test_scale_is_the_least_power_of_two(dtype):
    top = oc.TOP[dtype]
    for e in (-126, -20, 0, 7, 100):
        assert oc.need_scale(top * 2.0 ** e, dtype) == 2.0 ** e
        assert oc.need_scale(top * 2.0 ** e * (1 + 2.0 ** -40), dtype) == 2.0 ** (e + 1)
    assert oc.need_scale(0.0, dtype) == 2.0 ** -126


@pytest.mark.parametrize("dtype", FP8)
def test_write_does_not_depend_on_how_tokens_are_cut(dtype):
    g = torch.Generator().manual_seed(2)
    x = (torch.randn(40, 2, 64, generator=g) * torch.rand(40, 1, 1, generator=g).mul(6).exp()).to(torch.bfloat16)
    codes = torch.zeros(3, 2, 16, 64).to(dtype)
    whole, scale = oc.write_ref(x, codes, torch.ones(3, 2), list(range(40)))
    c, s, at = codes, torch.ones(3, 2), 0
    for n in (1, 3, 20, 1, 15):
        out, s64 = oc.write_ref(x[at:at + n], c, s, list(range(at, at + n)))
        c, s, at = out.to(dtype), s64.float(), at + n
    assert torch.equal(s.double(), scale)
    # apart from what the codes' smallest step rounds: at most one such step per rescaling
    tiny = 2.0 ** (oc._FORMAT[dtype][0] - oc._FORMAT[dtype][1])
    assert float((c.float().double() - whole).abs().max()) <= 2 * tiny
    value = whole * scale[:, :, None, None]
    err = (value.transpose(1, 2).reshape(48, 2, 64)[:40] - x.double()).abs()
    half = 2.0 ** -(oc._FORMAT[dtype][1] + 1)
    step = scale.repeat_interleave(16, 0)[:40, :, None] * tiny
    assert bool((err <= torch.maximum(half * x.double().abs(), step / 2)).all())


MASKS = [dict(), dict(causal=False), dict(window=7), dict(causal=False, window=9), dict(block=13), dict(dilation=3),
         dict(prefix=11, window=4), dict(causal=False, block=8, prefix=3), dict(dilation=2, window=16)]


@pytest.mark.parametrize("mask", MASKS)
@pytest.mark.parametrize("score", [dict(), dict(softcap=3.0), dict(alibi_slopes=[0.3, 0.1, 0.2, 0.05]),
                                   dict(norm="sigmoid", bias=-2.0, post_scale=0.5), dict(norm="relu", head_scale=[1, 2, 3, 4.])])
def test_attend_oracle_is_the_generic_one_on_a_whole_prompt(mask, score):
    """Every token of a prompt as a query: the rectangle becomes the square the library has always had."""
    g = torch.Generator().manual_seed(3)
    S, H, Hkv, D, bs = 37, 4, 2, 64, 16
    q = torch.randn(S, H, D, generator=g).to(torch.bfloat16)
    kc, vc = ((torch.randn(5, Hkv, bs, D, generator=g) * 30).to(torch.float8_e4m3fn) for _ in range(2))
    ks, vs = torch.rand(5, Hkv, generator=g) / 30, torch.rand(5, Hkv, generator=g) / 30
    table = torch.tensor([[3, 0, 4]], dtype=torch.int32)
    full = dict(causal=True, window=0, dilation=1, block=0, prefix=0)
    full.update(mask)
    o, size, _ = oc.attend_ref(q, kc, vc, ks, vs, table, [S], [0, S], **full, **score)
    k, v = ((c.double() * s.double()[:, :, None, None])[table[0].long()].transpose(1, 2).reshape(1, -1, Hkv, D)[:, :S]
            .transpose(1, 2) for c, s in ((kc.float(), ks), (vc.float(), vs)))
    want = generic.attention_ref(q.transpose(0, 1)[None], k, v, dtype=torch.float64, **full, **score)
    assert torch.allclose(o, want[0].transpose(0, 1), rtol=1e-9, atol=1e-12)
    assert bool((size >= o.abs() - 1e-12).all())


def test_attend_oracle_skips_pages_outside_the_cache_and_short_requests():
    q = torch.ones(4, 1, 64, dtype=torch.bfloat16)
    kc = torch.zeros(2, 1, 16, 64).to(torch.float8_e4m3fn)
    vc = torch.stack([torch.full((1, 16, 64), 1.0), torch.full((1, 16, 64), 3.0)]).to(torch.float8_e4m3fn)
    one = torch.ones(2, 1)
    table = torch.tensor([[0, 1], [0, -1], [7, 1], [0, 1]], dtype=torch.int32)
    o, _, _ = oc.attend_ref(q, kc, vc, one, one, table, [32, 32, 32, 0], [0, 1, 2, 3, 4])
    assert [float(o[t, 0, 0]) for t in range(4)] == [2.0, 1.0, 3.0, 0.0]


def test_tables_oracle():
    table, slots, pos, cu, lens, left, missing = oc.tables_ref(
        [[5, -1, -1], [-1, -1, -1], [6, 7, -1]], [10, 0, 32], [8, 17, 3], [1, 2, 3, 4], 4, 16, 30)
    assert table == [[5, 4, -1], [3, 2, -1], [6, 7, 1]]
    assert slots[:8] == [5 * 16 + p for p in range(10, 16)] + [64, 65]
    assert cu == [0, 8, 25, 28] and lens == [18, 17, 35] and left == 0 and missing == 0
    assert pos[8:10] == [0, 1] and slots[28:] == [-1, -1]


# ---- the walk ---------------------------------------------------------------------

@pytest.mark.skipif(shutil.which("g++") is None, reason="no host compiler")
def test_walk_against_the_masks_definition(tmp_path):
    exe = tmp_path / "check_cache_walk"
    subprocess.run(["g++", "-std=c++17", "-O1", "-g", "-fsanitize=address,undefined", "-fno-sanitize-recover=all",
                    f"-I{ROOT / 'chia_proj_amd' / 'csrc'}", str(ROOT / "tests" / "cpp" / "check_cache_walk.cpp"),
                    "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert out.returncode == 0 and " 0 failures" in out.stdout, out.stdout + out.stderr


# ---- the C ABI --------------------------------------------------------------------

def _fields(text, name):
    body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), text, re.S).group(1)
    body = re.sub(r"/\*.*?\*/", "", body, flags=re.S)
    out = []
    for decl in filter(None, (d.strip() for d in body.split(";"))):
        out += [re.sub(r"\[.*\]", "", part.strip().split()[-1].lstrip("*")) for part in decl.split(",")]
    return out


STRUCTS = {"chia_cache_tables_args": _lib.CacheTablesArgs, "chia_cache_release_args": _lib.CacheReleaseArgs,
           "chia_cache_write_args": _lib.CacheWriteArgs, "chia_cache_attn_args": _lib.CacheAttnArgs}


def test_exports_and_struct_mirrors(lib_built):
    text = HEADER.read_text()
    declared = set(re.findall(r"^(?:int|int64_t) (chia_cache_[a-z_]+)\(", text, re.M))
    assert declared == set(_lib.CACHE_EXPORTS)
    for name in declared:
        assert hasattr(lib_built, name)
    for name, cls in STRUCTS.items():
        assert _fields(text, name) == [f[0] for f in cls._fields_], name


@pytest.mark.skipif(shutil.which("gcc") is None, reason="no host compiler")
def test_struct_sizes_and_offsets(tmp_path):
    """The ctypes mirrors lay their fields where a C compiler lays the header's."""
    lines = ["#include <stddef.h>", "#include <stdio.h>", '#include "chia_cache.h"', "int main(void) {"]
    for name, cls in STRUCTS.items():
        lines.append('printf("%%zu\\n", sizeof(%s));' % name)
        lines += ['printf("%%zu\\n", offsetof(%s, %s));' % (name, f[0]) for f in cls._fields_]
    src, exe = tmp_path / "o.c", tmp_path / "o"
    src.write_text("\n".join(lines + ["return 0; }"]))
    subprocess.run(["gcc", f"-I{ROOT / 'include'}", str(src), "-o", str(exe)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    want = []
    for cls in STRUCTS.values():
        want += [ctypes.sizeof(cls)] + [getattr(cls, f[0]).offset for f in cls._fields_]
    assert got == want


def _tables_args(**kw):
    a = dict(block_size=16, block_tables=16, table_stride=4, requests=2, width=4, context_lens=16, new_lens=16,
             free_blocks=16, free_count=16, free_capacity=4, max_tokens=4, slots=16, positions=16, cu_seqlens=16,
             seq_lens=16, free_left=16, missing=16)
    a.update(kw)
    return _lib.CacheTablesArgs(**a)


def _write_args(**kw):
    a = dict(format=0, k=16, v=16, k_cache=16, v_cache=16, k_scale=16, v_scale=16, slots=16, tokens=4, kv_heads=2,
             head_dim=64, num_blocks=4, block_size=16)
    a.update(kw)
    return _lib.CacheWriteArgs(**a)


def _attn_args(attn=None, **kw):
    t = _lib.AttnArgs(norm=0, batch=2, heads=4, seqlen=64, head_dim=64, causal=1, scale=0.125, kv_heads=2, q=16, k=16,
                      v=16, o=16, **(attn or {}))
    a = dict(format=0, k_scale=16, v_scale=16, block_tables=16, table_stride=4, width=4, seq_lens=16, num_blocks=8,
             queries=2, max_query=1, block_size=16)
    a.update(kw)
    c = _lib.CacheAttnArgs(**a)
    c.attn = ctypes.pointer(t)
    return c


@pytest.mark.parametrize("fn,make,kw,status", [
    ("tables", _tables_args, dict(block_size=24), -2), ("tables", _tables_args, dict(block_size=8), -2),
    ("tables", _tables_args, dict(block_size=512), -2), ("tables", _tables_args, dict(requests=0), -2),
    ("tables", _tables_args, dict(width=0), -2), ("tables", _tables_args, dict(table_stride=3), -2),
    ("tables", _tables_args, dict(max_tokens=-1), -2), ("tables", _tables_args, dict(free_capacity=-1), -2),
    ("tables", _tables_args, dict(block_tables=None), -1), ("tables", _tables_args, dict(free_blocks=None), -1),
    ("tables", _tables_args, dict(missing=None), -1), ("tables", _tables_args, dict(slots=None), -1),
    ("tables", _tables_args, dict(slots=18), -7), ("tables", _tables_args, dict(struct_size=8), -8),
    ("write", _write_args, dict(format=2), -6), ("write", _write_args, dict(head_dim=96), -3),
    ("write", _write_args, dict(block_size=20), -2), ("write", _write_args, dict(tokens=-1), -2),
    ("write", _write_args, dict(num_blocks=0), -2), ("write", _write_args, dict(num_blocks=1 << 28), -2),
    ("write", _write_args, dict(kv_heads=0), -2), ("write", _write_args, dict(k=None), -1),
    ("write", _write_args, dict(slots=None), -1), ("write", _write_args, dict(v_cache=24), -7),
    ("write", _write_args, dict(k_scale=18), -7), ("write", _write_args, dict(struct_size=0), -8),
    ("attn", _attn_args, dict(format=3), -6), ("attn", _attn_args, dict(attn=dict(head_dim=80)), -3),
    ("attn", _attn_args, dict(attn=dict(norm=5)), -6), ("attn", _attn_args, dict(attn=dict(window=-1)), -4),
    ("attn", _attn_args, dict(attn=dict(dilation=2, prefix=3)), -4), ("attn", _attn_args, dict(attn=dict(scale=0.0)), -5),
    ("attn", _attn_args, dict(attn=dict(softcap=-1.0)), -5), ("attn", _attn_args, dict(attn=dict(kv_heads=3)), -2),
    ("attn", _attn_args, dict(attn=dict(seqlen=0)), -2), ("attn", _attn_args, dict(block_size=15), -2),
    ("attn", _attn_args, dict(width=0), -2), ("attn", _attn_args, dict(table_stride=-1), -2),
    ("attn", _attn_args, dict(num_blocks=0), -2), ("attn", _attn_args, dict(queries=3), -2),
    ("attn", _attn_args, dict(max_query=0), -2), ("attn", _attn_args, dict(seq_lens=None), -1),
    ("attn", _attn_args, dict(block_tables=None), -1), ("attn", _attn_args, dict(k_scale=18), -7),
    ("attn", _attn_args, dict(workspace=8), -7), ("attn", _attn_args, dict(struct_size=4), -8),
    ("attn", _attn_args, dict(attn=dict(struct_size=4)), -8), ("attn", _attn_args, dict(reserved0=1), -8),
])
def test_refusals_before_any_launch(lib_built, fn, make, kw, status):
    kw = dict(kw)
    if "attn" in kw:
        base = dict(kw.pop("attn"))
        a = _attn_args(**kw)
        for name, val in base.items():
            setattr(a.attn.contents, name, val)
    else:
        a = make(**kw)
    assert getattr(lib_built, "chia_cache_" + fn)(ctypes.byref(a), None) == status


def test_workspace_is_asked_for_and_checked(lib_built):
    a = _attn_args()
    a.attn.contents.seqlen = 60000
    a.width, a.table_stride, a.num_blocks = 4096, 4096, 8192
    need = lib_built.chia_cache_attn_workspace_size(ctypes.byref(a))
    assert need > 0 and need % (2 * 4 * (64 + 2) * 4) == 0
    assert lib_built.chia_cache_attn(ctypes.byref(a), None) == -9  # none given
    a.workspace, a.workspace_bytes = 16, need - 1
    assert lib_built.chia_cache_attn(ctypes.byref(a), None) == -9
    a.attn.contents.seqlen = 16
    assert lib_built.chia_cache_attn_workspace_size(ctypes.byref(a)) == 0
    assert lib_built.chia_cache_attn_workspace_size(None) == -1


def test_no_tokens_is_no_launch(lib_built):
    assert lib_built.chia_cache_write(ctypes.byref(_write_args(tokens=0, k=None)), None) == 0
    a = _attn_args(queries=0)
    a.attn.contents.cu_seqlens = 16
    assert lib_built.chia_cache_attn(ctypes.byref(a), None) == 0


# ---- the Python layer -------------------------------------------------------------

def _i32(*shape):
    return torch.zeros(*shape, dtype=torch.int32)


def test_python_refusals():
    t = _i32(2, 4)
    with pytest.raises(ValueError, match="GPU"):
        lib.extend_block_tables(t, _i32(2), _i32(2), _i32(3), _i32(1), block_size=16, max_tokens=4)
    with pytest.raises(TypeError, match="int32"):
        lib.extend_block_tables(t.long(), _i32(2), _i32(2), _i32(3), _i32(1), block_size=16, max_tokens=4)
    with pytest.raises(ValueError, match="unit last stride"):
        lib.release_block_tables(_i32(4, 2).t(), _i32(2), _i32(2).bool(), _i32(3), _i32(1), block_size=16)
    kc = torch.zeros(4, 2, 16, 64).to(torch.float8_e4m3fn)
    sc = torch.ones(4, 2)
    k = torch.zeros(3, 2, 64, dtype=torch.bfloat16)
    with pytest.raises(TypeError, match="k_cache"):
        lib.write_cache(k, k, kc.float(), kc, sc, sc, _i32(3))
    with pytest.raises(ValueError, match="one shape"):
        lib.write_cache(k, k, kc, kc[:2], sc, sc, _i32(3))
    with pytest.raises(ValueError, match="one shape"):
        lib.write_cache(k, k, kc, kc.float().to(torch.float8_e5m2), sc, sc, _i32(3))
    with pytest.raises(ValueError, match="block_size"):
        bad = torch.zeros(4, 2, 24, 64).to(torch.float8_e4m3fn)
        lib.write_cache(k, k, bad, bad, sc, sc, _i32(3))
    with pytest.raises(ValueError, match="multiples of 16"):
        bad = torch.zeros(4, 2, 16, 72).to(torch.float8_e4m3fn)[..., :64]
        lib.write_cache(k, k, bad, bad, sc, sc, _i32(3))
    with pytest.raises(ValueError, match="forward only"):
        lib.attention_cache(torch.zeros(2, 4, 64, dtype=torch.bfloat16, requires_grad=True), kc, kc, sc, sc, t, _i32(2))
    with pytest.raises(ValueError, match="GPU"):
        lib.attention_cache(torch.zeros(2, 4, 64, dtype=torch.bfloat16), kc, kc, sc, sc, t, _i32(2))


def test_fake_shapes():
    ops = torch.ops.chia_attn
    m = lambda *s, d=torch.int32: torch.empty(*s, dtype=d, device="meta")  # noqa: E731
    step = ops.extend_block_tables(m(3, 8), m(3), m(3), m(9), m(1), 16, 40)
    assert [tuple(t.shape) for t in step] == [(40,), (40,), (4,), (3,), (1,), (1,)]
    assert all(t.dtype == torch.int32 for t in step)
    c, s = m(9, 2, 16, 64, d=torch.float8_e4m3fn), m(9, 2, d=torch.float32)
    k = m(40, 2, 64, d=torch.bfloat16)
    assert ops.write_cache(k, k, c, c.clone(), s, s.clone(), m(40)) is None
    o = ops.attention_cache(m(40, 4, 64, d=torch.bfloat16), c, c, s, s, m(3, 8), m(3), m(4), None, None, "softmax", True,
                            0, 1, 0, 0, None, None, None, 0.0, 0.0, 1.0)
    assert o.shape == (40, 4, 64) and o.dtype == torch.bfloat16
    assert tuple(ops.release_block_tables(m(3, 8), m(3), m(3, d=torch.bool), m(9), m(1), 16).shape) == (1,)


def test_package_exports():
    for name in ("extend_block_tables", "release_block_tables", "write_cache", "attention_cache", "CacheStep"):
        assert name in lib.__all__ and hasattr(lib, name)
