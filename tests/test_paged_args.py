"""Refusals of the operators over a paged KV cache that need no device, and the plain forms' own closed cases."""
import ctypes

import numpy as np
import pytest
import torch

from tests import paged_reference as R

P = ctypes.c_void_p(256)   # never followed: the call is refused first
F32, F16, BF16 = 0, 1, 30


@pytest.fixture(scope="module")
def lib():
    from smallmind_amd import _lib
    return _lib.load()


@pytest.mark.parametrize("args,code", [((F32, 8, 4, 64, 64), -5), ((8, 8, 4, 64, 64), -5), ((F16, 0, 4, 64, 64), -1), ((F16, 8, 0, 64, 64), -1),
                                       ((F16, -1, 4, 64, 64), -1), ((F16, 8, 4, 0, 64), -5), ((F16, 8, 4, 60, 64), -5),
                                       ((F16, 8, 4, 264, 64), -5), ((F16, 8, 4, 64, 0), -5), ((F16, 8, 4, 64, 8), -5), ((F16, 8, 4, 64, 48), -5),
                                       ((F16, 8, 4, 64, 2048), -5), ((F16, 8, 4, 64, -64), -5), ((F16, 1 << 30, 1, 64, 64), -5),
                                       ((F16, 8, 65536, 64, 64), -5), ((BF16, (1 << 21) - 1, 65535, 256, 1024), -2)])
def test_cache_create_refuses(lib, args, code):
    h = ctypes.c_void_p(77)
    assert lib.smx_paged_cache_create(*args, ctypes.byref(h)) == code
    assert h.value is None
    assert b"smx_paged_cache_create" in lib.smx_last_error()


def test_null_caches_are_refused(lib):
    n = ctypes.c_int64()
    assert lib.smx_paged_cache_create(F16, 8, 4, 64, 64, None) == -1
    assert lib.smx_paged_cache_info(None, None, None, None, None, None, None) == -1
    assert lib.smx_paged_cache_destroy(None) == 0
    assert lib.smx_paged_append(None, F32, None, 0, 0, P, 64, P, 64, None, None, 0.0, None, None, P, 1, F32, None, None) == -1
    assert lib.smx_paged_read(None, P, 1, P, P, None) == -1
    assert lib.smx_attention_paged_work_bytes(None, F32, 1, 1, 1, 1, 64, None, ctypes.byref(n)) == -1
    assert lib.smx_attention_mass_work_bytes(None, F32, 1, 1, 1, 64, ctypes.byref(n)) == -1
    assert lib.smx_attention_paged(None, F32, P, 64, P, None, 1, 1, 1, P, P, P, 1, 1, 64, None, P, 1 << 20, None) == -1
    assert lib.smx_attention_mass(None, F32, P, 64, P, None, 0, 0, P, 1, 1, 1, P, P, P, 1, 1, 64, None, P, 1 << 20, None) == -1
    assert lib.smx_paged_evict(None, P, 64, P, 1, 64, 32, 8, P, 1, P, 1, P, P, P, None) == -1


def rotation(**k):
    from smallmind_amd._lib import RotationC
    d = dict(cos=256, sin=256, n_pos=8, n_rot=64, halves=0, n_axes=1, sections=(0, 0, 0, 0))
    d.update(k)
    return RotationC(d["cos"], d["sin"], d["n_pos"], d["n_rot"], d["halves"], d["n_axes"], (ctypes.c_int32 * 4)(*d["sections"]))


def test_qk_norm_rope_refuses(lib):
    def run(tin=F32, q=P, qs=128, nh=2, k=P, ks=64, kv=1, hd=64, gq=None, gk=None, eps=1e-6, rot=None, pos=P, n=3, tout=F32, qo=P, ko=P):
        return lib.smx_qk_norm_rope(tin, q, qs, nh, k, ks, kv, hd, gq, gk, eps, None if rot is None else ctypes.byref(rot), pos, n, tout, qo,
                                    ko, None)
    assert run(n=0) == 0        # nothing to do
    odd = ctypes.c_void_p(258)
    for bad in (dict(q=None, k=None), dict(qo=None), dict(ko=None), dict(n=-1), dict(nh=0), dict(nh=65536, qs=1 << 30), dict(kv=0),
                dict(qs=127), dict(ks=63), dict(q=odd), dict(k=odd), dict(qo=odd), dict(ko=odd), dict(tin=F16, q=ctypes.c_void_p(257)),
                dict(gq=P, eps=-1.0), dict(gk=P, eps=float("nan")), dict(gq=P, eps=float("inf")), dict(gq=ctypes.c_void_p(257)),
                dict(rot=rotation(cos=None)), dict(rot=rotation(sin=None)), dict(rot=rotation(), pos=None), dict(rot=rotation(cos=257)),
                dict(rot=rotation(n_pos=0)), dict(rot=rotation(n_rot=0)), dict(rot=rotation(n_rot=63)), dict(rot=rotation(n_rot=66)),
                dict(rot=rotation(halves=2)), dict(rot=rotation(n_axes=0)), dict(rot=rotation(n_axes=5)),
                dict(rot=rotation(n_axes=2, sections=(16, 15, 0, 0))), dict(rot=rotation(n_axes=2, sections=(33, -1, 0, 0))),
                dict(rot=rotation(n_axes=3, sections=(2**31 - 1, 2**31 - 1, 34, 0)))):
        assert run(**bad) == -1, bad
        assert b"smx_qk_norm_rope" in lib.smx_last_error()
    for bad in (dict(tin=2), dict(tout=8), dict(hd=60), dict(hd=264, qs=1024, ks=512), dict(hd=0), dict(n=2**31 - 1)):
        assert run(**bad) == -5, bad


def test_writes_into_their_inputs_are_refused(lib):
    """3 tokens of 2 heads of queries and 1 of keys, 64 fp32 values each, in rows of a fused projection 1024 bytes apart."""
    base, end = 1 << 20, (1 << 20) + 3 * 1024
    for qo, ko in ((base, end), (base + 1024 * 2 + 508, end), (base - 1532, end), (end, base + 512), (end, base + 1024 * 2 + 764),
                   (end, base - 764), (end, base + 256)):
        p = [ctypes.c_void_p(x) for x in (base, base + 512, qo, ko)]
        assert lib.smx_qk_norm_rope(F32, p[0], 256, 2, p[1], 256, 1, 64, None, None, 0.0, None, None, 3, F32, p[2], p[3], None) == -1, (qo, ko)
        assert b"lies in the inputs' memory" in lib.smx_last_error()
    # one token's stride may be anything
    p = [ctypes.c_void_p(x) for x in (base, base + 512, base + 252, end)]
    assert lib.smx_qk_norm_rope(F32, p[0], 1 << 62, 2, p[1], 1 << 62, 1, 64, None, None, 0.0, None, None, 1, F32, p[2], p[3], None) == -1


def test_python_refuses_before_any_call():
    import types

    from smallmind_amd import quantization as Q
    cos = torch.zeros(4, 8)
    for bad in (dict(cos=torch.zeros(4)), dict(sin=torch.zeros(4, 7)), dict(cos=torch.zeros(4, 8, dtype=torch.float64)), dict(sections=[4, 5]),
                dict(sections=[9, -1]), dict(sections=[]), dict(sections=[2, 2, 2, 1, 1]), dict(cos=torch.zeros(8, 4).t())):
        with pytest.raises(ValueError):
            Q.Rotation(**{**dict(cos=cos, sin=cos), **bad})
    with pytest.raises(ValueError, match="float16 or bfloat16"):
        Q.GpuPagedCache(torch.float32, 4, 1, 64)
    big = (1 << 32) + 1
    for at in range(4):
        sizes = [4, 1, 64, 64]
        sizes[at] += big - 1
        with pytest.raises(ValueError, match="out of range"):
            Q.GpuPagedCache(torch.float16, *sizes)
    cache = types.SimpleNamespace(device=torch.device("cuda", 0), head_dim=64, page_size=16, n_kv_head=1, dtype=torch.float16,
                                  _handle=lambda: None)
    q, one, two, tab = torch.zeros(1, 1, 64), torch.zeros(1, dtype=torch.int32), torch.zeros(2, dtype=torch.int32), torch.zeros(1, 4, dtype=torch.int32)
    lse = torch.zeros(1, 1)
    for bad in (dict(q=torch.zeros(1, 64)), dict(q=torch.zeros(1, 1, 32)), dict(q=q.double()), dict(q=q.bfloat16()), dict(starts=one),
                dict(starts=two.long()), dict(lens=two), dict(tables=torch.zeros(4, dtype=torch.int32)), dict(tables=torch.zeros(2, 4, dtype=torch.int32)),
                dict(tables=tab.long()), dict(max_q=big), dict(max_len=big), dict(max_len=1 << 31), dict(window=big), dict(cap=-1.0),
                dict(cap=float("nan")), dict(scale=0.0), dict(scale=float("inf")), dict(slopes=torch.zeros(2)), dict(slopes=torch.zeros(1).double()),
                dict(prefix=two), dict(prefix=torch.zeros(1))):
        a = {**dict(q=q, starts=two, lens=one, tables=tab, max_q=1, max_len=64), **bad}
        with pytest.raises(ValueError):
            Q.attention_paged(a.pop("q"), cache, a.pop("starts"), a.pop("lens"), a.pop("tables"), a.pop("max_q"), a.pop("max_len"), **a)
        a = {**dict(q=q, starts=two, lens=one, tables=tab, max_q=1, max_len=64), **bad}
        with pytest.raises(ValueError):
            Q.attention_mass(a.pop("q"), lse, cache, a.pop("starts"), a.pop("lens"), a.pop("tables"), a.pop("max_q"), a.pop("max_len"), **a)
    for bad in (torch.zeros(1, 64), torch.zeros(2, 1, 64), torch.zeros(1, 2, 64), torch.zeros(1, 1, 64).double()):
        with pytest.raises(ValueError):
            Q.attention_mass(q, lse, cache, two, one, tab, 1, 64, mass=bad)
    with pytest.raises(ValueError):
        Q.attention_mass(q, torch.zeros(2, 1), cache, two, one, tab, 1, 64)
    with pytest.raises(ValueError, match="out must"):
        Q.attention_paged(q, cache, two, one, tab, 1, 64, out=torch.zeros(1, 1, 64).half())


def test_factors_below_fp32_are_refused_in_python():
    """0 in fp32, which would be taken for the default scale and for no cap."""
    from smallmind_amd import quantization as Q
    for bad in (dict(scale=1e-46), dict(scale=1e-300), dict(cap=1e-46), dict(cap=5e-324)):
        with pytest.raises(ValueError, match="below the range"):
            Q._rules(1, 1, **{**dict(scale=None, cap=0.0, slopes=None, window=0, prefix=None), **bad})
    for scale in (1.4e-45, 2e-45, 1.0):
        assert Q._rules(1, 1, scale, 0.0, None, 0, None)._obj.scale > 0.0


def test_plain_rotation_keeps_lengths_and_turns_by_axes():
    rng = np.random.default_rng(0)
    x = rng.normal(0, 1, (5, 2, 16))
    a = rng.uniform(0, 6, (9, 6))
    pos = rng.integers(0, 9, (2, 5))
    for halves in (False, True):
        y, _ = R.turned(x, None, 0.0, np.cos(a), np.sin(a), pos, [2, 4], halves)
        assert np.allclose((y ** 2).sum(-1), (x ** 2).sum(-1)) and np.array_equal(y[..., 12:], x[..., 12:])
        z = (x[..., :6] + 1j * x[..., 6:12]) if halves else x[..., 0:12:2] + 1j * x[..., 1:12:2]
        ang = np.concatenate([a[pos[0], :2], a[pos[1], 2:]], 1)[:, None]
        w = z * np.exp(1j * ang)
        got = (y[..., :6] + 1j * y[..., 6:12]) if halves else y[..., 0:12:2] + 1j * y[..., 1:12:2]
        assert np.allclose(got, w)


def test_plain_attention_and_received_weights_agree():
    rng = np.random.default_rng(1)
    q, k, v = rng.normal(0, 1, (6, 8)), rng.normal(0, 1, (10, 8)), rng.normal(0, 1, (10, 8))
    see = R.visible(4, 6, 10, prefix=2, window=3)
    assert see[0].tolist() == [True, True, True, True, True] + [False] * 5
    assert R.visible(-2, 3, 4).sum() == 1 and not R.visible(-2, 3, 4)[:2].any()
    S = R.Scores(q, k, np.arange(4, 10), torch.float32, torch.float16, cap=5.0, slope=0.1)
    out, bound, lse, _ = R.attention(S, v, see, torch.float32, torch.float16)
    w, _ = R.received(S, lse, see)
    assert np.isclose(w.sum(), 6) and (bound < 1e-3).all()
    assert np.allclose(out[0], np.exp(S.s[0, :5] - lse[0]) @ v[:5])


def test_plain_eviction():
    m = np.array([1.0, 3.0, 3.0, np.nan, 0.5, 3.0, 9.0, 9.0])
    assert R.evict(m, 8, 4, 2) == [1, 2, 6, 7]
    assert R.evict(m, 6, 8, 0) == [0, 1, 2, 3, 4, 5]
    assert R.evict(m, 6, 5, 0) == [0, 1, 2, 4, 5]
    assert R.evict(m, 8, 3, 3) == [5, 6, 7] and R.evict(m, 0, 3, 3) == []


def test_structs_are_laid_out_as_in_the_header(tmp_path):
    import os
    import subprocess

    from smallmind_amd import _lib
    structs = {"smx_rotation": _lib.RotationC, "smx_attention_rules": _lib.AttentionRulesC}
    src = tmp_path / "layout.c"
    src.write_text("#include <stddef.h>\n#include <stdio.h>\n#include \"smx.h\"\nint main(void) {\n" + "".join(
        f'printf("%d\\n", (int)sizeof({n}));\n' + "".join(f'printf("%d\\n", (int)offsetof({n}, {f}));\n' for f, _ in c._fields_)
        for n, c in structs.items()) + "return 0; }\n")
    include = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include")
    subprocess.run(["gcc", "-std=c99", "-I", include, str(src), "-o", str(tmp_path / "layout")], check=True, capture_output=True)
    got = [int(x) for x in subprocess.run([str(tmp_path / "layout")], check=True, capture_output=True, text=True).stdout.split()]
    want = []
    for c in structs.values():
        want += [ctypes.sizeof(c)] + [getattr(c, f).offset for f, _ in c._fields_]
    assert got == want


def test_the_documented_calls_fit_the_binding():
    """The C# sample of the paged operators: each call's arguments by number and kind, and names that the binding has."""
    import os
    import re
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    cs = open(os.path.join(root, "smallmind_amd", "bindings", "csharp", "Smx.cs")).read()
    text = open(os.path.join(root, "INTEGRATION.md")).read()
    block = next(b for b in re.findall(r"```csharp\n(.*?)```", text, re.S) if "smx_paged_cache_create" in b)
    block = re.sub(r"//[^\n]*", "", block)
    assert "SMX_TYPE" not in block
    for struct, field in (("Rotation", "CosDev SinDev NPos NRot Halves NAxes"), ("AttentionRules", "Window")):
        body = re.search(r"public struct %s\b.*?\n        \}" % struct, cs, re.S).group(0)
        used = re.search(r"new %s \{(.*?)\}" % struct, block).group(1)
        assert re.findall(r"(\w+) =", used) == field.split() and all(re.search(r"\b%s\b" % f, body) for f in field.split())
    calls = re.findall(r"(smx_\w+)\((.*?)\);", block, re.S)
    assert len(calls) == 7
    for name, args in calls:
        params = re.search(r"extern int %s\((.*?)\);" % name, cs, re.S).group(1).split(",")
        args = args.split(",")
        assert len(args) == len(params), name
        for a, p in zip(args, params):
            kinds = [w for w in ("ref", "out", "in") if w in p.split()], [w for w in ("ref", "out", "in") if w in a.split()]
            assert kinds[0] == kinds[1], (name, a, p)
