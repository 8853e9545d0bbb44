"""Refusals of the serving operators that need no device, and the plain forms' own closed cases."""
import ctypes

import numpy as np
import pytest

from tests import kv_reference as R

P = ctypes.c_void_p(256)   # never followed: the call is refused first


@pytest.fixture(scope="module")
def lib():
    from smallmind_amd import _lib
    return _lib.load()


@pytest.mark.parametrize("args,code", [((0, 4, 64, 64), -1), ((1, 0, 64, 64), -1), ((1, 4, 64, 0), -1), ((-1, 4, 64, 64), -1),
                                       ((1, 4, 0, 64), -5), ((1, 4, 60, 64), -5), ((1, 4, 264, 64), -5),
                                       ((1, 4, 64, (1 << 24) + 1), -5), ((1, 65536, 64, 64), -5),
                                       (((1 << 24) + 1, 1, 64, 64), -5), ((1 << 24, 65535, 256, 1 << 24), -2)])
def test_cache_create_refuses(lib, args, code):
    h = ctypes.c_void_p(77)
    assert lib.smx_kv_cache_create(*args, ctypes.byref(h)) == code
    assert h.value is None
    assert lib.smx_last_error()


def test_null_arguments_are_refused(lib):
    assert lib.smx_kv_cache_create(1, 1, 64, 64, None) == -1
    assert lib.smx_kv_cache_info(None, None, None, None, None, None) == -1
    assert lib.smx_kv_cache_destroy(None) == 0
    assert lib.smx_kv_append(None, P, 64, P, 64, P, P, 1, None) == -1
    assert lib.smx_kv_read(None, P, P, 1, P, P, None) == -1
    n = ctypes.c_int64()
    assert lib.smx_attention_work_bytes(None, 1, 1, 1, 0, 64, ctypes.byref(n)) == -1
    assert lib.smx_attention_cached(None, P, 64, P, 1, 1, 1, P, P, 64, P, 1 << 20, None) == -1
    assert lib.smx_attention_shared(None, P, 64, P, 1, 1, 1, 0, 64, P, P, 64, P, 1 << 20, None) == -1


def test_verify_draft_refuses(lib):
    def run(target=P, ts=100, draft=P, ds=100, tokens=P, u=P, ud=P, n_seq=2, n_draft=3, vocab=100, out=P, acc=P):
        return lib.smx_verify_draft(target, ts, draft, ds, tokens, None, u, ud, n_seq, n_draft, vocab, out, acc, None)
    for bad in (dict(target=None), dict(tokens=None), dict(u=None), dict(ud=None), dict(out=None), dict(acc=None),
                dict(n_seq=0), dict(n_draft=-1), dict(n_draft=65536), dict(vocab=0), dict(vocab=(1 << 24) + 1, ts=1 << 25, ds=1 << 25),
                dict(ts=99), dict(ds=99), dict(target=ctypes.c_void_p(258)), dict(draft=ctypes.c_void_p(257))):
        assert run(**bad) == -1, bad
        assert b"smx_verify_draft" in lib.smx_last_error()


def test_plain_rows():
    c, s = R.encode(np.array([[127.0, 0.5, 1.5, -2.5, -126.6], [0, 0, 0, 0, 0]], np.float32))
    assert s.tolist() == [1.0, 0.0] and c[0].tolist() == [127, 0, 2, -2, -127] and not c[1].any()
    c, s = R.encode(np.array([[1.0, np.inf], [np.nan, 2.0]], np.float32))
    assert np.isnan(s).all() and not c.any()


def test_plain_attention_is_the_mean_for_equal_scores():
    v = np.arange(12, dtype=np.float64).reshape(4, 3)
    out, _ = R.attention(np.zeros((2, 3)), np.ones((4, 3)), v, np.array([[1, 1, 0, 0], [0, 0, 0, 0]], bool))
    assert np.allclose(out, [v[:2].mean(0), [0, 0, 0]])


def test_plain_verification_keeps_the_target_distribution():
    # over a grid of the three random numbers the first token is distributed as the target has it
    p, q = np.array([0.5, 0.2, 0.3]), np.array([0.2, 0.6, 0.2])
    grid = (np.arange(60) + 0.5) / 60
    count = np.zeros(3)
    for uq in grid:
        x = int(np.searchsorted(np.cumsum(q), uq, side="right"))
        for ua in grid:
            out, acc = R.verify(np.stack([p, p])[None], q[None, None], np.array([[x]]), np.array([[ua]]), np.array([0.5]),
                                None, 3)
            if acc[0]:
                count[x] += 60
            else:
                for ud in grid:
                    o, _ = R.verify(np.stack([p, p])[None], q[None, None], np.array([[x]]), np.array([[ua]]),
                                    np.array([ud]), None, 3)
                    count[o[0, 0]] += 1
    assert np.allclose(count / count.sum(), p, atol=0.01)


BIG = (1 << 32) + 1    # a C int takes it for 1


@pytest.mark.parametrize("at", range(4))
def test_cache_sizes_past_32_bits_are_refused(at):
    from smallmind_amd.quantization import GpuKvCache
    sizes = [1, 1, 64, 64]
    sizes[at] += BIG - 1
    with pytest.raises(ValueError, match="out of range"):
        GpuKvCache(*sizes)


@pytest.mark.parametrize("prefix,max_len", [((BIG, 10), 64), ((0, BIG), 64), ((0, -BIG), 64), ((0, 10), BIG), ((), BIG), ((), 1 << 31)])
def test_lengths_past_32_bits_are_refused(prefix, max_len):
    import types

    import torch

    from smallmind_amd import quantization as Q
    cache = types.SimpleNamespace(device=torch.device("cuda", 0), head_dim=64, ctx=64, _handle=lambda: None)
    q, i = torch.zeros(1, 1, 1, 64), torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ValueError, match="out of range"):
        if prefix:
            Q.attention_shared(q, cache, *prefix, i, i, max_len)
        else:
            Q.attention_cached(q, cache, i, i, max_len)


def test_verify_sizes_past_32_bits_are_refused(monkeypatch):
    import torch

    from smallmind_amd import quantization as Q
    for shape in ((1, 1, BIG), (BIG, 1, 1), (1, BIG + 1, 1)):
        t = torch.empty(1).expand(shape)
        monkeypatch.setattr(torch.Tensor, "get_device", lambda self: 0)
        with pytest.raises(ValueError, match="out of range"):
            Q.verify_draft(t, None, None, None, None)
        monkeypatch.undo()
