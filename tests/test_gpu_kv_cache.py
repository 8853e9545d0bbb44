"""The 8-bit KV cache, the attention over it and the verification of drafted tokens on the GPU, against
plain 64-bit forms."""
import ctypes
import math

import numpy as np
import pytest

from tests import kv_reference as R

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def Q(gpu):
    from smallmind_amd import quantization
    return quantization


def dev(a, dtype=None):
    import torch
    return torch.from_numpy(np.ascontiguousarray(a if dtype is None else np.asarray(a, dtype))).cuda()


def i32(a):
    return dev(a, np.int32)


# ---- rows written and read back -------------------------------------------------------------------
def places(kind, n, slots, ctx, rng):
    """n distinct places of a cache as callers come with them."""
    if kind == "run":           # a prompt behind an odd number of positions
        return np.full(n, slots - 1), 3 + np.arange(n)
    if kind == "aligned":
        return np.full(n, 0), np.arange(n)
    if kind == "batch":         # a token for each of many sequences, positions all over
        return np.arange(n) % slots, (np.arange(n) // slots * 5 + 7 * (np.arange(n) % slots)) % ctx
    if kind == "runs":          # several tokens for each of several sequences
        return np.arange(n) // 5 % slots, (np.arange(n) % 5 + 1 + 5 * (np.arange(n) // 5 // slots)) % ctx
    p = rng.permutation(slots * ctx)[:n]
    return p // ctx, p % ctx


@pytest.mark.parametrize("hd", [8, 16, 32, 40, 64, 80, 96, 128, 136, 160, 192, 208, 224, 256])
@pytest.mark.parametrize("kind,n", [("run", 1), ("run", 131), ("aligned", 64), ("batch", 17), ("runs", 93), ("random", 150)])
def test_rows_come_back_as_they_were_encoded(Q, hd, kind, n):
    rng = np.random.default_rng(hd * 1000 + n)
    kv, slots, ctx = 3, 19, 150
    s, p = places(kind, n, slots, ctx, rng)
    assert len({(a, b) for a, b in zip(s.tolist(), p.tolist())}) == n
    k = (rng.normal(0, 1, (n, kv, hd)) * np.exp2(rng.integers(-20, 20, (n, kv, 1)))).astype(np.float32)
    v = rng.normal(0, 2, (n, kv, hd)).astype(np.float32)
    c = Q.GpuKvCache(slots, kv, hd, ctx)
    c.append(dev(k), dev(v), i32(s), i32(p))
    all_s, all_p = np.repeat(np.arange(slots), ctx), np.tile(np.arange(ctx), slots)
    gk, gv = c.read(i32(all_s), i32(all_p))
    ek, ev = np.zeros((slots, ctx, kv, hd), np.float32), np.zeros((slots, ctx, kv, hd), np.float32)
    ek[s, p], ev[s, p] = R.held(k), R.held(v)
    assert np.array_equal(gk.cpu().numpy().reshape(ek.shape), ek)
    assert np.array_equal(gv.cpu().numpy().reshape(ev.shape), ev)
    c.close()


@pytest.mark.parametrize("hd,kv", [(8, 2), (64, 2), (128, 3), (256, 3), (232, 2)])
@pytest.mark.parametrize("kind", ["prompts", "mixed"])
def test_many_rows(Q, hd, kv, kind):
    """Enough rows for the kernels of many (and of more than the caches hold): runs of odd lengths at odd
    positions, and runs among single tokens and places that do not exist."""
    import torch
    rng = np.random.default_rng(hd + kv)
    slots, per, ctx = 9, 1001, 1100
    n = slots * per
    s, p = np.repeat(np.arange(slots), per), np.tile(np.arange(per) + 33, slots)
    if kind == "mixed":
        order = np.arange(n)
        for a in range(0, n, 700):      # every few hundred tokens, 90 in another order
            b = min(n, a + 90)
            order[a:b] = rng.permutation(order[a:b])
        s, p = s[order].copy(), p[order].copy()
        s[::97], p[::89] = -1, ctx
    k, v = (rng.normal(0, 1, (n, kv, hd)).astype(np.float32) for _ in range(2))
    c = Q.GpuKvCache(slots, kv, hd, ctx)
    c.append(dev(k), dev(v), i32(s), i32(p))
    gk, gv = c.read(i32(s), i32(p))
    ok = (s >= 0) & (p < ctx)
    for g, x in ((gk, k), (gv, v)):
        assert np.array_equal(g.cpu().numpy(), np.where(ok[:, None, None], R.held(x), np.float32(0)))
    # nothing else was written
    gk, gv = c.read(i32(np.repeat(np.arange(slots), ctx)), i32(np.tile(np.arange(ctx), slots)))
    seen = np.zeros((slots, ctx), bool)
    seen[s[ok], p[ok]] = True
    for g in (gk, gv):
        rows = (g.abs().amax((1, 2)) > 0).cpu().numpy().reshape(slots, ctx)
        assert np.array_equal(rows, seen)
    c.close()
    torch.cuda.empty_cache()


def test_places_that_the_cache_does_not_have(Q):
    rng = np.random.default_rng(3)
    c = Q.GpuKvCache(2, 2, 64, 70)
    s = np.array([0, -1, 2, 1, 1, 1, 0, 0, 2**31 - 1, -2**31])
    p = np.array([5, 5, 5, -1, 70, 69, 6, 2**31 - 1, 0, -2**31])
    k, v = (rng.normal(0, 1, (10, 2, 64)).astype(np.float32) for _ in range(2))
    c.append(dev(k), dev(v), i32(s), i32(p))
    ok = [0, 5, 6]
    gk, gv = c.read(i32(s), i32(p))
    for g, x in ((gk, k), (gv, v)):
        e = np.zeros_like(x)
        e[ok] = R.held(x[ok])
        assert np.array_equal(g.cpu().numpy(), e)
    gk, _ = c.read(i32(np.repeat([0, 1], 70)), i32(np.tile(np.arange(70), 2)))
    assert int((gk.abs().sum((1, 2)) > 0).sum()) == 3
    c.close()


def test_values_next_to_a_border(Q):
    """Multiples and halves of a step and their neighbours in fp32, for scales of every size."""
    rows = []
    for top in (127.0, 1.0, 3.7e-3, 2.0 ** -120, 127 * 2.0 ** -149, 190 * 2.0 ** -149, 2.0 ** -149, 3.0e38, 1e-30, 88.3):
        top = np.float32(top)
        step = np.float32(np.float64(top) / 127)
        h = ((np.arange(-126, 126) + 0.5) * np.float64(step)).astype(np.float32)
        h = np.concatenate([h, np.nextafter(h, np.float32(np.inf)), np.nextafter(h, np.float32(-np.inf)),
                            (np.arange(-126, 127) * np.float64(step)).astype(np.float32)])
        h = np.clip(h, -top, top)
        h = np.concatenate([h, np.zeros(-len(h) % 63, np.float32)]).reshape(-1, 63)
        rows.append(np.concatenate([np.full((len(h), 1), top, np.float32), h], 1))
    x = np.concatenate(rows)[:, None]
    n = len(x)
    c = Q.GpuKvCache(1, 1, 64, n)
    c.append(dev(x), dev(-x), i32(np.zeros(n)), i32(np.arange(n)))
    k, v = c.read(i32(np.zeros(n)), i32(np.arange(n)))
    assert np.array_equal(k.cpu().numpy(), R.held(x)) and np.array_equal(v.cpu().numpy(), R.held(-x))
    c.close()


def test_rows_that_are_not_finite(Q):
    rng = np.random.default_rng(8)
    x = rng.normal(0, 1, (6, 2, 64)).astype(np.float32)
    x[1, 0, 63], x[2, 1, 0], x[4, 0, 5], x[5, :, :] = np.nan, np.inf, -np.inf, 0.0
    c = Q.GpuKvCache(1, 2, 64, 64)
    c.append(dev(x), dev(x), i32(np.zeros(6)), i32(np.arange(6)))
    k, v = c.read(i32(np.zeros(6)), i32(np.arange(6)))
    e = R.held(x)
    assert np.isnan(e[1, 0]).all() and not np.isnan(e[1, 1]).any()
    assert np.array_equal(k.cpu().numpy(), e, equal_nan=True) and np.array_equal(v.cpu().numpy(), e, equal_nan=True)
    c.close()


@pytest.mark.parametrize("hd,off", [(64, 0), (64, 1), (40, 3), (128, 2)])
def test_rows_of_a_fused_projection(Q, hd, off):
    import torch
    rng = np.random.default_rng(hd + off)
    n, heads, kv = 70, 4, 2
    width = (heads + 2 * kv) * hd + 5
    buf = dev(rng.normal(0, 1, n * width + off).astype(np.float32))
    f = buf[off:].view(n, width)
    k, v = f[:, heads * hd:(heads + kv) * hd].unflatten(1, (kv, hd)), f[:, (heads + kv) * hd:(heads + 2 * kv) * hd].unflatten(1, (kv, hd))
    c = Q.GpuKvCache(1, kv, hd, n)
    at = i32(np.arange(n))
    c.append(k, v, torch.zeros_like(at), at)
    gk, gv = c.read(torch.zeros_like(at), at)
    assert np.array_equal(gk.cpu().numpy(), R.held(k.cpu().numpy())) and np.array_equal(gv.cpu().numpy(), R.held(v.cpu().numpy()))
    c.close()


def test_a_cache_of_more_than_4_gib(Q):
    import torch
    rng = np.random.default_rng(4)
    c = Q.GpuKvCache(9, 8, 128, 262144)     # 4.9 GB
    assert c.nbytes > (1 << 32)
    s, p = np.array([8, 8, 8, 0, 7, 8, 8]), np.array([262143, 262142, 0, 262143, 100000, 131072, 200001])
    k, v = (rng.normal(0, 1, (7, 8, 128)).astype(np.float32) for _ in range(2))
    c.append(dev(k), dev(v), i32(s), i32(p))
    gk, gv = c.read(i32(s), i32(p))
    assert np.array_equal(gk.cpu().numpy(), R.held(k)) and np.array_equal(gv.cpu().numpy(), R.held(v))
    # attention over all of the last slot: the zeros of the positions never written weigh equally
    q = rng.normal(0, 1, (1, 1, 8, 128)).astype(np.float32)
    out = Q.attention_cached(dev(q), c, i32([8]), i32([262144])).cpu().numpy()
    hk, hv = R.held(k).astype(np.float64), R.held(v).astype(np.float64)
    for h in range(8):
        rows = [0, 1, 2, 5, 6]
        w = np.exp(hk[rows, h] @ q[0, 0, h].astype(np.float64) / np.sqrt(128))
        ref = w @ hv[rows, h] / (w.sum() + 262144 - len(rows))
        # weights and their sum: 262144 terms in fp32 parts of 64 positions and more
        assert np.abs(out[0, 0, h] - ref).max() <= 1e-3 * np.abs(ref).max()
    c.close()
    torch.cuda.empty_cache()


# ---- attention ------------------------------------------------------------------------------------
class Filled:
    """A cache whose slots hold random rows, and what they stand for."""

    def __init__(self, Q, slots, kv, hd, ctx, seed, spread=1.0):
        rng = np.random.default_rng(seed)
        self.k = rng.normal(0, spread, (slots, ctx, kv, hd)).astype(np.float32)
        self.v = (rng.normal(0, 1, (slots, ctx, kv, hd)) * np.exp2(rng.integers(-3, 4, (slots, ctx, kv, 1)))).astype(np.float32)
        self.cache = Q.GpuKvCache(slots, kv, hd, ctx)
        n = slots * ctx
        self.cache.append(dev(self.k.reshape(n, kv, hd)), dev(self.v.reshape(n, kv, hd)), i32(np.repeat(np.arange(slots), ctx)),
                          i32(np.tile(np.arange(ctx), slots)))
        self.hk, self.hv = R.held(self.k), R.held(self.v)


def reference(f, q, slots, lens, prefix=None, max_len=None):
    n_seq, n_q, H, hd = q.shape
    kv = f.k.shape[2]
    G = H // kv
    out, bound = np.zeros(q.shape), np.zeros((n_seq, n_q, H))
    for b in range(n_seq):
        if not 0 <= slots[b] < f.k.shape[0]:
            continue
        n = max(0, min(int(lens[b]), f.k.shape[1] if max_len is None else max_len))
        for h in range(kv):
            k, v = f.hk[slots[b], :n, h], f.hv[slots[b], :n, h]
            P = 0
            if prefix:
                P = prefix[1]
                k, v = np.concatenate([f.hk[prefix[0], :P, h], k]), np.concatenate([f.hv[prefix[0], :P, h], v])
            for i in range(n_q):
                vis = np.zeros((G, P + n), bool)
                vis[:, :P + max(0, n - n_q + 1 + i)] = True
                o, e = R.attention(q[b, i, h * G:(h + 1) * G], k, v, vis)
                out[b, i, h * G:(h + 1) * G], bound[b, i, h * G:(h + 1) * G] = o, e
    return out, bound


def close(got, want):
    ref, bound = want
    err = np.abs(got.cpu().numpy().astype(np.float64) - ref).max(-1)
    assert (err <= bound).all(), (float((err - bound).max()), np.unravel_index((err - bound).argmax(), err.shape))


@pytest.mark.parametrize("hd", [8, 32, 40, 64, 80, 96, 128, 160, 192, 224, 256])
@pytest.mark.parametrize("group,n_q", [(1, 1), (3, 1), (8, 1), (1, 5), (5, 4), (4, 9), (20, 1), (7, 11)])
def test_attention_cached(Q, hd, group, n_q):
    f = Filled(Q, 7, 2, hd, 330, hd + group + n_q)
    rng = np.random.default_rng(hd * group + n_q)
    lens = np.array([1, 64, 0, 330, 65, 256, 63])
    slots = np.array([6, 0, 1, 2, 3, 4, 5])
    q = rng.normal(0, 1.3, (7, n_q, 2 * group, hd)).astype(np.float32)
    got = Q.attention_cached(dev(q), f.cache, i32(slots), i32(lens))
    close(got, reference(f, q, slots, lens))
    assert not got[2].any()
    f.cache.close()


@pytest.mark.parametrize("hd", [32, 64, 80, 128, 256])
@pytest.mark.parametrize("group,n_q,n_seq", [(1, 1, 1), (1, 1, 5), (4, 1, 9), (2, 3, 7), (8, 4, 3)])
@pytest.mark.parametrize("P", [1, 64, 129, 600])
def test_attention_shared(Q, hd, group, n_q, n_seq, P):
    f = Filled(Q, n_seq + 1, 2, hd, 600, hd + group + n_q + P)
    rng = np.random.default_rng(hd * group + n_q + P)
    lens = np.array([0, 70, 1, 300, 64, 5, 0, 11, 2])[:n_seq]
    slots = np.arange(n_seq)[::-1].copy()
    q = rng.normal(0, 1.3, (n_seq, n_q, 2 * group, hd)).astype(np.float32)
    got = Q.attention_shared(dev(q), f.cache, n_seq, P, i32(slots), i32(lens), 300)
    close(got, reference(f, q, slots, lens, (n_seq, P)))
    f.cache.close()


@pytest.mark.parametrize("hd", [8, 96, 160, 192, 224])
@pytest.mark.parametrize("group,n_q,n_seq,P", [(8, 4, 3, 129), (4, 1, 5, 600), (3, 2, 1, 64), (1, 7, 11, 200)])
def test_attention_shared_at_other_widths(Q, hd, group, n_q, n_seq, P):
    f = Filled(Q, n_seq + 1, 2, hd, 600, hd + P)
    rng = np.random.default_rng(hd * group + P)
    lens = np.array([9, 70, 0, 300, 64, 5, 1, 11, 2, 63, 65])[:n_seq]
    slots = np.arange(n_seq)
    q = rng.normal(0, 1.3, (n_seq, n_q, 2 * group, hd)).astype(np.float32)
    close(Q.attention_shared(dev(q), f.cache, n_seq, P, i32(slots), i32(lens), 300), reference(f, q, slots, lens, (n_seq, P)))
    f.cache.close()


def test_more_new_tokens_than_positions_and_many_of_them(Q):
    """A prompt's chunk of 150 tokens of several lengths: blocks of rows that see nothing, part of a chunk, all."""
    f = Filled(Q, 5, 1, 64, 700, 13)
    rng = np.random.default_rng(14)
    q = rng.normal(0, 1, (5, 150, 3, 64)).astype(np.float32)
    slots, lens = np.array([0, 1, 2, 3, 4]), np.array([700, 150, 20, 0, 151])
    close(Q.attention_cached(dev(q), f.cache, i32(slots), i32(lens)), reference(f, q, slots, lens))
    close(Q.attention_shared(dev(q), f.cache, 4, 77, i32(slots), i32(lens)), reference(f, q, slots, lens, (4, 77)))
    f.cache.close()


def test_a_cache_that_does_not_fit_leaves_no_error_behind(Q):
    from smallmind_amd._lib import SmxError
    with pytest.raises(SmxError):      # 145 TB
        Q.GpuKvCache(1 << 10, 64, 128, 1 << 23)
    c = Q.GpuKvCache(1, 1, 64, 8)
    x = np.ones((1, 1, 64), np.float32)
    c.append(dev(x), dev(x), i32([0]), i32([0]))
    assert np.array_equal(c.read(i32([0]), i32([0]))[0].cpu().numpy(), R.held(x))
    c.close()


def test_more_than_a_launch_takes_is_refused(Q):
    """Sizes whose grids pass 2^32 threads; nothing is launched."""
    import torch

    from smallmind_amd._lib import load
    L, c = load(), Q.GpuKvCache(1, 1, 8, 4096)
    t = torch.zeros(4096, device="cuda")
    i = torch.zeros(64, dtype=torch.int32, device="cuda")
    for n_tok in (2**31 - 1, 2**31 - 64, 2**30, 2**29):
        assert L.smx_kv_append(c._h, t.data_ptr(), 8, t.data_ptr(), 8, i.data_ptr(), i.data_ptr(), n_tok, None) == -1
        assert L.smx_kv_read(c._h, i.data_ptr(), i.data_ptr(), n_tok, t.data_ptr(), t.data_ptr(), None) == -1
    n = ctypes.c_int64()
    for n_seq, n_q, P, code in ((2**24, 1, 0, -5), (2**24 - 1, 1, 0, 0), (2**24 - 1, 1, 64, -5), (2**23, 8, 64, 0)):
        assert L.smx_attention_work_bytes(c._h, n_seq, n_q, 1, P, 64, ctypes.byref(n)) == code, (n_seq, n_q, P)
    assert L.smx_verify_draft(t.data_ptr(), 8, None, 8, i.data_ptr(), None, t.data_ptr(), t.data_ptr(), 2**22, 1, 8, i.data_ptr(),
                              i.data_ptr(), None) == -5
    c.close()


@pytest.mark.parametrize("hd", [64, 256])
@pytest.mark.parametrize("k_up,q_up,v_up", [(96, -96, 96), (-90, 90, -80), (60, -50, 0)])
def test_sizes_next_to_the_documented_limits(Q, hd, k_up, q_up, v_up):
    rng = np.random.default_rng([hd, k_up + 128])
    f = Filled(Q, 2, 2, hd, 200, hd)
    unit = (rng.uniform(-1, 1, s).astype(np.float32) for s in ((2, 200, 2, hd), (2, 200, 2, hd), (2, 3, 6, hd)))
    f.k, f.v, q = (x * np.float32(2.0 ** up) for x, up in zip(unit, (k_up, v_up, q_up)))
    f.cache.append(dev(f.k.reshape(400, 2, hd)), dev(f.v.reshape(400, 2, hd)), i32(np.repeat([0, 1], 200)),
                   i32(np.tile(np.arange(200), 2)))
    f.hk, f.hv = R.held(f.k), R.held(f.v)
    close(Q.attention_cached(dev(q), f.cache, i32([0, 1]), i32([200, 77])), reference(f, q, [0, 1], [200, 77]))
    close(Q.attention_shared(dev(q), f.cache, 1, 130, i32([0, 1]), i32([200, 77])),
          reference(f, q, [0, 1], [200, 77], (1, 130)))
    f.cache.close()


def test_one_slot_for_many_sequences(Q):
    """600 sequences in three slots: the form for more than the caches hold, and equal rows give equal outputs."""
    import torch
    f = Filled(Q, 3, 2, 128, 1000, 21)
    rng = np.random.default_rng(22)
    q = rng.normal(0, 1, (3, 1, 4, 128)).astype(np.float32)
    slots, lens = np.array([2, 0, 1]), np.array([1000, 517, 64])
    got = Q.attention_cached(dev(np.tile(q, (200, 1, 1, 1))), f.cache, i32(np.tile(slots, 200)), i32(np.tile(lens, 200)))
    got = got.reshape(200, 3, 1, 4, 128)
    assert torch.equal(got, got[:1].expand_as(got))
    close(got[0], reference(f, q, slots, lens))
    f.cache.close()


@pytest.mark.parametrize("P", [0, 130])
@pytest.mark.parametrize("length", [40, 2000])
def test_outputs_that_are_not_aligned(Q, P, length):
    import torch

    from smallmind_amd._lib import call
    f = Filled(Q, 2, 1, 64, 2000, 23)
    rng = np.random.default_rng(24)
    q = rng.normal(0, 1, (1, 2, 4, 64)).astype(np.float32)
    n = ctypes.c_int64()
    call("smx_attention_work_bytes", f.cache._h, 1, 2, 4, P, length, ctypes.byref(n))
    work = torch.empty(n.value + 16, dtype=torch.uint8, device="cuda")
    buf = torch.full((1 + q.size + 8,), 7.0, device="cuda")
    dq, slots, lens = dev(q), i32([0]), i32([length])
    call("smx_attention_shared", f.cache._h, dq.data_ptr(), 256, buf[1:].data_ptr(), 1, 2, 4, 1, P, slots.data_ptr(),
         lens.data_ptr(), length, work.data_ptr(), n.value, None)
    torch.cuda.synchronize()
    assert bool((buf[0] == 7.0) & (buf[1 + q.size:] == 7.0).all())
    close(buf[1:1 + q.size].reshape(q.shape), reference(f, q, [0], [length], (1, P) if P else None))
    f.cache.close()


def test_calls_from_several_threads(Q):
    import threading

    import torch
    f = Filled(Q, 5, 2, 64, 400, 15)
    q = torch.randn(4, 2, 8, 64, device="cuda")
    slots, lens = i32([0, 1, 2, 3]), i32([400, 7, 130, 64])
    want = Q.attention_shared(q, f.cache, 4, 300, slots, lens)
    torch.cuda.synchronize()
    bad = []

    def work():
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                got = Q.attention_shared(q, f.cache, 4, 300, slots, lens)
                torch.cuda.current_stream().synchronize()
                if not bool((got == want).all()):
                    bad.append(1)
    threads = [threading.Thread(target=work) for _ in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad
    f.cache.close()


def test_attention_over_a_prefix_alone_and_over_none(Q):
    f = Filled(Q, 4, 2, 64, 500, 9)
    rng = np.random.default_rng(1)
    q = rng.normal(0, 1, (3, 2, 8, 64)).astype(np.float32)
    slots, lens = np.array([0, -1, 2]), np.array([400, 400, 7])
    for P in (100, 500):
        close(Q.attention_shared(dev(q), f.cache, 3, P, i32(slots), i32(lens), 0), reference(f, q, slots, lens, (3, P), 0))
    a = Q.attention_shared(dev(q), f.cache, 3, 0, i32(slots), i32(lens))
    b = Q.attention_cached(dev(q), f.cache, i32(slots), i32(lens))
    assert bool((a == b).all()) and not b[1].any()
    assert not Q.attention_cached(dev(q), f.cache, i32(slots), i32(lens), 0).any()
    f.cache.close()


def test_attention_of_many_lengths_of_one_sequence(Q):
    f = Filled(Q, 1, 1, 64, 1300, 12)
    rng = np.random.default_rng(2)
    lens = np.array([1, 2, 15, 16, 17, 31, 33, 48, 62, 63, 64, 65, 127, 128, 129, 255, 256, 257, 511, 513, 1023, 1025, 1299, 1300,
                     5000, -3])
    q = rng.normal(0, 2, (len(lens), 1, 2, 64)).astype(np.float32)
    slots = np.zeros(len(lens), int)
    close(Q.attention_cached(dev(q), f.cache, i32(slots), i32(lens)), reference(f, q, slots, lens))
    close(Q.attention_cached(dev(q), f.cache, i32(slots), i32(lens), 100), reference(f, q, slots, lens, None, 100))
    f.cache.close()


@pytest.mark.parametrize("spread", [0.0, 1e-12, 6.0, 300.0])
def test_attention_of_flat_and_sharp_scores(Q, spread):
    f = Filled(Q, 2, 2, 64, 700, 21, spread)
    rng = np.random.default_rng(5)
    q = rng.normal(0, 2, (2, 3, 4, 64)).astype(np.float32)
    slots, lens = np.array([0, 1]), np.array([700, 401])
    close(Q.attention_cached(dev(q), f.cache, i32(slots), i32(lens)), reference(f, q, slots, lens))
    close(Q.attention_shared(dev(q), f.cache, 1, 300, i32(slots), i32(lens)), reference(f, q, slots, lens, (1, 300)))
    f.cache.close()


def test_values_and_queries_of_very_different_sizes(Q):
    """Rows of V from 2^-40 to 2^40 beside one another, queries with one element far above the rest, tiny and
    huge ones: every row within its bound, which goes by the largest value that the row sees."""
    rng = np.random.default_rng(6)
    n, hd = 200, 64
    k = rng.normal(0, 1, (n, 1, hd)).astype(np.float32)
    v = (rng.normal(0, 1, (n, 1, hd)) * np.exp2(rng.integers(-40, 41, (n, 1, 1)))).astype(np.float32)
    f = Filled(Q, 1, 1, hd, n, 0)
    f.cache.append(dev(k), dev(v), i32(np.zeros(n)), i32(np.arange(n)))
    f.hk[0], f.hv[0] = R.held(k), R.held(v)
    q = rng.normal(0, 1, (5, 1, 1, hd)).astype(np.float32)
    q[1, 0, 0, 3] = 40.0
    q[2] *= 1e-30
    q[3] = 0.0
    q[4] *= 1e-42
    slots, lens = np.zeros(5, int), np.array([n, n, n, 70, 3])
    close(Q.attention_cached(dev(q), f.cache, i32(slots), i32(lens)), reference(f, q, slots, lens))
    f.cache.close()


def test_what_is_not_seen_does_not_count(Q):
    """NaN rows behind a sequence's length, in other slots, and at a drafted token that only later ones see."""
    f = Filled(Q, 3, 2, 64, 200, 31)
    nan = np.full((1, 2, 64), np.nan, np.float32)
    for p in (150, 151, 199):
        f.cache.append(dev(nan), dev(nan), i32([0]), i32([p]))
    f.cache.append(dev(nan), dev(nan), i32([1]), i32([0]))
    f.cache.append(dev(f.k[2, 88:89]), dev(nan), i32([2]), i32([88]))
    rng = np.random.default_rng(7)
    q = rng.normal(0, 1, (2, 4, 4, 64)).astype(np.float32)
    slots, lens = np.array([0, 2]), np.array([150, 90])
    got = Q.attention_cached(dev(q), f.cache, i32(slots), i32(lens)).cpu()
    ref, bound = reference(f, q, slots, lens)
    close(got[:1], (ref[:1], bound[:1]))
    close(got[1:, :2], (ref[1:, :2], bound[1:, :2]))        # these see positions 0 .. 87
    assert got[1, 2:].isnan().all()
    # a prefix with a NaN reaches every row, one behind its length none
    assert Q.attention_shared(dev(q), f.cache, 1, 10, i32(slots), i32(lens)).isnan().all()
    assert not Q.attention_shared(dev(q), f.cache, 0, 150, i32([2, 2]), i32([40, 3])).isnan().any()
    f.cache.close()


def test_a_query_that_is_not_finite_stays_alone(Q):
    f = Filled(Q, 2, 2, 64, 100, 33)
    rng = np.random.default_rng(8)
    q = rng.normal(0, 1, (2, 2, 8, 64)).astype(np.float32)
    slots, lens = np.array([0, 1]), np.array([100, 1])
    ref, bound = reference(f, q, slots, lens)
    q[0, 1, 3, 7], q[0, 0, 0, 0], q[1, 0, 2, 2] = np.inf, np.nan, np.nan
    got = Q.attention_cached(dev(q), f.cache, i32(slots), i32(lens)).cpu()
    assert got[0, 1, 3].isnan().all() and got[0, 0, 0].isnan().all()
    assert not got[1, 0].any()          # sees nothing
    ok = np.ones((2, 2, 8), bool)
    ok[0, 1, 3] = ok[0, 0, 0] = False
    err = np.abs(got.numpy() - ref).max(-1)
    assert (err[ok] <= bound[ok]).all()
    f.cache.close()


@pytest.mark.parametrize("off", [0, 1, 2])
def test_queries_in_the_rows_of_a_fused_projection(Q, off):
    f = Filled(Q, 4, 2, 64, 90, 35)
    rng = np.random.default_rng(9)
    width = (8 + 4) * 64 + off
    buf = dev(rng.normal(0, 1, 4 * 3 * width + off).astype(np.float32))[off:].view(4, 3, width)
    q = buf[:, :, :512].unflatten(2, (8, 64))
    slots, lens = np.arange(4), np.array([90, 3, 44, 70])
    close(Q.attention_cached(q, f.cache, i32(slots), i32(lens)), reference(f, q.cpu().numpy(), slots, lens))
    f.cache.close()


def test_rows_behind_the_outputs_and_the_work_memory_stay(Q):
    import torch

    from smallmind_amd._lib import call
    f = Filled(Q, 3, 2, 64, 600, 36)
    q = torch.randn(3, 2, 8, 64, device="cuda")
    slots, lens = i32([0, 1, 2]), i32([600, 0, 77])
    need = ctypes.c_int64()
    call("smx_attention_work_bytes", f.cache._h, 3, 2, 8, 500, 600, ctypes.byref(need))
    assert need.value > 0
    out = torch.full((q.numel() + 512,), 7.5, device="cuda")
    work = torch.full((need.value + 256,), 91, dtype=torch.uint8, device="cuda")
    call("smx_attention_shared", f.cache._h, q.data_ptr(), 512, out.data_ptr(), 3, 2, 8, 2, 500, slots.data_ptr(),
         lens.data_ptr(), 600, work.data_ptr(), need.value, None)
    torch.cuda.synchronize()
    assert bool((out[q.numel():] == 7.5).all()) and bool((work[need.value:] == 91).all())
    want = Q.attention_shared(q, f.cache, 2, 500, slots, lens)
    assert bool((out[:q.numel()] == want.reshape(-1)).all())
    f.cache.close()


def test_refusals(Q):
    import torch

    from smallmind_amd._lib import load
    L = load()
    c = Q.GpuKvCache(2, 2, 64, 128)
    t = torch.zeros(4096, device="cuda")
    i = torch.zeros(64, dtype=torch.int32, device="cuda")
    n = ctypes.c_int64()

    def cached(**k):
        a = dict(q=t.data_ptr(), stride=256, out=t.data_ptr(), n_seq=2, n_q=1, n_head=4, slots=i.data_ptr(), lens=i.data_ptr(),
                 max_len=128, work=None, bytes=0)
        a.update(k)
        return L.smx_attention_cached(c._h, *a.values(), None)

    def shared(slot, length, **k):
        a = dict(q=t.data_ptr(), stride=256, out=t.data_ptr(), n_seq=2, n_q=1, n_head=4, slot=slot, length=length,
                 slots=i.data_ptr(), lens=i.data_ptr(), max_len=128, work=None, bytes=0)
        a.update(k)
        return L.smx_attention_shared(c._h, *a.values(), None)

    for bad in (dict(q=None), dict(out=None), dict(slots=None), dict(lens=None), dict(stride=255), dict(n_seq=0), dict(n_q=0),
                dict(n_head=0), dict(n_head=5), dict(max_len=-1), dict(max_len=129), dict(q=t.data_ptr() + 2)):
        assert cached(**bad) == -1, bad
    assert cached(n_seq=2**30, n_head=64, stride=64 * 64) == -5
    assert shared(2, 10) == -1 and shared(-1, 10) == -1 and shared(0, 129) == -1 and shared(0, -1) == -1
    assert shared(0, 10) == -1 and b"work" in L.smx_last_error()
    assert shared(0, 10, work=t.data_ptr(), bytes=16) == -1
    assert L.smx_attention_work_bytes(c._h, 1, 1, 3, 0, 128, ctypes.byref(n)) == -1
    ap = lambda **k: L.smx_kv_append(c._h, *{**dict(k=t.data_ptr(), ks=128, v=t.data_ptr(), vs=128, s=i.data_ptr(),  # noqa: E731
                                                   p=i.data_ptr(), n=1), **k}.values(), None)
    for bad in (dict(k=None), dict(v=None), dict(s=None), dict(p=None), dict(ks=127), dict(vs=127), dict(n=-1), dict(k=t.data_ptr() + 1)):
        assert ap(**bad) == -1, bad
    assert ap(n=0) == 0
    with pytest.raises(ValueError):
        c.append(torch.zeros(3, 2, 64, device="cuda"), torch.zeros(3, 2, 64, device="cuda"), i[:2], i[:2])
    with pytest.raises(ValueError):
        c.append(torch.zeros(2, 2, 64, device="cuda").half(), torch.zeros(2, 2, 64, device="cuda"), i[:2], i[:2])
    with pytest.raises(ValueError):
        c.append(torch.zeros(2, 64, 2, device="cuda").transpose(1, 2), torch.zeros(2, 2, 64, device="cuda"), i[:2], i[:2])
    with pytest.raises(ValueError):
        c.append(torch.zeros(2, 2, 64), torch.zeros(2, 2, 64, device="cuda"), i[:2], i[:2])
    with pytest.raises(ValueError):
        Q.attention_cached(torch.zeros(2, 1, 4, 64, device="cuda"), c, i[:2].long(), i[:2])
    with pytest.raises(ValueError):
        Q.attention_cached(torch.zeros(2, 1, 4, 32, device="cuda"), c, i[:2], i[:2])
    with pytest.raises(ValueError):
        Q.attention_cached(torch.zeros(2, 1, 1, 4, 64, device="cuda")[0], c, i[:2], i[:2])
    c.close()
    with pytest.raises(ValueError):
        c.read(i[:1], i[:1])
    with pytest.raises(Q.SmxError):
        Q.GpuKvCache(1, 1, 63, 64)


def test_calls_on_other_streams_and_again(Q):
    """The same call gives the same bits, on any stream, with other calls in flight."""
    import torch
    f = Filled(Q, 6, 2, 128, 900, 41)
    q = torch.randn(5, 2, 8, 128, device="cuda")
    slots, lens = i32(np.arange(5)), i32([900, 1, 333, 64, 257])
    want = Q.attention_shared(q, f.cache, 5, 700, slots, lens)
    plain = Q.attention_cached(q, f.cache, slots, lens)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for _ in range(4):
        for s in streams:
            with torch.cuda.stream(s):
                got.append((Q.attention_shared(q, f.cache, 5, 700, slots, lens), Q.attention_cached(q, f.cache, slots, lens)))
    torch.cuda.synchronize()
    assert all(bool((a == want).all()) and bool((b == plain).all()) for a, b in got)
    f.cache.close()


def test_captured_steps_replay(Q):
    """Two captured graphs, each writing a token of its sequences and attending, replayed in turn with eager work
    between: lengths and positions are read on the device, so every replay is the next step."""
    import torch
    rng = np.random.default_rng(50)
    hd, kv, H, n = 64, 2, 6, 3
    f = Filled(Q, 2 * n + 1, kv, hd, 320, 51)
    steps = 5
    xk, xv = (rng.normal(0, 1, (2, steps, n, kv, hd)).astype(np.float32) for _ in range(2))
    xq = rng.normal(0, 1, (2, steps, n, 1, H, hd)).astype(np.float32)
    start = np.array([[63, 0, 310], [127, 255, 5]])
    state = []
    for gi in range(2):
        st = dict(k=dev(xk[gi, 0]), v=dev(xv[gi, 0]), q=dev(xq[gi, 0]), slots=i32(np.arange(n) + gi * n), pos=i32(start[gi]),
                  lens=i32(start[gi] + 1))
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        g = torch.cuda.CUDAGraph()
        with torch.cuda.stream(s):
            Q.attention_shared(st["q"], f.cache, 2 * n, 300, st["slots"], st["lens"])
        torch.cuda.synchronize()
        with torch.cuda.graph(g, stream=s):
            f.cache.append(st["k"], st["v"], st["slots"], st["pos"])
            st["out"] = Q.attention_shared(st["q"], f.cache, 2 * n, 300, st["slots"], st["lens"])
            st["pos"].add_(1)
            st["lens"].add_(1)
        st["graph"] = g
        state.append(st)
    for step in range(steps):
        for gi, st in enumerate(state):
            st["k"].copy_(dev(xk[gi, step]))
            st["v"].copy_(dev(xv[gi, step]))
            st["q"].copy_(dev(xq[gi, step]))
            st["graph"].replay()
        Q.attention_cached(state[0]["q"], f.cache, state[0]["slots"], state[0]["lens"])     # eager work between replays
        torch.cuda.synchronize()
        for gi, st in enumerate(state):
            sl = np.arange(n) + gi * n
            f.hk[sl, start[gi] + step], f.hv[sl, start[gi] + step] = R.held(xk[gi, step]), R.held(xv[gi, step])
            close(st["out"], reference(f, xq[gi, step], sl, start[gi] + step + 1, (2 * n, 300)))
    f.cache.close()


def by_terms(f, q, slots, lens, prefix=None):
    """reference() with the bound that goes by each row's own weighted terms, for every element."""
    n_seq, n_q, H, hd = q.shape
    kv, P = f.hk.shape[2], prefix[1] if prefix else 0
    G = H // kv
    out, bound = np.zeros(q.shape), np.zeros(q.shape)
    for b in range(n_seq):
        n = max(0, min(int(lens[b]), f.hk.shape[1]))
        for h in range(kv):
            k, v = f.hk[slots[b], :n, h], f.hv[slots[b], :n, h]
            if P:
                k, v = np.concatenate([f.hk[prefix[0], :P, h], k]), np.concatenate([f.hv[prefix[0], :P, h], v])
            at = slice(h * G, (h + 1) * G)
            for i in range(n_q):
                vis = np.zeros((G, P + n), bool)
                vis[:, :P + max(0, n - n_q + 1 + i)] = True
                out[b, i, at], bound[b, i, at] = R.attention_by_terms(q[b, i, at], k, v, vis)
    return out, bound


def close_by_terms(got, want):
    ref, bound = want
    err = np.abs(got.cpu().numpy().astype(np.float64) - ref)
    assert (err <= bound).all(), (float((err / np.maximum(bound, 1e-300)).max()), np.argwhere(~(err <= bound))[:4])


class Held:
    """A cache holding the rows k, v [slots][ctx][kv][hd]."""

    def __init__(self, Q, k, v):
        slots, ctx, kv, hd = k.shape
        n = slots * ctx
        self.cache = Q.GpuKvCache(slots, kv, hd, ctx)
        self.cache.append(dev(k.reshape(n, kv, hd)), dev(v.reshape(n, kv, hd)), i32(np.repeat(np.arange(slots), ctx)),
                          i32(np.tile(np.arange(ctx), slots)))
        self.hk, self.hv = R.held(k), R.held(v)


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("group", [1, 6])
@pytest.mark.parametrize("up", [20, 30, 60, 90])
def test_large_values_that_only_later_tokens_see(Q, hd, group, up):
    """Drafted tokens whose V is far above the rest: the tokens before them do not see it, and keep all their bits."""
    rng = np.random.default_rng([hd, group, up])
    n_q, lens, P = 4, np.array([40, 64, 67, 300]), 90
    k, v = (rng.normal(0, 1, (5, 300, 2, hd)).astype(np.float32) for _ in range(2))
    for b, n in enumerate(lens):
        v[b, n - 3:n] *= np.exp2(np.float32(up) * np.array([1, 0.5, 1], np.float32))[:, None, None]
    f = Held(Q, k, v)
    q = rng.normal(0, 1, (4, n_q, 2 * group, hd)).astype(np.float32)
    slots = np.arange(4)
    close_by_terms(Q.attention_cached(dev(q), f.cache, i32(slots), i32(lens)), by_terms(f, q, slots, lens))
    close_by_terms(Q.attention_shared(dev(q), f.cache, 4, P, i32(slots), i32(lens)), by_terms(f, q, slots, lens, (4, P)))
    f.cache.close()


@pytest.mark.parametrize("hd", [32, 64, 128, 256])
@pytest.mark.parametrize("up", [25, 40, 80])
def test_large_values_that_the_softmax_ignores(Q, hd, up):
    """Positions with a weight of e^-100 and a V far above the rest (early, late, in other waves' tiles, in a prefix), and one
    with nearly all the weight and a V of zeros: the others keep their bits."""
    rng = np.random.default_rng([hd, up])
    n, lens, P = 500, np.array([500, 333, 64, 20]), 200
    slots = np.arange(4)
    q = rng.choice([-1.0, 1.0], (4, 1, 2, hd)).astype(np.float32)
    k, v = (rng.normal(0, 1, (5, n, 1, hd)).astype(np.float32) for _ in range(2))
    # scores against every query: 0 +- a few; with `away` added to them by the first element
    q[..., 0] = 8.0
    k[..., 0] = 0.0
    away = math.sqrt(hd) / 8.0
    for s in range(5):
        hidden = rng.choice(n, 40, replace=False)
        if s < 4:
            hidden = hidden[hidden < lens[s] - 4]
        hidden = np.union1d(hidden, [0, 5])
        k[s, hidden], v[s, hidden] = 0.0, v[s, hidden] * np.float32(2.0 ** up)
        k[s, hidden, :, 0] = -100 * away
    k[3, 7], v[3, 7], v[0, 130] = 0.0, 0.0, 0.0
    k[3, 7, :, 0] = 25 * away
    f = Held(Q, k, v)
    close_by_terms(Q.attention_cached(dev(q), f.cache, i32(slots), i32(lens)), by_terms(f, q, slots, lens))
    for seqs in (4, 1):      # (both ways through a prefix)
        t = slice(0, seqs)
        qs = np.tile(q[t], (1, 1, 10, 1)) if seqs == 4 else q[t]
        close_by_terms(Q.attention_shared(dev(qs), f.cache, 4, P, i32(slots[t]), i32(lens[t])), by_terms(f, qs, slots[t], lens[t], (4, P)))
    f.cache.close()


@pytest.mark.parametrize("hd", [8, 64, 128, 256])
def test_operands_keep_both_parts(Q, hd):
    """Two positions, and values that one fp16 part would round all in one direction: for q by more than the bound, and
    for V's scales likewise."""
    up = np.float32(1 + 0.97 * 2.0 ** -11)
    q = np.full((1, 1, 1, hd), up, np.float32)
    k = np.zeros((1, 2, 1, hd), np.float32)
    k[0, 0] = 2.0 / math.sqrt(hd)            # a score of 2 beside one of 0
    v = np.zeros((1, 2, 1, hd), np.float32)
    v[0, 0], v[0, 1] = 127 * up, -127 * up
    f = Held(Q, k, v)
    want = by_terms(f, q, [0], [2])
    for wrong in (R.attention_by_terms(np.float16(q[0, 0]).astype(np.float64), f.hk[0, :, 0], f.hv[0, :, 0], np.ones((1, 2), bool))[0],
                  want[0][0, 0] / up):
        assert (np.abs(wrong - want[0][0, 0]) > want[1][0, 0]).all()
    close_by_terms(Q.attention_cached(dev(q), f.cache, i32([0]), i32([2])), want)
    close_by_terms(Q.attention_shared(dev(q), f.cache, 0, 2, i32([0]), i32([0])), by_terms(f, q, [0], [0], (0, 2)))
    f.cache.close()


@pytest.mark.parametrize("hd", [16, 64, 256])
@pytest.mark.parametrize("k_up,q_up", [(0, 12), (0, 24), (10, 16), (10, 19), (30, 30), (80, 30), (-60, 100), (89, -89), (89, 24)])
def test_scores_of_every_size(Q, hd, k_up, q_up):
    """K rows of whole multiples of 2^k_up and queries of 2^q_up: scores, up to 2^126, are exact in fp32, and so is which of them
    are the largest.  With a step of 2^10 or more between scores these alone have weight, and the output is the mean of their V."""
    rng = np.random.default_rng([hd, k_up + 100])
    n, P, kv, n_q = 700, 300, 2, 3
    codes = rng.integers(-100, 1, (3, n, kv))
    codes[0] = np.sort(codes[0], 0)                     # the maximum moves with every few positions
    codes[1] = np.sort(codes[1], 0)[::-1]
    codes[2] -= 20                                      # all scores far below 0
    k = np.zeros((3, n, kv, hd), np.float64)
    k[..., 0] = 127                                     # the scale is 2^k_up; no query asks for this element
    k[..., 1:9] = codes[..., None]
    f = Held(Q, (k * 2.0 ** k_up).astype(np.float32), rng.normal(0, 1, (3, n, kv, hd)).astype(np.float32))
    assert np.array_equal(f.hk, k * 2.0 ** k_up)
    q = np.zeros((3, n_q, 2 * kv, hd), np.float32)
    q[..., 1:9] = 2.0 ** q_up
    # a step between scores: 8 q k / sqrt(hd); one of 2^10 in fp32 makes a weight of exp2(-2^10) = 0
    step = 8 * 2.0 ** (k_up + q_up) / math.sqrt(hd)
    assert step >= 2.0 ** 10 or (k_up, q_up) == (89, -89)
    slots, lens = np.array([2, 0, 1]), np.array([700, 611, 66])
    for prefix in (None, (2, P)):
        for b, (slot, length) in enumerate(zip(slots, lens)):
            if prefix is None:
                got = Q.attention_cached(dev(q[b:b + 1]), f.cache, i32([slot]), i32([length]))
            else:
                got = Q.attention_shared(dev(q[b:b + 1]), f.cache, *prefix, i32([slot]), i32([length]))
            ref, bound = by_terms(f, q[b:b + 1], [slot], [length], prefix)
            if step >= 2.0 ** 10:
                # equal scores have equal weights, whatever their size: what is left of the bound is sums and V's parts
                bound = bound * 0
                for i in range(n_q):
                    for h in range(2 * kv):
                        c, v = codes[slot, :length - n_q + 1 + i, h // 2], f.hv[slot, :length - n_q + 1 + i, h // 2]
                        if prefix:
                            c, v = np.concatenate([codes[2, :P, h // 2], c]), np.concatenate([f.hv[2, :P, h // 2], v])
                        v = v[c == c.max()].astype(np.float64)
                        assert np.allclose(ref[0, i, h], v.mean(0), rtol=1e-12, atol=1e-12)
                        bound[0, i, h] = np.abs(v).mean(0) * (2.0 ** -21 + (3 * len(v) + 16) * 2.0 ** -24) + len(v) * 2.0 ** -38 * np.abs(v).max()
            close_by_terms(got, (ref, bound))
    # all three at once, through the other way of the prefix
    qq = np.tile(q, (1, 2, 2, 1))
    a = Q.attention_shared(dev(qq), f.cache, 2, P, i32(slots), i32(lens)).cpu().numpy()
    if step >= 2.0 ** 10:
        assert np.isfinite(a).all() and (np.abs(a) <= np.abs(f.hv).max() * 1.001).all()
        i, h = 5, 0
        c, v = np.concatenate([codes[2, :P, 0], codes[2, :700, 0]]), np.concatenate([f.hv[2, :P, 0], f.hv[2, :700, 0]])
        v = v[c == c.max()].astype(np.float64)
        tol = np.abs(v).mean(0) * (2.0 ** -21 + (3 * len(v) + 16) * 2.0 ** -24) + len(v) * 2.0 ** -38 * np.abs(v).max()
        assert (np.abs(a[0, i, h] - v.mean(0)) <= tol).all()
    f.cache.close()


def test_small_differences_of_large_scores(Q):
    """Scores of some 2^24 that differ by whole numbers: exact in fp32, so the weights are those of the differences, in one tile, over the
    tiles of several waves and over parts."""
    rng = np.random.default_rng(5)
    hd, n = 64, 1500
    less = rng.integers(0, 12, n)
    less[rng.integers(0, n, 9)] = 0
    k = np.zeros((1, n, 1, hd), np.float32)
    k[..., 0], k[..., 1] = 127, 127 - less[None, :, None]
    # (2^13 127 127 + 8 (127 - less)) / 8: whole numbers below 2^24
    q = np.zeros((1, 1, 1, hd), np.float32)
    q[..., 0], q[..., 1] = 2.0 ** 13 * 127, 8.0
    f = Held(Q, k, rng.normal(0, 1, (1, n, 1, hd)).astype(np.float32))
    p = np.exp(-less * 1.0)[:, None]
    for length in (50, 300, 1500):
        w, v = p[:length], f.hv[0, :length, 0].astype(np.float64)
        ref, A = (w * v).sum(0) / w.sum(), (w * np.abs(v)).sum(0) / w.sum()
        # exponents, differences of up to 11, within 3 roundings; the exponential 2^-22; the weights' parts; the sums
        tol = A * (2 * (11 * 3 * 2.0 ** -24 + 2.0 ** -22) + 2.0 ** -22 + (3 * length + 16) * 2.0 ** -24)
        for got in (Q.attention_cached(dev(q), f.cache, i32([0]), i32([length])),
                    Q.attention_shared(dev(q), f.cache, 0, length, i32([0]), i32([0])),
                    Q.attention_shared(dev(np.tile(q, (1, 1, 20, 1))), f.cache, 0, length, i32([0]), i32([0]))):
            g = got.cpu().numpy()[0, 0].astype(np.float64)
            assert (np.abs(g - ref) <= tol).all(), (length, float((np.abs(g - ref) / tol).max()))
    f.cache.close()


class Long(Held):
    """Positions whose scores and values go up and down from tile to tile, so that a part lost, doubled or joined by the wrong
    maximum moves the output by far more than sums of this length may be off."""

    def __init__(self, Q, slots, n, kv, hd, seed):
        rng = np.random.default_rng(seed)
        tiles = -(-n // 64)
        k, v = (rng.normal(0, 0.5, (slots, n, kv, hd)).astype(np.float32) for _ in range(2))
        up = lambda x: np.repeat(x, 64, 1)[:, :n].astype(np.float32)  # noqa: E731
        k[..., 0] += up(rng.normal(0, 2, (slots, tiles, kv)))
        v += up(rng.uniform(0, 6, (slots, tiles, kv, 1)))
        super().__init__(Q, k, v)


@pytest.mark.parametrize("hd", [40, 64, 128, 256])
def test_more_than_sixteen_parts(Q, hd):
    """One long sequence alone: its positions and a prefix in dozens of parts, of which some are empty."""
    import torch
    n, kv, H = 8131, 2, 4
    f = Long(Q, 3, n, kv, hd, hd)
    rng = np.random.default_rng(hd + 1)
    q = rng.normal(0, 0.4, (2, 2, H, hd)).astype(np.float32)
    q[..., 0] = math.sqrt(hd) / 2
    work = ctypes.c_int64()

    def parts(n_seq, n_q, P, longest):
        from smallmind_amd._lib import call
        call("smx_attention_work_bytes", f.cache._h, n_seq, n_q, H, P, longest, ctypes.byref(work))
        return work.value // (n_seq * n_q * H * (hd + 2) * 4)

    assert parts(1, 2, 0, n) > 16 and parts(2, 2, 8000, 100) > 16
    for slot, length in ((0, n), (2, 4500), (1, 65)):      # (the shorter ones: parts without positions behind them)
        got = [Q.attention_cached(dev(q[:1]), f.cache, i32([slot]), i32([length])) for _ in range(3)]
        assert torch.equal(got[0], got[1]) and torch.equal(got[0], got[2])
        close_by_terms(got[0], by_terms(f, q[:1], [slot], [length]))
    for slots, lens, P in (([0], [n], 8000), ([1], [0], n), ([0, -1], [77, 100], 8000), ([0, 1], [0, 100], 7937)):
        b = len(slots)
        got = [Q.attention_shared(dev(q[:b]), f.cache, 2, P, i32(slots), i32(lens), max(lens)) for _ in range(3)]
        assert torch.equal(got[0], got[1]) and torch.equal(got[0], got[2])
        for i in range(b):
            if slots[i] < 0:
                assert not got[0][i].any()
            else:
                close_by_terms(got[0][i:i + 1], by_terms(f, q[i:i + 1], slots[i:i + 1], lens[i:i + 1], (2, P)))
    # 2 x 8 x 4 rows of a KV head, more than 16: the other way through the prefix, in as many parts
    qq = np.tile(q, (1, 4, 2, 1))
    got = Q.attention_shared(dev(qq), f.cache, 2, 8000, i32([0, 1]), i32([0, 100]), 100)
    close_by_terms(got, by_terms(f, qq, [0, 1], [0, 100], (2, 8000)))
    f.cache.close()
    torch.cuda.empty_cache()


@pytest.mark.parametrize("hd,group,n_q", [(64, 5, 8), (128, 4, 33), (80, 2, 1)])
def test_lengths_far_below_max_len(Q, hd, group, n_q):
    """What a captured step has: max_len is the context's limit, the lengths are anything."""
    f = Long(Q, 4, 5003, 2, hd, hd)
    rng = np.random.default_rng(hd)
    q = rng.normal(0, 0.5, (4, n_q, 2 * group, hd)).astype(np.float32)
    slots, lens = np.array([3, 0, 1, 2]), np.array([900, 40, 5003, 0])
    close_by_terms(Q.attention_cached(dev(q), f.cache, i32(slots), i32(lens)), by_terms(f, q, slots, lens))
    close_by_terms(Q.attention_shared(dev(q), f.cache, 2, 700, i32(slots), i32(lens)), by_terms(f, q, slots, lens, (2, 700)))
    f.cache.close()


# ---- verification of drafted tokens ---------------------------------------------------------------
def drafts(rng, n_seq, n_draft, vocab, zeros=False):
    lg = rng.normal(0, 2.5, (n_seq, n_draft + 1, vocab))
    ld = lg[:, :n_draft] + rng.normal(0, 0.7, (n_seq, n_draft, vocab))
    soft = lambda x: np.exp(x - x.max(-1, keepdims=True)) / np.exp(x - x.max(-1, keepdims=True)).sum(-1, keepdims=True)  # noqa: E731
    p, q = soft(lg), soft(ld)
    if zeros:       # as top-k leaves them
        p, q = np.where(p > p.mean(-1, keepdims=True), p, 0.0), np.where(q > q.mean(-1, keepdims=True), q, 0.0)
    p, q = p.astype(np.float32), q.astype(np.float32)
    x = np.array([[rng.choice(vocab, p=q[b, i].astype(np.float64) / q[b, i].astype(np.float64).sum()) for i in range(n_draft)]
                  for b in range(n_seq)], np.int32).reshape(n_seq, n_draft)
    return p, q, x, rng.random((n_seq, n_draft), dtype=np.float32), rng.random(n_seq, dtype=np.float32)


def check_verify(Q, p, q, x, ua, ud, lens=None):
    vocab = p.shape[2]
    out, acc = Q.verify_draft(dev(p), None if q is None else dev(q), dev(x), dev(ua), dev(ud), None if lens is None else i32(lens))
    eo, ea = R.verify(p, q, x, ua, ud, lens, vocab)
    assert np.array_equal(acc.cpu().numpy(), ea), (acc.cpu().numpy(), ea)
    assert np.array_equal(out.cpu().numpy(), eo), (out.cpu().numpy(), eo)
    return out, acc


@pytest.mark.parametrize("vocab", [1, 2, 63, 64, 65, 1000, 1024, 1025, 16384, 16385, 50257, 70001])
@pytest.mark.parametrize("n_seq,n_draft", [(1, 1), (3, 4), (7, 2)])
def test_verify_draft(Q, vocab, n_seq, n_draft):
    rng = np.random.default_rng(vocab + n_seq)
    for zeros in (False, True) if vocab > 2 else (False,):
        p, q, x, ua, ud = drafts(rng, n_seq, n_draft, vocab, zeros)
        check_verify(Q, p, q, x, ua, ud)
        check_verify(Q, p, None, x, ua, ud)
        lens = rng.integers(-1, n_draft + 2, n_seq)
        check_verify(Q, p, q, x, ua, ud, lens)
    ua[:] = 0.0
    ud[:] = 0.0
    check_verify(Q, p, q, x, ua, ud)
    ud[:] = np.float32(1 - 2.0 ** -24)
    check_verify(Q, p, q, x, ua, ud)


def test_verify_captured_and_replayed(Q):
    import torch
    rng = np.random.default_rng(77)
    sets = [drafts(rng, 5, 4, 1003) for _ in range(4)]
    now = [dev(a) for a in sets[0]]
    run = lambda t: Q.verify_draft(*t)  # noqa: E731
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        run(now)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        out = run(now)
    for data in sets + sets[:1]:
        for t, a in zip(now, data):
            t.copy_(dev(a))
        g.replay()
        want = run([dev(a) for a in data])
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_verify_many_drafts_and_none(Q):
    rng = np.random.default_rng(2)
    p, q, x, ua, ud = drafts(rng, 4, 70, 33)
    check_verify(Q, p, np.minimum(q, p[:, :70]), x, np.minimum(ua, 0.5), ud)     # long accepted runs
    check_verify(Q, p, q, x, ua, ud, np.array([70, 65, 64, 0]))
    e = np.zeros((4, 0, 33), np.float32)
    check_verify(Q, p[:, :1], e, x[:, :0], ua[:, :0], ud)
    check_verify(Q, p[:, :1], None, x[:, :0], ua[:, :0], ud)


def test_verify_of_odd_probabilities(Q):
    rng = np.random.default_rng(5)
    p, q, x, ua, ud = drafts(rng, 12, 2, 300)
    ua[:] = 0.999
    q[0], p[0, :2] = q[0], q[0]                 # equal: ratio 1 accepts
    p[1, 0, x[1, 0]] = 0.0                      # refused; drawn from the difference
    p[2, 0] = q[2, 0] * np.float32(0.5)         # refused with nothing left of the difference: drawn from p
    p[3, 0] = 0.0                               # no weight at all
    p[4, 0, ::3] = np.nan
    q[5, 0, ::2] = np.nan
    x[6, 0], x[7, 0], x[8, 0] = -5, 300, 2**31 - 1
    p[9, 0], p[9, 0, 299] = 0.0, 1.0            # everything on the last token
    p[10, 0], p[10, 0, 0] = 0.0, 1.0
    p[11, 0] = np.float32(1.0 / 300)
    out, acc = check_verify(Q, p, q, x, ua, ud)
    assert acc[3] == 0 and out[3].tolist() == [-1, -1, -1]
    check_verify(Q, p, None, x, ua, ud)


def test_verify_where_a_row_holds_nan(Q):
    """By what is documented, value by value: a NaN in the target's row is a 0; one in the draft's refuses its token,
    which then weighs nothing beside max(p - q, 0) of the others, and may come again only from p alone."""
    nan = np.nan
    p = np.array([[[0.5, 0.25, 0.25, 0.0], [1, 0, 0, 0]]] * 6, np.float32)
    q = np.array([[[0.25, 0.5, 0.25, 0.0]]] * 6, np.float32)
    x, ua, ud = np.zeros((6, 1), np.int32), np.zeros((6, 1), np.float32), np.zeros(6, np.float32)
    q[1, 0, 0] = nan                                  # the token's own: refused, though p = 0.5 > 0; nothing left: from p
    q[2, 0], p[2, 0] = [nan, 0.1, 0.25, 0.0], [0.5, 0.25, 0.25, 0.0]     # only token 1 has a difference
    p[3, 0, 0] = nan                                  # counts as 0: refused, drawn from the rest
    p[3, 0, 2] = 0.5
    x[4, 0], q[4, 0], p[4, 0] = 1, [0.25, 0.5, nan, 0.0], [0.5, 0.0, 0.5, 0.0]     # refused; 2 does not count
    ud[4] = 0.999
    x[5, 0], q[5, 0] = 1, [nan, 0.125, 0.25, 0.0]     # accepted: its own probabilities are numbers
    out, acc = Q.verify_draft(dev(p), dev(q), dev(x), dev(ua), dev(ud))
    assert acc.tolist() == [1, 0, 0, 0, 0, 1]
    assert out.tolist() == [[0, 0], [0, -1], [1, -1], [2, -1], [0, -1], [1, 0]]


def test_verify_rows_of_wider_matrices_and_unaligned(Q):
    rng = np.random.default_rng(6)
    p, q, x, ua, ud = drafts(rng, 3, 3, 777)
    wp, wq = np.zeros((3, 4, 800), np.float32), np.zeros((3, 3, 901), np.float32)
    wp[:, :, 1:778], wq[:, :, 3:780] = p, q
    out, acc = Q.verify_draft(dev(wp)[:, :, 1:778], dev(wq)[:, :, 3:780], dev(x), dev(ua), dev(ud))
    eo, ea = R.verify(p, q, x, ua, ud, None, 777)
    assert np.array_equal(out.cpu().numpy(), eo) and np.array_equal(acc.cpu().numpy(), ea)
    with pytest.raises(ValueError):
        Q.verify_draft(dev(p), dev(q)[:, :2], dev(x), dev(ua), dev(ud))
    with pytest.raises(ValueError):
        Q.verify_draft(dev(p).transpose(1, 2), None, dev(x), dev(ua), dev(ud))
    with pytest.raises(ValueError):
        Q.verify_draft(dev(p), dev(q), dev(x), dev(ua).double(), dev(ud))


# ---- a run of them together -----------------------------------------------------------------------
def test_speculative_serving_over_a_shared_prompt(Q):
    """Three chats behind one prompt: in every round each drafts tokens, writes their rows, the target attends over
    prompt and chat for all of them at once, its probabilities verify the drafts, and the lengths move on by what
    was accepted.  Every round is replayed in 64 bits from what the cache holds."""
    import torch
    rng = np.random.default_rng(77)
    n, H, kv, hd, V, D, P = 3, 8, 2, 64, 200, 3, 190
    d = H * hd
    emb = rng.normal(0, 1, (V, (H + 2 * kv) * hd)).astype(np.float32)         # the fused projection of each token
    head = rng.normal(0, 0.6, (d, V)).astype(np.float32)
    cache = Q.GpuKvCache(n + 1, kv, hd, 256)
    prompt = rng.integers(0, V, P)
    tk = lambda t: np.asarray(t)  # noqa: E731
    E = dev(emb)

    def rows(tokens):
        f = E[dev(tk(tokens).reshape(-1), np.int64)]
        return f[:, :d].unflatten(1, (H, hd)), f[:, d:d + kv * hd].unflatten(1, (kv, hd)), f[:, d + kv * hd:].unflatten(1, (kv, hd))

    _, k, v = rows(prompt)
    cache.append(k, v, i32(np.full(P, n)), i32(np.arange(P)))
    f = type("F", (), {})()
    f.k = np.zeros((n + 1, 256, kv, hd), np.float32)
    f.hk, f.hv = f.k.copy(), f.k.copy()
    put = lambda s, p, t: (f.hk.__setitem__((s, p), R.held(emb[t, d:d + kv * hd].reshape(kv, hd))),  # noqa: E731
                           f.hv.__setitem__((s, p), R.held(emb[t, d + kv * hd:].reshape(kv, hd))))
    for p, t in enumerate(prompt):
        put(n, p, t)
    last, lens = rng.integers(0, V, n), np.zeros(n, int)
    slots = np.arange(n)
    accepted_all = 0
    for _ in range(6):
        draft_p = rng.dirichlet(np.full(V, 0.3), (n, D)).astype(np.float32)
        x = np.array([[rng.choice(V, p=draft_p[b, i].astype(np.float64) / draft_p[b, i].astype(np.float64).sum())
                       for i in range(D)] for b in range(n)], np.int32)
        ua, ud = rng.random((n, D), dtype=np.float32), rng.random(n, dtype=np.float32)
        toks = np.concatenate([last[:, None], x], 1)
        q, k, v = rows(toks)
        pos = lens[:, None] + np.arange(D + 1)
        cache.append(k, v, i32(np.repeat(slots, D + 1)), i32(pos.reshape(-1)))
        new = i32(lens + D + 1)
        out = Q.attention_shared(q.reshape(n, D + 1, H, hd), cache, n, P, i32(slots), new, 256)
        for b in range(n):
            for i in range(D + 1):
                put(b, lens[b] + i, toks[b, i])
        close(out, reference(f, q.reshape(n, D + 1, H, hd).cpu().numpy(), slots, lens + D + 1, (n, P)))
        logits = out.reshape(n, D + 1, d) @ dev(head)
        probs = torch.empty_like(logits)
        for b in range(n):
            for i in range(D + 1):
                probs[b, i] = Q.sample(logits[b, i].contiguous(), 0.5, temperature=0.9, top_k=60)[1]
        # drafts from the target's own neighbourhood, so that some are taken
        mix = (0.5 * probs[:, :D] + 0.5 * dev(draft_p)).contiguous()
        got, acc = Q.verify_draft(probs, mix, dev(x), dev(ua), dev(ud))
        eo, ea = R.verify(probs.cpu().numpy(), mix.cpu().numpy(), x, ua, ud, None, V)
        assert np.array_equal(got.cpu().numpy(), eo) and np.array_equal(acc.cpu().numpy(), ea)
        accepted_all += int(ea.sum())
        lens = lens + 1 + ea                     # the refused drafts' places are written over by the next round
        last = eo[np.arange(n), ea]
        assert (last >= 0).all()
    cache.close()
