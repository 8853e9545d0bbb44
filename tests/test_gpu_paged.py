"""The paged KV cache on the GPU against plain 64-bit forms: writes with norms and rotation, attention of ragged batches,
received weights, eviction."""
import ctypes
import math

import numpy as np
import pytest
import torch

from tests import paged_reference as R

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
TYPES = {"f32": F32, "f16": F16, "bf16": BF16}


@pytest.fixture(scope="module")
def Q(gpu):
    from smallmind_amd import quantization
    return quantization


def dev(a, dtype=None):
    t = torch.from_numpy(np.ascontiguousarray(a))
    return (t if dtype is None else t.to(dtype)).cuda()


def i32(a):
    return dev(np.asarray(a, np.int32))


def f64(t):
    return t.detach().double().cpu().numpy()


def close(got, want, bound):
    got = f64(got)
    bad = np.isnan(want) != np.isnan(got)
    ok = np.where(np.isnan(want), True, np.abs(got - want) <= bound) & ~bad
    assert ok.all(), (int((~ok).sum()), ok.size, np.argwhere(~ok)[:5].tolist(), got[~ok][:5], want[~ok][:5],
                      np.broadcast_to(bound, want.shape)[~ok][:5])


# ---- rows written and read back -------------------------------------------------------------------
@pytest.mark.parametrize("hd", [8, 16, 32, 40, 64, 80, 96, 104, 128, 136, 192, 200, 256])
@pytest.mark.parametrize("cache,tin,page", [(F16, F32, 16), (BF16, BF16, 64), (F16, F16, 1024), (BF16, F32, 32), (F16, BF16, 128)])
def test_rows_come_back_rounded(Q, hd, cache, tin, page):
    rng = np.random.default_rng(hd)
    kv, pages, n = 3, 3, 37
    k, v = (dev(rng.normal(0, 1, (n, kv, hd)) * np.exp2(rng.integers(-12, 12, (n, kv, 1))), tin) for _ in range(2))
    at = rng.permutation(pages * page)[:n]
    c = Q.GpuPagedCache(cache, pages, kv, hd, page)
    assert c.append(k, v, i32(at)) is None
    gk, gv = c.read(i32(np.arange(pages * page)))
    assert gk.dtype is cache and gk.shape == (pages * page, kv, hd)
    for g, x in ((gk, k), (gv, v)):
        e = np.zeros(g.shape)
        e[at] = R.rounded(f64(x), cache)
        assert np.array_equal(f64(g), e)
    c.close()
    with pytest.raises(ValueError, match="closed"):
        c.read(i32([0]))


def test_places_that_the_cache_does_not_have(Q):
    rng = np.random.default_rng(3)
    c = Q.GpuPagedCache(F16, 2, 2, 64, 16)
    p = np.array([5, -1, 32, 31, 2**31 - 1, -2**31, 6])
    k, v = (rng.normal(0, 1, (7, 2, 64)).astype(np.float32) for _ in range(2))
    q = c.append(dev(k), dev(v), i32(p), q=dev(k))
    assert np.array_equal(q.cpu().numpy(), k)              # the queries come back whatever the place
    ok = (p >= 0) & (p < 32)
    for g, x in zip(c.read(i32(p)), (k, v)):
        assert np.array_equal(f64(g), np.where(ok[:, None, None], R.rounded(x, F16), 0))
    gk, _ = c.read(i32(np.arange(32)))
    assert int((gk.abs().sum((1, 2)) > 0).sum()) == 3
    c.append(dev(k[:0]), dev(v[:0]), i32(p[:0]))
    assert c.read(i32([]))[0].shape == (0, 2, 64)


@pytest.mark.parametrize("cache", [F16, BF16])
def test_positions_that_are_not_finite(Q, cache):
    rng = np.random.default_rng(8)
    k, v = (rng.normal(0, 1, (8, 2, 64)).astype(np.float32) for _ in range(2))
    k[1, 0, 63], k[2, 1, 0], v[4, 0, 5], v[5, 1, 9], v[6, 0, 0] = np.nan, np.inf, -np.inf, np.nan, 1e6    # (fp16: infinite)
    c = Q.GpuPagedCache(cache, 1, 2, 64, 16)
    c.append(dev(k), dev(v), i32(np.arange(8)))
    ek, ev = R.held(k, v, cache)
    gk, gv = c.read(i32(np.arange(8)))
    assert np.array_equal(f64(gk), ek, equal_nan=True) and np.array_equal(f64(gv), ev, equal_nan=True)
    assert np.isnan(ev[4, 0]).all() and not np.isnan(ev[4, 1]).any()
    c.append(dev(np.zeros_like(k)), dev(np.ones_like(v)), i32(np.arange(8)))      # written over
    gk, gv = c.read(i32(np.arange(8)))
    assert not gk.any() and bool((gv == 1).all())


def tables(rng, n_pos, half, off=0):
    a = np.arange(n_pos)[:, None] * 10000.0 ** (-np.arange(half) / half)
    buf = [np.concatenate([np.zeros(off), f(a).ravel()]).astype(np.float32) for f in (np.cos, np.sin)]
    return [dev(b)[off:].view(n_pos, half) for b in buf]


@pytest.mark.parametrize("hd,n_rot,sections,halves,norm,tin,tout", [
    (64, 64, None, False, True, F32, F32), (64, 64, None, True, True, F32, F16), (128, 128, [16, 24, 24], True, True, BF16, BF16),
    (128, 64, [8, 12, 12], False, True, F16, F32), (80, 80, [10, 15, 15], True, False, F32, F32), (40, 20, None, True, True, F32, BF16),
    (96, 96, [17, 30, 1], False, True, F32, F32), (256, 256, [64, 0, 63, 1], True, True, F16, F16), (8, 2, None, True, True, F32, F32),
    (8, 8, [1, 1, 1, 1], False, False, BF16, F32), (200, 72, [5, 31], True, True, F32, F32), (104, 104, None, True, True, F32, F32),
    (32, 6, [1, 2], False, True, F32, F32), (16, None, None, False, True, F32, F32)])
@pytest.mark.parametrize("off", [0, 1])
def test_norms_and_rotation(Q, hd, n_rot, sections, halves, norm, tin, tout, off):
    """Dense rows and rows written to a cache, from the rows of a fused projection, aligned or not."""
    rng = np.random.default_rng(hd + off)
    n, H, kv, n_pos = 67, 5, 2, 50
    width = (H + 2 * kv) * hd + off * 3
    f = dev(rng.normal(0, 2, n * width + off), tin)[off:].view(n, width)
    q, k, v = f[:, :H * hd].unflatten(1, (H, hd)), f[:, H * hd:(H + kv) * hd].unflatten(1, (kv, hd)), f[:, (H + kv) * hd:(H + 2 * kv) * hd].unflatten(1, (kv, hd))
    gq, gk = (rng.normal(1, 0.3, hd).astype(np.float32) if norm else None for _ in range(2))
    rot = pos = cos = sin = None
    if n_rot:
        cos, sin = tables(rng, n_pos, n_rot // 2, off)
        rot = Q.Rotation(cos, sin, sections, halves)
        pos = rng.integers(0, n_pos, (rot.n_axes, n)).astype(np.int32)
    args = dict(q_gamma=None if gq is None else dev(gq), k_gamma=None if gk is None else dev(gk), eps=1e-5, rotation=rot,
                pos=None if pos is None else dev(pos), dtype=tout)
    qo, ko = Q.qk_norm_rope(q, k, **args)
    np_tab = (None, None) if cos is None else (cos.cpu().numpy(), sin.cpu().numpy())
    sec = sections or [n_rot // 2 if n_rot else 0]
    for got, x, g in ((qo, q, gq), (ko, k, gk)):
        want, e = R.turned(f64(x), g, 1e-5, *np_tab, pos, sec, halves)
        assert got.dtype is tout
        close(got, want, e + R.HALF_STEP[tout] * (np.abs(want) + e) + R.LEAST[tout])
    c = Q.GpuPagedCache(BF16, 9, kv, hd, 16)
    places = rng.permutation(9 * 16)[:n]
    q2 = c.append(k, v, i32(places), q=q, **args)
    assert torch.equal(q2, qo)
    rk, rv = c.read(i32(places))
    want, e = R.turned(f64(k), gk, 1e-5, *np_tab, pos, sec, halves)
    close(rk, want, e + R.HALF_STEP[BF16] * (np.abs(want) + e))
    assert np.array_equal(f64(rv), R.rounded(f64(v), BF16))
    c.close()


def test_positions_without_an_angle(Q):
    rng = np.random.default_rng(5)
    cos, sin = tables(rng, 4, 8)
    x = dev(rng.normal(0, 1, (5, 2, 32)), F32)
    pos = i32([0, -1, 4, 3, 2**31 - 1])
    for halves in (False, True):
        q, k = Q.qk_norm_rope(x, x, rotation=Q.Rotation(cos, sin, halves=halves), pos=pos)
        nan = torch.isnan(q).cpu().numpy()
        assert nan[[1, 2, 4], :, :16].all() and not nan[..., 16:].any() and not nan[[0, 3]].any()
    c = Q.GpuPagedCache(F16, 1, 2, 32, 16)
    c.append(x, x, i32(np.arange(5)), rotation=Q.Rotation(cos, sin), pos=pos)
    gk, gv = c.read(i32(np.arange(5)))
    assert np.array_equal(np.isnan(f64(gv)).all((1, 2)), [False, True, True, False, True]) and np.isnan(f64(gk[1])).all()


@pytest.mark.parametrize("exponent,tin", [(-66, F32), (-61, BF16), (65, F32), (66, BF16), (118, F32)])
@pytest.mark.parametrize("hd", [8, 104, 256])
def test_norms_of_rows_whose_squares_leave_fp32(Q, hd, exponent, tin):
    """Beside ordinary rows; eps 0, so that small rows are not lost in it."""
    rng = np.random.default_rng([hd, 100 + exponent])
    n = 9
    x = rng.normal(0, 1, (n, 3, hd)) * np.exp2(np.where(rng.uniform(size=(n, 3, 1)) < 0.6, exponent, 0))
    x = dev(x, tin)
    g = rng.normal(1, 0.3, hd).astype(np.float32)
    cos, sin = tables(rng, 16, hd // 2)
    pos = rng.integers(0, 16, (1, n)).astype(np.int32)
    q, k = Q.qk_norm_rope(x, x[:, :2], dev(g), dev(g), 0.0, Q.Rotation(cos, sin, halves=True), dev(pos), dtype=F32)
    want, e = R.turned(f64(x), g, 0.0, cos.cpu().numpy(), sin.cpu().numpy(), pos, [hd // 2], True)
    close(q, want, e)
    close(k, want[:, :2], e[:, :2])


# ---- batches ---------------------------------------------------------------------------------------
class Batch:
    """Sequences of these lengths with `new` new tokens each, their pages shuffled in a cache whose other pages hold NaN."""

    def __init__(self, Q, rng, cache, io, H, kv, hd, page, lens, new, pad=0, spread=1.0, extra_pages=3, q_off=0, slack=0):
        self.cache_type, self.io, self.H, self.kv, self.hd, self.page = cache, io, H, kv, hd, page
        self.lens, self.new = list(lens), list(new)
        per = [-(-n // page) for n in lens]
        pool = sum(per) + extra_pages
        order = rng.permutation(pool)
        self.tables = np.full((len(lens), max(max(per), 1)), -7)
        at = 0
        for b, n in enumerate(per):
            self.tables[b, :n] = order[at:at + n]
            at += n
        self.c = Q.GpuPagedCache(cache, pool, kv, hd, page)
        every = np.arange(pool * page)
        junk = np.full((len(every), kv, hd), np.nan, np.float32)
        self.c.append(dev(junk), dev(junk), i32(every))
        self.k, self.v = [], []
        for b, n in enumerate(lens):
            k = rng.normal(0, 1, (n, kv, hd)) * spread
            k[:, :, ::7] *= 2
            k, v = R.rounded(k, cache), R.rounded(rng.normal(0, 1, (n, kv, hd)), cache)
            self.k.append(k), self.v.append(v)
            if n:
                self.c.append(dev(k, cache), dev(v, cache), self.places(b, np.arange(n)))
        n_tok = sum(new) + pad
        width = (H + 2 * kv) * hd + slack
        f = dev(R.rounded(rng.normal(0, 1.5, n_tok * width + q_off), io), io)[q_off:].view(n_tok, width)
        self.q = f[:, :H * hd].unflatten(1, (H, hd))
        self.starts = np.concatenate([[0], np.cumsum(new)])
        self.max_q, self.max_len = max(max(new), 1), max(max(lens), 1)

    def places(self, b, pos):
        return i32(self.tables[b, pos // self.page] * self.page + pos % self.page)

    def args(self):
        return self.c, i32(self.starts), i32(self.lens), i32(self.tables), self.max_q, self.max_len

    def rows(self, b, scale=None, cap=0.0, slopes=None, window=0, prefix=None, every=1):
        """For every `every`th KV head of sequence b: (head, query heads, Scores of tokens x heads, seen)."""
        n, m, G = self.lens[b], self.new[b], self.H // self.kv
        qb = f64(self.q[self.starts[b]:self.starts[b + 1]])
        t = np.arange(n - m, n)
        see = R.visible(n - m, m, n, min(prefix[b], n) if prefix is not None else 0, window)
        for h in range(b % every, self.kv, every):
            for g in range(G):
                yield h, h * G + g, R.Scores(qb[:, h * G + g], self.k[b][:, h], t, self.io, self.cache_type, scale, cap,
                                             0.0 if slopes is None else slopes[h * G + g]), see

    def check(self, out, lse, skip=(), every=1, **rules):
        out, lse = out.cpu(), lse.cpu()
        for b in range(len(self.lens)):
            if b in skip or not self.new[b]:
                continue
            at = slice(self.starts[b], self.starts[b + 1])
            for h, head, S, see in self.rows(b, every=every, **rules):
                o, e, l, le = R.attention(S, self.v[b][:, h], see, self.io, self.cache_type)
                close(out[at, head], o, e)
                got = f64(lse[at, head])
                fin = np.isfinite(l)
                assert np.array_equal(got[~fin], l[~fin], equal_nan=True)
                assert (np.abs(got[fin] - l[fin]) <= le[fin]).all()


def kernel_rules(rules):
    r = dict(rules)
    if r.get("slopes") is not None:
        r["slopes"] = dev(np.asarray(r["slopes"], np.float32))
    if r.get("prefix") is not None:
        r["prefix"] = i32(r["prefix"])
    return r


def run(Q, B, rules=None, **k):
    return Q.attention_paged(B.q, *B.args(), lse=True, **kernel_rules(rules or {}), **k)


LENS = [1, 15, 16, 17, 31, 32, 33, 63, 64, 65, 100, 128, 129, 300]


@pytest.mark.parametrize("cache,io", [(F16, F32), (F16, F16), (BF16, BF16), (BF16, F32)])
@pytest.mark.parametrize("H,kv,hd,page", [(4, 2, 64, 16), (8, 1, 128, 64), (3, 3, 32, 16), (6, 2, 80, 32), (4, 4, 96, 16), (2, 1, 256, 64),
                                          (5, 1, 40, 16), (2, 2, 8, 16), (2, 1, 136, 128), (3, 1, 200, 16), (2, 1, 104, 1024)])
def test_single_tokens(Q, cache, io, H, kv, hd, page):
    rng = np.random.default_rng(hd)
    B = Batch(Q, rng, cache, io, H, kv, hd, page, LENS, [1] * len(LENS))
    B.check(*run(Q, B))
    B.c.close()


@pytest.mark.parametrize("cache,io", [(F16, F32), (F16, F16), (BF16, BF16), (BF16, F32)])
@pytest.mark.parametrize("H,kv,hd,page", [(4, 2, 64, 16), (8, 1, 128, 64), (3, 3, 32, 16), (6, 2, 80, 32), (4, 4, 96, 16), (2, 1, 256, 64),
                                          (5, 1, 40, 16), (2, 2, 8, 16), (2, 1, 136, 128)])
@pytest.mark.parametrize("shape", ["chunks", "mixed", "prompts"])
def test_chunks(Q, cache, io, H, kv, hd, page, shape):
    rng = np.random.default_rng(hd + len(shape))
    lens, new = {"chunks": ([200, 131, 97], [70, 33, 64]),
                 "mixed": ([150, 1, 90, 260, 64, 40, 17], [129, 1, 1, 4, 64, 0, 9]),
                 "prompts": ([300, 65, 1], [300, 65, 1])}[shape]
    B = Batch(Q, rng, cache, io, H, kv, hd, page, lens, new)
    B.check(*run(Q, B))
    B.c.close()


RULES = [dict(cap=20.0), dict(cap=2.0, scale=0.3), dict(slopes=True), dict(window=1), dict(window=37), dict(window=64, prefix=True),
         dict(prefix=True), dict(cap=30.0, slopes=True, window=50, prefix=True, scale=0.05), dict(window=10 ** 6), dict(slopes=True, prefix=True)]


@pytest.mark.parametrize("rules", RULES)
@pytest.mark.parametrize("cache,io,H,kv,hd", [(F16, F32, 4, 2, 64), (BF16, BF16, 8, 2, 128), (F16, F16, 3, 1, 40)])
@pytest.mark.parametrize("shape", ["decode", "mixed", "prompts"])
def test_rules(Q, rules, cache, io, H, kv, hd, shape):
    rng = np.random.default_rng(hd)
    lens, new = {"decode": ([1, 64, 65, 200, 333], [1, 1, 1, 1, 1]),
                 "mixed": ([150, 1, 290, 260, 64], [130, 1, 1, 7, 64]),
                 "prompts": ([300, 65, 33], [300, 65, 33])}[shape]
    B = Batch(Q, rng, cache, io, H, kv, hd, 16, lens, new)
    rules = dict(rules)
    if rules.get("slopes"):
        rules["slopes"] = np.exp2(-np.arange(H) * 1.3 - 1).astype(np.float32)
        rules["slopes"][-1] = 0.0
    if rules.get("prefix"):
        rules["prefix"] = [[0, 3, 70, 500, 64][b] for b in range(len(lens))]
    B.check(*run(Q, B, rules), **rules)
    mass(Q, B, rules)
    B.c.close()


def mass(Q, B, rules, before=None):
    """The received weights of a batch, with the plain form's own lse, over what there was."""
    n_seq = len(B.lens)
    lse = np.zeros((B.q.shape[0], B.H), np.float32)
    for b in range(n_seq):
        for h, head, S, see in B.rows(b, **rules):
            lse[B.starts[b]:B.starts[b + 1], head] = R.attention(S, B.v[b][:, h], see, B.io, B.cache_type)[2]
    got = Q.attention_mass(B.q, dev(lse), *B.args(), mass=before, **kernel_rules(rules))
    assert got.shape == (n_seq, B.kv, B.max_len)
    got = f64(got)
    for b in range(n_seq):
        want, bound = np.zeros((B.kv, B.max_len)), np.zeros((B.kv, B.max_len))
        for h, head, S, see in B.rows(b, **rules):
            w, e = R.received(S, lse[B.starts[b]:B.starts[b + 1], head].astype(np.float64), see)
            want[h, :B.lens[b]] += w
            bound[h, :B.lens[b]] += e + 2.0 ** -24 * np.nan_to_num(w) * 4
        if before is not None:
            w = f64(before[b])[:, :B.max_len]
            want[:, :w.shape[1]] += w
            bound[:, :w.shape[1]] += np.abs(w) * 2.0 ** -23
            want[:, B.lens[b]:] = 0
        bad = np.isnan(want) != np.isnan(got[b])
        assert not bad.any() and (np.nan_to_num(np.abs(got[b] - want)) <= np.nan_to_num(bound)).all(), (b, np.nanmax(np.abs(got[b] - want) - bound))


@pytest.mark.parametrize("cache,io,hd", [(F16, F16, 64), (BF16, BF16, 32), (BF16, BF16, 128), (F16, F32, 32), (F16, F16, 96), (BF16, BF16, 256)])
@pytest.mark.parametrize("heads", [150, 300])
def test_many_blocks(Q, cache, io, hd, heads):
    """More blocks of rows than compute units, and more than two for each."""
    rng = np.random.default_rng([hd, heads])
    B = Batch(Q, rng, cache, io, heads, heads, hd, 16, [200, 90, 33], [170, 40, 1])
    for rules in ({}, dict(window=37, prefix=[20, 0, 33], slopes=rng.uniform(0.01, 0.3, heads))):
        out, lse = run(Q, B, rules)
        B.check(out, lse, every=7, **rules)


def test_rows_that_see_nothing_and_rows_of_no_sequence(Q):
    rng = np.random.default_rng(11)
    for cache, io, H, kv in ((F16, F32, 4, 2), (BF16, BF16, 40, 1)):
        # lengths below the number of new tokens (their first tokens would lie before position 0), of zero, sequences without tokens
        B = Batch(Q, rng, cache, io, H, kv, 64, 16, [3, 0, 5, 40, 0], [7, 2, 0, 3, 1], pad=6)
        out = torch.full(B.q.shape, 7.5, dtype=io, device="cuda")
        got, lse = run(Q, B, out=out)
        assert got is out
        B.check(got, lse)
        assert not got[:4].any() and not got[7:9].any() and bool((lse[:4] == -math.inf).all())
        assert bool((got[sum(B.new):] == 7.5).all())
        mass(Q, B, {})
        # the same with a prefix that rows before position 0 see
        B.check(*run(Q, B, dict(prefix=[2, 1, 0, 0, 3])), prefix=[2, 1, 0, 0, 3])
        B.c.close()


def test_an_empty_batch(Q):
    rng = np.random.default_rng(12)
    B = Batch(Q, rng, F16, F32, 4, 2, 64, 16, [20, 30], [0, 0])
    out, lse = run(Q, B)
    assert out.shape == (0, 4, 64) and lse.shape == (0, 4)
    before = dev(rng.uniform(0, 1, (2, 2, 25)).astype(np.float32))
    mass(Q, B, {}, before)
    out, lse = Q.attention_paged(torch.zeros(2, 4, 64, device="cuda"), B.c, i32([0, 1, 2]), i32([0, 0]), i32(np.zeros((2, 0))), 1, 0, lse=True)
    assert not out.any() and bool((lse == -math.inf).all())
    assert Q.attention_mass(torch.zeros(2, 4, 64, device="cuda"), lse, B.c, i32([0, 1, 2]), i32([0, 0]), i32(np.zeros((2, 0))), 1, 0).shape == (2, 2, 0)


@pytest.mark.parametrize("cache,io,hd", [(F16, F32, 64), (BF16, BF16, 128)])
@pytest.mark.parametrize("lens,new", [([5000, 1], [1, 1]), ([4000], [40]), ([2000, 3100], [3, 90]), ([9000], [1])])
def test_long_contexts_in_parts(Q, cache, io, hd, lens, new):
    rng = np.random.default_rng(hd + len(lens))
    B = Batch(Q, rng, cache, io, 4, 1, hd, 32, lens, new)
    need = ctypes.c_int64()
    from smallmind_amd import _lib
    _lib.call("smx_attention_paged_work_bytes", B.c._h, 0 if io is F32 else 30, sum(new), 4, len(lens), B.max_q, B.max_len, None, ctypes.byref(need))
    assert need.value > 0
    B.check(*run(Q, B))
    B.check(*run(Q, B, dict(window=700)), window=700)
    B.check(*run(Q, B, dict(window=70, prefix=[100] * len(lens))), window=70, prefix=[100] * len(lens))
    mass(Q, B, {}, dev(rng.uniform(0, 5, (len(lens), 1, max(lens) - 20)).astype(np.float32)))
    B.c.close()


@pytest.mark.parametrize("off,slack", [(1, 0), (0, 3), (8, 5)])
@pytest.mark.parametrize("io", [F32, F16])
def test_queries_in_rows_of_any_alignment(Q, io, off, slack):
    rng = np.random.default_rng(off)
    for new in ([1, 1, 1], [40, 9, 1]):
        B = Batch(Q, rng, F16, io, 6, 2, 72, 16, [60, 30, 90], new, q_off=off, slack=slack)
        buf = torch.empty(B.q.numel() + 1, dtype=io, device="cuda")
        out = buf[off:off + B.q.numel()].view(B.q.shape) if off < 2 else buf[:B.q.numel()].view(B.q.shape)
        B.check(*run(Q, B, out=out))
        B.c.close()


def test_bad_pages_are_not_seen_and_shared_pages_are(Q):
    rng = np.random.default_rng(21)
    for cache, io, new in ((F16, F32, [1, 1, 1]), (BF16, BF16, [50, 3, 40])):
        B = Batch(Q, rng, cache, io, 4, 2, 64, 16, [100, 100, 100], new)
        # sequence 1 begins with sequence 0's first three pages; sequence 2 lacks two of its own
        B.tables[1, :3] = B.tables[0, :3]
        B.k[1][:48], B.v[1][:48] = B.k[0][:48], B.v[0][:48]
        B.tables[2, 1], B.tables[2, 6] = B.c.n_pages, -1
        out, lse = run(Q, B)
        B.check(out, lse, skip=(2,))
        see = R.visible(100 - new[2], new[2], 100)
        see[:, 16:32] = see[:, 96:] = False
        for h, head, S, _ in B.rows(2):
            o, e, l, _ = R.attention(S, B.v[2][:, h], see, io, cache)
            close(out[B.starts[2]:B.starts[3], head], o, e)
        B.c.close()


def test_what_is_not_finite_reaches_only_who_sees_it(Q):
    rng = np.random.default_rng(22)
    for cache, io in ((F16, F32), (BF16, BF16), (F16, F16)):
        B = Batch(Q, rng, cache, io, 4, 2, 64, 16, [100, 60], [80, 1])
        for b, p, h, what in ((0, 70, 0, np.nan), (0, 90, 1, np.inf), (1, 59, 1, -np.inf)):
            for x in (B.k, B.v):
                x[b][p, h] = np.nan
            v = np.ones((1, 2, 64), np.float32) * what
            other = 1 - h
            k1, v1 = B.k[b][p:p + 1].copy(), B.v[b][p:p + 1].copy()
            k1[:, h], v1[:, h] = 1.0, v[:, h]
            B.c.append(dev(k1, cache), dev(v1, cache), B.places(b, np.array([p])))
        out, lse = run(Q, B)
        B.check(out, lse)
        assert np.isnan(f64(out)[50:80, :2]).all() and not np.isnan(f64(out)[:50, :2]).any()
        mass(Q, B, {})
        # a query that is not finite: its own row alone
        q = B.q.clone()
        q[3, 1, 5], q[80, 2, 0] = math.inf, math.nan
        o2, _ = Q.attention_paged(q, *B.args(), lse=True)
        o2, o1 = f64(o2), f64(out)
        assert np.isnan(o2[3, 1]).all() and np.isnan(o2[80, 2]).all()
        o2[3, 1], o2[80, 2] = o1[3, 1], o1[80, 2]
        assert np.array_equal(o1, o2, equal_nan=True)
        B.c.close()


@pytest.mark.parametrize("cache,io", [(F16, F32), (F16, F16), (BF16, BF16), (BF16, F32)])
@pytest.mark.parametrize("scale", [1e-3, 30.0, 1e9])
def test_scores_of_every_size(Q, cache, io, scale):
    """From nearly equal weights to one that takes all (scores past 2^24 among them), with maxima that grow on the way."""
    rng = np.random.default_rng(30)
    for lens, new in (([500, 130], [1, 1]), ([400, 130], [100, 60])):
        B = Batch(Q, rng, cache, io, 4, 2, 64, 16, lens, new)
        if scale > 1e6:
            # keys that grow along the sequence, far apart beside the scores' rounding: the weights are those of one position
            for b, n in enumerate(lens):
                k = np.zeros((n, 2, 64))
                k[:, :, 3] = R.rounded(np.exp2(np.arange(n) % 11 - 5.0), cache)[:, None]
                B.k[b] = k
                B.c.append(dev(k, cache), dev(B.v[b], cache), B.places(b, np.arange(n)))
            got, _ = run(Q, B, dict(scale=scale))
            for b in range(len(lens)):
                qb = f64(B.q[B.starts[b]:B.starts[b + 1]])
                for i in range(new[b]):
                    n = lens[b] - new[b] + 1 + i
                    for head in range(4):
                        s = qb[i, head, 3] * B.k[b][:n, head // 2, 3] * scale
                        want = B.v[b][:n, head // 2][s == s.max()].mean(0)
                        close(got[B.starts[b] + i, head], want, 2.0 ** -20 * 5 + 4 * R.HALF_STEP[io] * (np.abs(want) + 1))
        else:
            B.check(*run(Q, B, dict(scale=scale)), scale=scale)
        B.c.close()


def test_values_of_any_size_keep_their_weights(Q):
    rng = np.random.default_rng(31)
    for cache, io, top in ((F16, F32, 6.0e4), (BF16, F32, 1e30), (BF16, BF16, 1e30)):
        B = Batch(Q, rng, cache, io, 4, 1, 64, 16, [300], [1])
        B.v[0] = R.rounded(B.v[0] * np.exp2(rng.integers(-10, 2, (300, 1, 64))) * top / 2.0 ** 4 / 6, cache)
        B.c.append(dev(B.k[0], cache), dev(B.v[0], cache), B.places(0, np.arange(300)))
        B.check(*run(Q, B))
        B.c.close()


def test_a_cache_of_more_than_4_gib(Q):
    rng = np.random.default_rng(40)
    page, kv, hd = 64, 8, 128
    pages = (5 << 30) // (page * kv * hd * 4)
    c = Q.GpuPagedCache(BF16, pages, kv, hd, page)
    assert c.nbytes > 5 * (1 << 30) - (1 << 20)
    n = 130
    tab = np.array([[pages - 1, 3, pages - 2]])
    k, v = (R.rounded(rng.normal(0, 1, (n, kv, hd)), BF16) for _ in range(2))
    at = i32(tab[0, np.arange(n) // page] * page + np.arange(n) % page)
    c.append(dev(k, BF16), dev(v, BF16), at)
    gk, gv = c.read(at)
    assert np.array_equal(f64(gk), k) and np.array_equal(f64(gv), v)
    q = dev(R.rounded(rng.normal(0, 1, (1, kv, hd)), BF16), BF16)
    out = Q.attention_paged(q, c, i32([0, 1]), i32([n]), i32(tab), 1, n)
    for h in range(kv):
        S = R.Scores(f64(q[:, h]), k[:, h], np.array([n - 1]), BF16, BF16)
        o, e, _, _ = R.attention(S, v[:, h], np.ones((1, n), bool), BF16, BF16)
        close(out[:, h], o, e)
    new = i32([[0, pages - 3]])
    m = dev(rng.uniform(0, 1, (1, kv, n)).astype(np.float32))
    kept, lens, _ = c.evict(m, i32([n]), 70, 10, i32(tab), new)
    gk, gv = c.read(i32(np.where(np.arange(70) < 64, np.arange(70), (pages - 3) * 64 + np.arange(70) - 64)))
    kept = kept.cpu().numpy()[0]
    for h in range(kv):
        assert np.array_equal(f64(gk[:, h]), k[kept[h], h]) and np.array_equal(f64(gv[:, h]), v[kept[h], h])
    c.close()
    torch.cuda.empty_cache()


# ---- eviction ----------------------------------------------------------------------------------------
@pytest.mark.parametrize("cache,hd,page", [(F16, 64, 16), (BF16, 128, 64), (F16, 40, 32), (BF16, 256, 16)])
@pytest.mark.parametrize("keep,recent", [(1, 0), (1, 1), (33, 0), (64, 20), (64, 64), (100, 7), (500, 50)])
def test_eviction(Q, cache, hd, page, keep, recent):
    rng = np.random.default_rng(hd + keep)
    lens, kv = [0, 1, 33, 64, 100, 101, 333], 2
    B = Batch(Q, rng, cache, cache, 2, kv, hd, page, lens, [0] * len(lens))
    pages = -(-keep // page)
    c = Q.GpuPagedCache(cache, B.c.n_pages + pages * len(lens) + 1, kv, hd, page)
    for b, n in enumerate(lens):
        if n:
            c.append(dev(B.k[b], cache), dev(B.v[b], cache), B.places(b, np.arange(n)))
    new = B.c.n_pages + rng.permutation(pages * len(lens)).reshape(len(lens), pages)
    m = np.round(rng.exponential(1, (len(lens), kv, 333)), 1).astype(np.float32)     # many are equal
    m[:, :, ::11] = 0.0
    m[2, 0, :5], m[4, 1, 3], m[4, 1, 7], m[5, 0, :101] = [np.nan, np.inf, -np.inf, -0.0, 0.0], np.nan, -1.0, 2.0
    buf = dev(np.concatenate([m, m[:, :, :3]], 2))                                    # rows further apart than they are wide
    kept, left, weights = c.evict(buf[:, :, :333], i32(lens), keep, recent, i32(B.tables), i32(new))
    kept, left, weights = kept.cpu().numpy(), left.cpu().numpy(), weights.cpu().numpy()
    rk, rv = c.read(i32(np.arange(c.n_pages * page)))
    rk, rv = f64(rk).reshape(-1, page, kv, hd), f64(rv).reshape(-1, page, kv, hd)
    for b, n in enumerate(lens):
        assert left[b] == min(n, keep)
        for h in range(kv):
            want = R.evict(m[b, h], n, keep, recent)
            assert kept[b, h].tolist() == want + [-1] * (keep - len(want))
            assert np.array_equal(weights[b, h, :len(want)], m[b, h][want], equal_nan=True) and not weights[b, h, len(want):].any()
            i = np.arange(len(want))
            assert np.array_equal(rk[new[b, i // page], i % page, h], B.k[b][want, h])
            assert np.array_equal(rv[new[b, i // page], i % page, h], B.v[b][want, h])
        for i in range(n):          # the old pages are as they were
            assert np.array_equal(rk[B.tables[b, i // page], i % page], B.k[b][i])
    assert not rk[-1].any()         # and a page that no table names
    c.close()
    B.c.close()


@pytest.mark.parametrize("n", [16383, 16384, 16385, 40000])
def test_eviction_of_long_sequences(Q, n):
    rng = np.random.default_rng(n)
    c = Q.GpuPagedCache(F16, 2 * -(-n // 1024), 1, 8, 1024)
    k = rng.normal(0, 1, (n, 1, 8)).astype(np.float16)
    c.append(dev(k), dev(-k), i32(np.arange(n)))
    tab = np.arange(-(-n // 1024))[None]
    for m in (rng.normal(0, 1, n).astype(np.float32), np.floor(rng.uniform(0, 5, n)).astype(np.float32), np.zeros(n, np.float32)):
        for keep, recent in ((n - 1, 0), (n // 3, 1000), (5, 2)):
            kept, _, _ = c.evict(dev(m.reshape(1, 1, n)), i32([n]), keep, recent, i32(tab), i32(tab + len(tab[0])))
            assert kept.cpu().numpy()[0, 0].tolist() == R.evict(m, n, keep, recent)
    c.close()


def test_eviction_with_pages_that_do_not_exist(Q):
    rng = np.random.default_rng(50)
    c = Q.GpuPagedCache(F16, 8, 1, 16, 16)
    k = rng.normal(0, 1, (64, 1, 16)).astype(np.float16)
    c.append(dev(k), dev(k), i32(np.arange(64)))
    m = dev(np.arange(64, dtype=np.float32).reshape(1, 1, 64))
    kept, lens, _ = c.evict(m, i32([70]), 40, 4, i32([[0, 99, 2, 3]]), i32([[4, -1, 6]]))     # (lengths beyond max_len count as that)
    assert int(lens) == 40 and kept.cpu().numpy().ravel().tolist() == list(range(24, 64))
    gk, _ = c.read(i32(np.arange(64, 128)))
    want = np.zeros((64, 1, 16))
    for i, p in enumerate(range(24, 64)):
        if i // 16 != 1:
            want[[0, None, 32][i // 16] + i % 16] = 0 if p // 16 == 1 else k[p]
    assert np.array_equal(f64(gk), want)


# ---- how calls are made -------------------------------------------------------------------------------
def test_refusals_with_a_cache(Q):
    from smallmind_amd import _lib
    rng = np.random.default_rng(60)
    B = Batch(Q, rng, F16, F32, 4, 2, 64, 16, [40], [2])
    h, lib, P = B.c._h, _lib.load(), ctypes.c_void_p(256)
    n = ctypes.c_int64()
    rules = _lib.AttentionRulesC

    def att(t=0, q=P, qs=256, out=P, lse=None, n_tok=2, nh=4, ns=1, st=P, le=P, ta=P, ts=3, mq=2, ml=40, r=None, w=P, wb=1 << 30):
        return lib.smx_attention_paged(h, t, q, qs, out, lse, n_tok, nh, ns, st, le, ta, ts, mq, ml, None if r is None else ctypes.byref(r), w, wb, None)
    odd = ctypes.c_void_p(257)
    for bad, code in ((dict(q=None), -1), (dict(out=None), -1), (dict(st=None), -1), (dict(le=None), -1), (dict(ta=None), -1), (dict(t=30), -5),
                      (dict(t=8), -5), (dict(nh=3), -1), (dict(nh=0), -1), (dict(n_tok=-1), -1), (dict(ns=0), -1), (dict(mq=0), -1), (dict(ml=-1), -1),
                      (dict(ml=(1 << 24) + 1, ts=1 << 21), -5), (dict(ts=2), -1), (dict(ts=-1), -1), (dict(qs=255), -1), (dict(q=odd), -1), (dict(out=odd), -1),
                      (dict(lse=odd), -1), (dict(st=odd), -1), (dict(n_tok=1 << 24), -5), (dict(w=ctypes.c_void_p(264)), -1),
                      (dict(r=rules(-1.0, 0.0, None, None, 0, 0)), -1), (dict(r=rules(0.0, float("nan"), None, None, 0, 0)), -1),
                      (dict(r=rules(0.0, 0.0, None, None, -1, 0)), -1), (dict(r=rules(0.0, 0.0, None, None, 0, 1)), -1),
                      (dict(r=rules(0.0, 0.0, 257, None, 0, 0)), -1), (dict(r=rules(0.0, 0.0, None, 258, 0, 0)), -1),
                      (dict(ml=40000, ts=4096, wb=16), -1), (dict(ml=40000, ts=4096, w=None), -1)):
        assert att(**bad) == code, bad
        assert b"smx_attention_paged" in lib.smx_last_error()
    assert lib.smx_attention_paged_work_bytes(h, 0, 2, 4, 1, 2, 40000, None, ctypes.byref(n)) == 0 and n.value > 16
    assert lib.smx_attention_paged_work_bytes(h, 0, 0, 4, 1, 2, 40000, None, ctypes.byref(n)) == 0 and n.value == 0

    def mas(lse=P, m=P, ms=40, mw=40, mo=P, q=P, w=P, wb=1 << 30):
        return lib.smx_attention_mass(h, 0, q, 256, lse, m, ms, mw, mo, 2, 4, 1, P, P, P, 3, 2, 40, None, w, wb, None)
    for bad in (dict(lse=None), dict(mo=None), dict(q=None), dict(ms=39), dict(mw=-1, ms=0), dict(ms=41), dict(lse=odd), dict(m=odd), dict(mo=odd)):
        assert mas(**bad) == -1, bad
    for args in ((0, 40, 32, 8, 3, 2), (1, 0, 32, 8, 3, 2), (1, 40, 0, 0, 3, 2), (1, 40, 32, 33, 3, 2), (1, 40, 32, -1, 3, 2), (1, 40, 32, 8, 2, 2),
                 (1, 40, 32, 8, 3, 1), (1, 41, 32, 8, 3, 2)):
        ns, ml, nk, nr, ts, ns2 = args
        assert lib.smx_paged_evict(h, P, 40, P, ns, ml, nk, nr, P, ts, P, ns2, P, P, P, None) == -1, args
    assert lib.smx_paged_evict(h, P, 40, P, 40000, 40, 32, 8, P, 3, P, 2, P, P, P, None) == -5
    assert lib.smx_paged_read(h, P, 1, ctypes.c_void_p(264), P, None) == -1
    assert lib.smx_paged_append(h, 0, None, 0, 0, P, 127, P, 128, None, None, 0.0, None, None, P, 1, 0, None, None) == -1
    assert lib.smx_paged_append(h, 0, P, 256, 4, P, 128, P, 128, None, None, 0.0, None, None, P, 1, 0, None, None) == -1
    with pytest.raises(ValueError, match="operands must be on"):
        Q.attention_paged(B.q.cpu(), *B.args())
    with pytest.raises(ValueError, match="operands must be on"):
        B.c.append(torch.zeros(1, 2, 64), torch.zeros(1, 2, 64), i32([0]))
    with pytest.raises(ValueError):
        B.c.append(torch.zeros(1, 2, 64).cuda(), torch.zeros(1, 2, 64).cuda().half(), i32([0]))
    out, _ = run(Q, B)
    B.check(out, _)             # the refused calls left nothing behind


def test_factors_beyond_fp32_are_refused(Q):
    from smallmind_amd._lib import SmxError
    B = Batch(Q, np.random.default_rng(65), F16, F32, 4, 2, 64, 16, [40], [2])
    for bad in (dict(scale=3e37), dict(cap=3e37), dict(cap=1e-40), dict(scale=10.0, cap=1e-37)):
        with pytest.raises(SmxError, match="range of fp32"):
            Q.attention_paged(B.q, *B.args(), **bad)
    out, lse = Q.attention_paged(B.q, *B.args(), lse=True, scale=1e-30, cap=1e30)      # (all scores all but 0)
    B.check(out, lse, scale=1e-30, cap=1e30)


def test_on_another_stream(Q):
    rng = np.random.default_rng(61)
    B = Batch(Q, rng, F16, F32, 4, 2, 64, 16, [3000, 70], [1, 30])
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        big = torch.randn(4096, 4096, device="cuda")
        for _ in range(20):
            big = big @ big * 1e-2
        q = B.q * (big[0, 0] * 0 + 1).nan_to_num(1.0)            # what the call reads comes late on its stream
        out, lse = Q.attention_paged(q, *B.args(), lse=True)
        m = Q.attention_mass(q, lse, *B.args())
    s.synchronize()
    B.check(out, lse)
    assert np.allclose(f64(m).sum((1, 2)), [4, 120], rtol=1e-4)


def test_captured_calls(Q):
    """A step in two graphs that run on different streams, replayed among eager work, with new inputs each time."""
    rng = np.random.default_rng(62)
    Bs = [Batch(Q, rng, F16, F32, 4, 2, 64, 16, lens, new) for lens, new in (([2900, 50], [1, 1]), ([1800, 90], [40, 3]))]
    cos, sin = tables(rng, 64, 32)
    rot = Q.Rotation(cos, sin, halves=True)
    graphs = []
    for B in Bs:
        B.steps = []
        n = B.q.shape[0]
        B.qs, B.outs = B.q.clone(), None
        tail = np.concatenate([B.places(b, np.arange(B.lens[b] - B.new[b], B.lens[b])).cpu().numpy() for b in range(2)])
        st = dict(k=dev(rng.normal(0, 1, (n, 2, 64)), F32), v=dev(rng.normal(0, 1, (n, 2, 64)), F32), places=i32(tail), pos=i32(np.arange(n) % 60),
                  new=i32(np.arange(2 * 4).reshape(2, 4)), args=B.args())
        spare = Q.GpuPagedCache(F16, 8, 2, 64, 16)

        def step(B=B, st=st):
            q = B.c.append(st["k"], st["v"], st["places"], q=B.qs, rotation=rot, pos=st["pos"])
            out, lse = Q.attention_paged(q, *st["args"], lse=True)
            m = Q.attention_mass(q, lse, *st["args"])
            return out, lse, m
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            step()
        s.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            outs = step()
        graphs.append((g, s, outs, step, st, B, spare))
    for rep in range(4):
        for g, s, outs, step, st, B, _ in graphs:
            B.qs.copy_(dev(rng.normal(0, 1.5, B.qs.shape), F32))
            st["k"].copy_(dev(rng.normal(0, 1, st["k"].shape), F32))
        torch.cuda.synchronize()
        for g, s, *_ in graphs:
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        got = [[x.clone() for x in outs] for _, _, outs, *_ in graphs]
        for (_, _, _, step, *_), have in zip(graphs, got):
            for x, y in zip(step(), have):
                assert torch.equal(x, y), rep
        torch.cuda.synchronize()


def test_captured_evictions(Q):
    """Two graphs of one cache, one whose rows move in the choosing launch and one with a launch for them."""
    rng = np.random.default_rng(64)
    for kv, hd, n, keep in ((2, 64, 700, 256), (2, 128, 900, 600)):
        page = 64
        pages, more = -(-n // page), -(-keep // page)
        c = Q.GpuPagedCache(BF16, 2 * pages + 4 * more, kv, hd, page)
        every = i32(np.arange(2 * pages * page))
        k = dev(rng.normal(0, 1, (len(every), kv, hd)), BF16)
        c.append(k, -k, every)
        tab, new = i32(np.arange(2 * pages).reshape(2, pages)), [i32(2 * pages + 2 * more * i + np.arange(2 * more).reshape(2, more)) for i in (0, 1)]
        mass, lens = dev(rng.uniform(0, 1, (2, kv, n)).astype(np.float32)), i32([n, n // 2])
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            c.evict(mass, lens, keep, 17, tab, new[0])
        s.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            outs = c.evict(mass, lens, keep, 17, tab, new[0])
        places = [i32((x.cpu().numpy()[:, :, None] * page + np.arange(page)).reshape(-1)) for x in new]
        for rep in range(4):
            mass.copy_(dev(np.floor(rng.uniform(0, 50 + rep, mass.shape)).astype(np.float32)))
            lens.copy_(i32([n - rep, n // 3 + rep]))
            torch.cuda.synchronize()
            g.replay()
            want = c.evict(mass, lens, keep, 17, tab, new[1])
            torch.cuda.synchronize()
            m, ln = mass.cpu().numpy(), lens.cpu().numpy()
            for x, y in zip(outs, want):
                assert torch.equal(x, y), rep
            for b in range(2):
                for h in range(kv):
                    assert [p for p in outs[0][b, h].tolist() if p >= 0] == R.evict(m[b, h], ln[b], keep, 17)
            for x, y in zip(c.read(places[0]), c.read(places[1])):
                for b in range(2):          # (beyond the rows kept now lie those that an earlier call kept)
                    rows = slice(b * more * page, b * more * page + int(outs[1][b]))
                    assert torch.equal(x[rows], y[rows]), rep
        c.close()


def test_the_same_call_twice_gives_the_same_bits(Q):
    rng = np.random.default_rng(63)
    B = Batch(Q, rng, BF16, BF16, 8, 2, 128, 16, [3000, 300, 64], [1, 200, 64])
    a, b = run(Q, B), run(Q, B)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    m = [Q.attention_mass(B.q, a[1], *B.args()) for _ in range(2)]
    assert torch.equal(*m)
    # in place: over what there was, from and to one tensor
    from smallmind_amd import _lib
    before = dev(rng.uniform(0, 1, m[0].shape).astype(np.float32))
    want = Q.attention_mass(B.q, a[1], *B.args(), mass=before)
    c, st, le, ta, mq, ml = B.args()
    need = ctypes.c_int64()
    _lib.call("smx_attention_mass_work_bytes", c._h, 30, 8, 3, mq, ml, ctypes.byref(need))
    work = torch.empty(max(need.value, 16), dtype=torch.uint8, device="cuda")
    _lib.call("smx_attention_mass", c._h, 30, B.q.data_ptr(), B.q.stride(0), a[1].data_ptr(), before.data_ptr(), ml, ml, before.data_ptr(),
              B.q.shape[0], 8, 3, st.data_ptr(), le.data_ptr(), ta.data_ptr(), ta.shape[1], mq, ml, None, work.data_ptr(), work.numel(),
              torch.cuda.current_stream().cuda_stream)
    assert torch.equal(before, want)


def test_a_conversation(Q):
    """The operators as a server uses them: prompts in chunks, decoding, an eviction when the pages run short, decoding on
    over what is left; every step against the plain form over what the cache says it holds."""
    rng = np.random.default_rng(70)
    H, kv, hd, page, n_seq = 6, 2, 64, 16, 3
    c = Q.GpuPagedCache(BF16, 64, kv, hd, page)
    cos, sin = tables(rng, 400, 16)
    rot = Q.Rotation(cos, sin, [6, 5, 5], halves=True)
    gq, gk = (dev(rng.normal(1, 0.2, hd).astype(np.float32)) for _ in range(2))
    table = np.arange(n_seq * 12).reshape(n_seq, 12)
    lens, at, total = np.zeros(n_seq, int), np.zeros(n_seq, int), None

    def step(new):
        nonlocal lens, at, total
        new = np.array(new)
        n = new.sum()
        seqs = np.repeat(np.arange(n_seq), new)
        i = np.concatenate([np.arange(m) for m in new])
        pos, idx = at[seqs] + i, lens[seqs] + i
        places = i32(table[seqs, idx // page] * page + idx % page)
        q, k, v = (dev(rng.normal(0, 1, (n, h, hd)), F32) for h in (H, kv, kv))
        p3 = i32(np.stack([pos, pos // 4, pos % 4]))
        q = c.append(k, v, places, q=q, q_gamma=gq, k_gamma=gk, rotation=rot, pos=p3, dtype=BF16)
        lens, at = lens + new, at + new
        starts = np.concatenate([[0], np.cumsum(new)])
        a = (c, i32(starts), i32(lens), i32(table), int(new.max()), int(lens.max()))
        out, lse = Q.attention_paged(q, *a, window=64, prefix=i32([4] * n_seq), lse=True)
        total = Q.attention_mass(q, lse, *a, mass=total, window=64, prefix=i32([4] * n_seq))
        for b in range(n_seq):
            n = lens[b]
            k, v = (f64(x) for x in c.read(i32(table[b, np.arange(n) // page] * page + np.arange(n) % page)))
            see = R.visible(n - new[b], new[b], n, 4, 64)
            for h in range(H):
                S = R.Scores(f64(q[starts[b]:starts[b + 1], h]), k[:, h // 3], None, BF16, BF16)
                o, e, _, _ = R.attention(S, v[:, h // 3], see, BF16, BF16)
                close(out[starts[b]:starts[b + 1], h], o, e)

    step([40, 7, 100])
    step([33, 1, 1])
    step([1, 50, 1])
    weights = f64(total)
    assert np.allclose(weights.sum(2), (lens * 3)[:, None], rtol=1e-4)
    new_table = 36 + np.arange(n_seq * 4).reshape(n_seq, 4)
    kept, left, total = c.evict(total, i32(lens), 48, 16, i32(table), i32(new_table))
    for b in range(n_seq):
        for h in range(kv):
            assert [p for p in kept[b, h].tolist() if p >= 0] == R.evict(weights[b, h].astype(np.float32), lens[b], 48, 16)
    lens, table = left.cpu().numpy().astype(int), np.concatenate([new_table, np.arange(36).reshape(n_seq, 12)[:, :8]], 1)
    step([1, 1, 1])
    step([1, 20, 1])
    c.close()


@pytest.mark.parametrize("n_seq", [130, 64, 70])
def test_many_sequences_of_different_lengths(Q, n_seq):
    """More workgroups than start at once: the longest sequences go first, equal ones and empty ones among them."""
    rng = np.random.default_rng(n_seq)
    lens = [int(n) for n in rng.integers(0, 90, n_seq)]
    lens[3], lens[-1], lens[10], lens[11] = 0, 4200, 77, 77
    new = [min(n, 1) for n in lens]
    B = Batch(Q, rng, F16, F32, 8, 8, 64, 16, lens, new, pad=2)
    out, lse = run(Q, B)
    B.check(out, lse, every=5)
    before = dev(rng.uniform(0, 1, (n_seq, 8, 100)).astype(np.float32))
    mass(Q, B, {}, before)


@pytest.mark.parametrize("cache,io", [(F16, F32), (BF16, BF16), (F16, F16), (BF16, F32)])
@pytest.mark.parametrize("H,kv", [(4, 2), (40, 1)])
def test_rows_that_see_nothing_whatever_their_query(Q, cache, io, H, kv):
    """Tokens before position 0, and one whose only position lies on a page that does not exist."""
    rng = np.random.default_rng(H)
    B = Batch(Q, rng, cache, io, H, kv, 64, 16, [3, 40], [7, 2])
    B.tables[1, 2] = -1
    B.q[2, 0, 3], B.q[3, H - 1, 0], B.q[8, 1, 9] = math.nan, math.inf, math.nan
    out, lse = run(Q, B, dict(window=1))
    blind = np.array([True] * 4 + [False] * 3 + [True] * 2)
    assert not out[blind].any() and bool((lse[blind] == -math.inf).all())
    assert np.isfinite(f64(out)[~blind]).all() and np.isfinite(f64(lse)[~blind]).all()
    B.c.close()


@pytest.mark.parametrize("cache,io,hd", [(BF16, BF16, 128), (F16, F16, 64), (F16, F32, 64), (BF16, F32, 128)])
@pytest.mark.parametrize("lens,new", [([5000, 30], [1, 1]), ([4000, 50], [40, 3]), ([300, 40], [200, 2])])
def test_queries_that_are_not_finite_in_contexts_of_parts(Q, cache, io, hd, lens, new):
    """Each its own row alone, whatever number of workgroups goes through the positions."""
    rng = np.random.default_rng([hd, lens[0]])
    B = Batch(Q, rng, cache, io, 4, 1, hd, 32, lens, new)
    clean, sums = (f64(x) for x in run(Q, B))
    for t, head, d, what in ((0, 1, 7, math.inf), (sum(new) - 1, 0, 0, -math.inf), (new[0] - 1, 3, hd - 1, math.nan), (new[0], 2, 5, math.inf)):
        B.q[t, head, d] = what
        clean[t, head], sums[t, head] = np.nan, np.nan
    out, lse = (f64(x) for x in run(Q, B))
    assert np.array_equal(out, clean, equal_nan=True) and np.array_equal(lse, sums, equal_nan=True)
    B.c.close()


# ---- what is not finite, and the ends of the ranges ---------------------------------------------------
def received(Q, B, lse, hidden=None, **rules):
    """attention_mass against the plain form with this lse; hidden: positions of sequence 0 that lie on pages that do not exist."""
    got = f64(Q.attention_mass(B.q, lse, *B.args(), **kernel_rules(rules)))
    l64 = f64(lse)
    for b in range(len(B.lens)):
        want, bound = np.zeros((B.kv, B.max_len)), np.zeros((B.kv, B.max_len))
        for h, head, S, see in B.rows(b, **rules):
            if hidden is not None and b == 0:
                see = see & ~hidden
            l = l64[B.starts[b]:B.starts[b + 1], head]
            w, e = R.received(S, np.where(np.isneginf(l), np.inf, l), see)
            want[h, :B.lens[b]] += w
            bound[h, :B.lens[b]] += e + 2.0 ** -24 * np.nan_to_num(w) * 4
        close(torch.from_numpy(got[b]), want, np.nan_to_num(bound))


@pytest.mark.parametrize("cache,io,hd", [(F16, F32, 64), (BF16, BF16, 128), (F16, F16, 64), (BF16, F32, 192)])
@pytest.mark.parametrize("rules", [{}, dict(window=37), dict(window=20, prefix=True), dict(window=50, cap=20.0), dict(window=90, slopes=True)])
@pytest.mark.parametrize("lens,new", [([100, 333], [1, 3]), ([200, 131], [150, 64]), ([900, 20], [700, 5])])
def test_received_weights_of_rows_that_are_not_finite(Q, cache, io, hd, rules, lens, new):
    """A query that is not finite, and positions that are not, count where they are seen and nowhere else."""
    rng = np.random.default_rng([hd, lens[0]])
    H, kv = 4, 2
    B = Batch(Q, rng, cache, io, H, kv, hd, 16, lens, new)
    rules = dict(rules)
    if rules.get("slopes"):
        rules["slopes"] = np.array([0.3, 0.1, 0.02, 0.0], np.float32)
    if rules.get("prefix"):
        rules["prefix"] = [9, 3]
    # a page that the cache does not have, before the last tokens of sequence 0
    gone = (lens[0] - 20) // 16
    B.tables[0, gone] = -1
    hidden = np.arange(lens[0]) // 16 == gone
    B.q[new[0] // 3, 1, 5] = math.nan
    B.q[B.starts[1], 2, 0] = math.inf
    B.q[new[0] // 2, 3, hd - 1] = -math.inf

    def check():
        _, lse = run(Q, B, rules)
        l = f64(lse)
        assert np.isnan(l[new[0] // 3, 1]) and np.isnan(l[B.starts[1], 2]) and np.isnan(l[new[0] // 2, 3])
        received(Q, B, lse, hidden, **rules)
    check()
    for b, p, h in ((0, lens[0] - new[0] // 2 - 1, 0), (1, lens[1] - 2, 1)):
        B.k[b][p, h] = B.v[b][p, h] = math.nan
        B.c.append(dev(B.k[b][p:p + 1], cache), dev(B.v[b][p:p + 1], cache), B.places(b, np.array([p])))
    check()
    B.c.close()


@pytest.mark.parametrize("new", [[1, 2], [70, 30]])
@pytest.mark.parametrize("scale", [1e-12, 1e-30, 1e-44])
def test_scores_below_fp32(Q, new, scale):
    """Queries of nothing, or all but nothing, and a scale that together leave fp32: every position counts alike."""
    rng = np.random.default_rng(77)
    for cache, io in ((F16, F32), (F16, F16), (BF16, F32)):
        B = Batch(Q, rng, cache, io, 4, 2, 64, 16, [100, 45], new)
        B.q[::2] = 0.0
        B.q[1::2] *= 2.0 ** -20
        B.check(*run(Q, B, dict(scale=scale)), scale=scale)
        mass(Q, B, dict(scale=scale))
        B.c.close()


@pytest.mark.parametrize("cache,io", [(F16, F16), (BF16, BF16), (F16, F32)])
@pytest.mark.parametrize("cap,scale", [(130.0, None), (5000.0, None), (1e6, None), (1e30, None), (1e36, 1e-6)])
@pytest.mark.parametrize("lens,new", [([300, 65], [1, 3]), ([260, 97], [130, 40])])
def test_caps_far_above_the_scores(Q, cache, io, cap, scale, lens, new):
    """The cap then changes little, and is off by little: 2^-20 of the score where tanh is computed, whatever the cap."""
    rng = np.random.default_rng(int(math.log2(cap)))
    if scale:
        cache = io = BF16
    B = Batch(Q, rng, cache, io, 4, 2, 64, 16, lens, new)
    if scale:
        B.q *= 2.0 ** 17     # (products of some 10^6 to 10^7)
    rules = dict(cap=cap) if scale is None else dict(cap=cap, scale=scale)
    out, lse = run(Q, B, rules)
    for b in range(len(lens)):
        at = slice(B.starts[b], B.starts[b + 1])
        for h, head, S, see in B.rows(b, **rules):
            if io == cache:
                # (that of the score without a cap, and the tanh's)
                S.e = R.Scores(f64(B.q[at, head]), B.k[b][:, h], None, io, cache, scale).e + np.abs(S.s) * 2.0 ** -20
            o, e, l, le = R.attention(S, B.v[b][:, h], see, io, cache)
            close(out[at, head], o, e)
            close(lse[at, head], l, le)
    B.c.close()


@pytest.mark.parametrize("cap", [128.0, 3000.0])
def test_large_caps_of_many_blocks(Q, cap):
    """More than two blocks for every compute unit, with a cap at and above the quick tanh's."""
    rng = np.random.default_rng(79)
    for cache, hd in ((F16, 64), (BF16, 32)):
        B = Batch(Q, rng, cache, cache, 300, 300, hd, 16, [200, 90, 33], [170, 40, 1])
        out, lse = run(Q, B, dict(cap=cap))
        for b in range(3):
            at = slice(B.starts[b], B.starts[b + 1])
            for h, head, S, see in B.rows(b, cap=cap, every=17):
                S.e = R.Scores(f64(B.q[at, head]), B.k[b][:, h], None, cache, cache).e + (np.abs(S.s) * 2.0 ** -20 if cap > 128 else cap * 2.0 ** -21)
                o, e, l, le = R.attention(S, B.v[b][:, h], see, cache, cache)
                close(out[at, head], o, e)
                close(lse[at, head], l, le)
        B.c.close()


@pytest.mark.parametrize("exponent,gamma,tin", [(126, 1, F32), (126, 1, BF16), (60, 72, F32), (60, 72, BF16), (-60, -80, F32), (-60, -80, BF16),
                                                (-132, 0, F32), (-140, 3, F32), (-132, 0, BF16)])
@pytest.mark.parametrize("hd,halves", [(8, True), (104, False), (128, True), (256, False)])
def test_norms_at_the_ends_of_the_range(Q, hd, halves, exponent, gamma, tin):
    """Rows, and weights, whose products leave fp32 though what they come to does not; beside ordinary rows."""
    rng = np.random.default_rng([hd, 300 + exponent])
    n = 9
    x = np.clip(rng.normal(0, 0.6, (n, 3, hd)), -1.9, 1.9) * np.exp2(np.where(rng.uniform(size=(n, 3, 1)) < 0.6, exponent, 0))
    x = dev(x, tin)
    assert bool(torch.isfinite(x).all()) and bool((x.double().abs().amax(2) > 0).all())
    g = (rng.normal(1, 0.3, hd) * 2.0 ** gamma).astype(np.float32)
    cos, sin = tables(rng, 16, hd // 2)
    pos = rng.integers(0, 16, (1, n)).astype(np.int32)
    a = dev(g), dev(g), 0.0, Q.Rotation(cos, sin, halves=halves), dev(pos)
    q, k = Q.qk_norm_rope(x, x[:, :2], *a, dtype=F32)
    want, e = R.turned(f64(x), g, 0.0, cos.cpu().numpy(), sin.cpu().numpy(), pos, [hd // 2], halves)
    close(q, want, e)
    close(k, want[:, :2], e[:, :2])
    c = Q.GpuPagedCache(BF16, 1, 2, hd, 16)
    c.append(x[:, :2], torch.ones_like(x[:, :2]), i32(np.arange(n)), q_gamma=a[0], k_gamma=a[1], eps=0.0, rotation=a[3], pos=a[4])
    close(c.read(i32(np.arange(n)))[0], want[:, :2], e[:, :2] + R.HALF_STEP[BF16] * (np.abs(want) + e)[:, :2])
    c.close()


@pytest.mark.parametrize("tin", [F16, BF16, F32])
def test_rows_of_zeros_with_the_least_eps(Q, tin):
    x = torch.zeros(3, 2, 64, dtype=tin, device="cuda")
    x[1] = 1.0
    g = torch.ones(64, device="cuda")
    q, _ = Q.qk_norm_rope(x, x, g, g, 1e-40, dtype=F32)
    close(q, f64(x), 72 * 2.0 ** -24)


def test_outputs_in_the_inputs_memory_are_refused(Q):
    from smallmind_amd._lib import SmxError
    rng = np.random.default_rng(80)
    B = Batch(Q, rng, F16, F16, 4, 2, 64, 16, [40, 9], [3, 1])
    n, row = 4, 4 * 64
    buf = torch.zeros(8 * n * row, dtype=F16, device="cuda")
    q = buf[n * row:2 * n * row].view(n, 4, 64).copy_(B.q)
    for at in (n * row, row, 2 * n * row - 8):                        # on q, from before it into it, on its end
        with pytest.raises(SmxError, match="lies in q's memory"):
            Q.attention_paged(q, *B.args(), out=buf[at:at + n * row].view(n, 4, 64))
    for at in (0, 2 * n * row):                                       # right before it, right behind
        out, lse = Q.attention_paged(q, *B.args(), out=buf[at:at + n * row].view(n, 4, 64), lse=True)
        assert out.data_ptr() == buf.data_ptr() + 2 * at
        B.check(out, lse)
    # between rows of q that lie far apart
    wide = buf.view(n, -1)[:, :row].unflatten(1, (4, 64)).copy_(B.q)
    B.check(*Q.attention_paged(wide, *B.args(), out=buf[row:row + n * row].view(n, 4, 64), lse=True))
    with pytest.raises(SmxError, match="lies in q's memory"):
        Q.attention_paged(wide, *B.args(), out=buf[5 * row:9 * row].view(n, 4, 64))
    B.c.close()


def test_outputs_of_rows_that_are_not_there_are_not_looked_at(Q):
    from smallmind_amd import _lib
    f, out = torch.randn(3, 2, 64, device="cuda"), torch.zeros(3, 2, 64, device="cuda")
    s = torch.cuda.current_stream().cuda_stream
    for q, k in ((f.data_ptr(), None), (None, f.data_ptr())):     # (the other's output names the input)
        qo, ko = (out.data_ptr(), f.data_ptr()) if q else (f.data_ptr(), out.data_ptr())
        out.zero_()
        _lib.call("smx_qk_norm_rope", 0, q, 128, 2, k, 128, 2, 64, None, None, 0.0, None, None, 3, 0, qo, ko, s)
        assert torch.equal(out, f)


def test_appends_into_their_inputs_are_refused(Q):
    from smallmind_amd import _lib
    lib, s = _lib.load(), torch.cuda.current_stream().cuda_stream
    c = Q.GpuPagedCache(F16, 1, 1, 64, 16)
    f = torch.randn(3, 256, device="cuda")                 # rows of 2 + 1 + 1 heads
    out, at = torch.zeros(3, 2, 64, device="cuda"), i32([0, 1, 2])

    def append(to):
        return lib.smx_paged_append(c._h, 0, f.data_ptr(), 256, 2, f.data_ptr() + 512, 256, f.data_ptr() + 768, 256, None, None, 0.0, None, None,
                                    at.data_ptr(), 3, 0, to, s)
    for off in (0, 512, 764, 2 * 1024 + 1020, -4):
        assert append(f.data_ptr() + off) == -1 and b"lies in the inputs' memory" in lib.smx_last_error()
    assert append(out.data_ptr()) == 0
    assert torch.equal(out.flatten(1), f[:, :128])
    assert torch.equal(c.read(at)[1].flatten(1), f[:, 192:].half())
    c.close()


def test_a_bound_of_new_tokens_that_says_nothing(Q):
    """max_q 2^31 - 1, for 4096 sequences of up to 2048 positions, all but three of them empty: the plan's numbers stay in range."""
    rng = np.random.default_rng(81)
    n = 4096
    B = Batch(Q, rng, BF16, BF16, 64, 8, 128, 1024, [40, 900, 0] + [0] * (n - 4) + [77], [5, 60, 0] + [0] * (n - 4) + [1])
    tab = i32(np.concatenate([B.tables, np.full((n, 1), -1)], 1))
    a = B.c, i32(B.starts), i32(B.lens), tab
    want, lse = Q.attention_paged(B.q, *a, 60, 900, lse=True)
    out, got = Q.attention_paged(B.q, *a, 2 ** 31 - 1, 2048, lse=True)
    B.check(out, got, every=8)
    B.check(want, lse, every=8)
    few, many = (f64(Q.attention_mass(B.q, lse, *a, q, 2048)[[0, 1, 2, n - 1]]) for q in (60, 2 ** 31 - 1))
    # (both add up each position's up to 480 weights in some order)
    assert not few[2].any() and (few[1].sum() > 0) and (np.abs(few - many) <= (480 + 70) * 2.0 ** -24 * 2 * few).all()
    assert not many[:, :, 900:].any()
    B.c.close()


@pytest.mark.parametrize("cache,io", [(F16, F16), (BF16, BF16), (F16, F32)])
@pytest.mark.parametrize("lens,new", [([300, 65], [1, 3]), ([260, 97], [130, 40])])
def test_received_weights_by_the_attentions_own_sums(Q, cache, io, lens, new):
    """With a cap, 16-bit queries' lse is off by 2^-21 of it where the weights' scores are not: a weight by as much of itself."""
    rng = np.random.default_rng(78)
    for rules in (dict(cap=50.0), dict(cap=30.0, scale=0.5, window=60), dict(slopes=np.array([0.3, 0.1, 0.02, 0.0], np.float32))):
        B = Batch(Q, rng, cache, io, 4, 2, 64, 16, lens, new)
        _, lse = run(Q, B, rules)
        got = f64(Q.attention_mass(B.q, lse, *B.args(), **kernel_rules(rules)))
        for b in range(len(lens)):
            want, bound = np.zeros((2, B.max_len)), np.zeros((2, B.max_len))
            for h, head, S, see in B.rows(b, **rules):
                _, _, l, le = R.attention(S, B.v[b][:, h], see, io, cache)
                w, e = R.received(S, l, see)
                each = np.where(see, np.exp(S.s - l[:, None]), 0.0)
                want[h, :lens[b]] += w
                bound[h, :lens[b]] += e + le @ each + 2.0 ** -24 * w * 4
            close(torch.from_numpy(got[b]), want, bound)
        B.c.close()


def test_evictions_and_received_weights_over_their_inputs_are_refused(Q):
    from smallmind_amd import _lib
    lib, s = _lib.load(), torch.cuda.current_stream().cuda_stream
    rng = np.random.default_rng(82)
    B = Batch(Q, rng, F16, F16, 4, 2, 64, 16, [40, 30], [2, 1], extra_pages=8)
    i = i32(np.zeros(256))
    m = dev(rng.uniform(0, 1, (2, 2, 48)).astype(np.float32))
    lens, tab, new = i32(B.lens), i32(B.tables), i32(np.full((2, 1), -1))

    def evict(kept=i.data_ptr(), left=i.data_ptr() + 512, mass=i.data_ptr() + 600):
        return lib.smx_paged_evict(B.c._h, m.data_ptr(), 48, lens.data_ptr(), 2, 40, 8, 2, tab.data_ptr(), 3, new.data_ptr(), 1, kept, left, mass, s)
    for bad in (dict(left=lens.data_ptr()), dict(mass=m.data_ptr()), dict(mass=m.data_ptr() + 4 * (3 * 48 + 39)), dict(kept=tab.data_ptr()),
                dict(kept=new.data_ptr()), dict(kept=lens.data_ptr() - 124)):
        assert evict(**bad) == -1 and b"lies in the inputs' memory" in lib.smx_last_error(), bad
    assert evict() == 0
    got = i.cpu().numpy()
    assert got[128:130].tolist() == [8, 8]
    for b in range(2):
        for h in range(2):
            assert got[:32].reshape(2, 2, 8)[b, h].tolist() == R.evict(m[b, h].cpu().numpy(), B.lens[b], 8, 2)

    _, lse = run(Q, B)
    c, st, le, ta, mq, ml = B.args()
    out = torch.zeros(2 * 2 * 40 + 64, device="cuda")
    was = out[:2 * 2 * 30]

    def mass(to, width=30, stride=30):
        return lib.smx_attention_mass(B.c._h, 1, B.q.data_ptr(), B.q.stride(0), lse.data_ptr(), was.data_ptr(), stride, width, to, 3, 4, 2, st.data_ptr(),
                                      le.data_ptr(), ta.data_ptr(), ta.shape[1], mq, ml, None, None, 0, s)
    for to in (was.data_ptr() + 4, was.data_ptr() + 4 * 119):
        assert mass(to) == -1 and b"overlap" in lib.smx_last_error()
    assert mass(m.data_ptr()) == 0 and mass(was.data_ptr(), 40, 40) == 0
    assert torch.equal(m.flatten()[:160], out[:160])
    B.c.close()
