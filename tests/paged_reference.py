"""Plain 64-bit forms of the operators over a paged KV cache, with bounds for what 32 bits and the matrix operands' types may
differ by."""
from __future__ import annotations

import math

import numpy as np
import torch

HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}   # relative
LEAST = {torch.float32: 2.0 ** -150, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}     # absolute


def rounded(x, dtype):
    """x (64-bit numpy) rounded once to dtype, as 64-bit numpy."""
    return torch.from_numpy(np.asarray(x, np.float64)).to(dtype).double().numpy()


def held(k, v, dtype):
    """What the cache gives back for rows k, v [..., hd]: rounded, NaN in both where either then is not finite."""
    with np.errstate(over="ignore"):
        k, v = rounded(k, dtype), rounded(v, dtype)
    bad = ~(np.isfinite(k).all(-1) & np.isfinite(v).all(-1))
    k[bad], v[bad] = np.nan, np.nan
    return k, v


def turned(x, gamma, eps, cos, sin, pos, sections, halves):
    """(rows x [n][heads][hd] normed and turned, how far fp32 arithmetic may be off).  pos [axes][n]; cos None: no rotation.

    The sum of squares has hd roundings, its mean, root, reciprocal and the two products 6 more: (hd + 8) 2^-24 of a value
    v.  A turned value is a sum of two products, each with its own rounding and that of the sum: 3 2^-24 of |a| + |b|
    more (the tables' values are inputs)."""
    x = np.asarray(x, np.float64)
    hd = x.shape[-1]
    e = np.zeros_like(x)
    if gamma is not None:
        x = x / np.sqrt((x ** 2).mean(-1, keepdims=True) + eps) * np.asarray(gamma, np.float64)
        e = np.abs(x) * (hd + 8) * 2.0 ** -24
    if cos is None:
        return x, e
    half = cos.shape[1]
    axis = np.repeat(np.arange(len(sections)), sections)
    at = np.stack([pos[a] for a in axis], 1)                       # [n][half]
    ok = (at >= 0) & (at < cos.shape[0])
    at = np.clip(at, 0, cos.shape[0] - 1)
    c = np.where(ok, cos.astype(np.float64)[at, np.arange(half)], np.nan)[:, None]
    s = np.where(ok, sin.astype(np.float64)[at, np.arange(half)], np.nan)[:, None]
    ia, ib = (np.arange(half), np.arange(half) + half) if halves else (2 * np.arange(half), 2 * np.arange(half) + 1)
    y, f = x.copy(), e.copy()
    a, b = x[..., ia], x[..., ib]
    y[..., ia], y[..., ib] = a * c - b * s, a * s + b * c
    both = np.abs(a * c) + np.abs(b * s), np.abs(a * s) + np.abs(b * c)
    f[..., ia], f[..., ib] = ((hd + 12) * 2.0 ** -24 * z for z in both)
    return y, f


def visible(first, m, n, prefix=0, window=0):
    """Which of n positions each of m tokens from position `first` on sees."""
    t, p = np.arange(first, first + m)[:, None], np.arange(n)
    see = (p <= t) & ((p > t - window) if window else True)
    return see | (p < prefix)


class Scores:
    """Scores of rows (tokens of one head) over n positions, and how far off each may be, in 64 bits.

    parts: an operand of fp32 queries is off by 2^-22 (F16 cache: two parts) or 2^-24 (BF16: three) of itself and, over F16,
    by 2^-38 of the row's largest; cache-typed ones are exact.  hd products per part are added in fp32, each sum within 2^-23 of
    what has been added (the matrix unit may truncate).  Three roundings turn a product into an exponent; a cap adds 2^-20
    of the score (the exponential branch of tanh: its argument, the exponential, 1 - e next to 0.4, the reciprocal) or, with
    cache-typed outputs, 2^-21 of the cap (1 - 2 / (1 + f): f is off by 2^-23 and by |2 y| 2^-24 of itself, the
    derivative 2 f / (1 + f)^2 is at most 1/2 and falls faster than |y| grows; the sum, the reciprocal (2^-23 of at most 1, twice) and the last
    sum), a bias 4 roundings of the larger of the two."""

    def __init__(self, q, k, t, io, cache, scale=None, cap=0.0, slope=0.0):
        q, k = np.asarray(q, np.float64), np.asarray(k, np.float64)
        hd = q.shape[-1]
        scale = 1.0 / math.sqrt(hd) if scale is None else float(np.float32(scale))
        parts = 1 if io == cache else 2 if cache == torch.float16 else 3
        with np.errstate(invalid="ignore"):
            s = scale * (q @ k.T)
            size = scale * (np.abs(q) @ np.abs(k).T)
            e = size * (parts * hd + 2) * 2.0 ** -23
            if parts > 1:
                e = e + size * (2.0 ** -22 if parts == 2 else 2.0 ** -24)
                if parts == 2:
                    e = e + scale * np.abs(q).max(-1, keepdims=True, initial=0) * np.abs(k).sum(-1) * 2.0 ** -38
            if cap:
                cap = float(np.float32(cap))
                s = cap * np.tanh(s / cap)
                e = e + (cap * 2.0 ** -21 if parts == 1 else np.abs(s) * 2.0 ** -20)
            if slope:
                bias = float(np.float32(slope)) * np.abs(t[:, None] - np.arange(k.shape[0]))
                e = e + 4 * 2.0 ** -24 * (np.abs(s) + bias)
                s = s - bias
            self.s, self.e = s, e + 3 * np.abs(s) * 2.0 ** -24


def attention(S, v, see, io, cache):
    """(out [rows][hd], its bound, lse [rows], its bound).

    Weight j is off by e_j + e_max + 2^-22 (exponential) of itself, by the rounding of its matrix operand (2^-22 or 2^-24 in
    parts, half a step of the type without), and over F16 by 2^-31 of the largest.  Each enters the numerator; the sum S of the
    weights moves by the first two.  The sums have 3 n + 80 roundings (parts, waves, the joining) of 2^-23.  The result is
    rounded to its type.  The exponent is taken from a reference up to 2^8 below the largest: |s| 2^-24 again, in 3 |s| above."""
    rows, hd = S.s.shape[0], v.shape[1]
    out, bound = np.zeros((rows, hd)), np.zeros((rows, hd))
    lse, lbound = np.full(rows, -np.inf), np.zeros(rows)
    same = io == cache
    op = HALF_STEP[cache] if same else 2.0 ** -22 if cache == torch.float16 else 2.0 ** -24
    for r in range(rows):
        j = see[r]
        n = int(j.sum())
        if not n:
            continue
        s, e, vv = S.s[r, j], S.e[r, j], v[j]
        if np.isnan(s).any():
            out[r], lse[r] = np.nan, np.nan
            continue
        top = s.max()
        p = np.exp(s - top)
        total, A = p.sum(), p @ np.abs(vv)
        e = e + e[s.argmax()] + 3 * abs(top) * 2.0 ** -24 + 2.0 ** -22
        out[r] = p @ vv / total
        lse[r] = top + math.log(total)
        drift = (p @ e) / total + (n + 80) * 2.0 ** -23
        bound[r] = ((p * e) @ np.abs(vv) + A * (drift + op + (3 * n + 80) * 2.0 ** -23)) / total
        if cache == torch.float16:
            bound[r] += 2.0 ** -31 * np.abs(vv).sum(0) / total
        bound[r] += HALF_STEP[io] * (np.abs(out[r]) + bound[r]) + LEAST[io]
        lbound[r] = drift + abs(lse[r]) * 2.0 ** -22 + 2.0 ** -22
    return out, bound, lse, lbound


def received(S, lse, see):
    """(weights that n positions receive from rows with these lse, summed, their bound): each weight off by its score's e, the
    roundings of lse and of the difference, the exponential; the sum by a rounding per row."""
    s, e = np.where(see, S.s, -np.inf), np.where(see, S.e, 0.0)
    with np.errstate(invalid="ignore"):
        w = np.where(see, np.exp(s - lse[:, None]), 0.0)
        l = np.where(np.isfinite(lse), np.abs(lse), 0.0)[:, None]
        off = w * (e + (3 * l + np.where(see, np.abs(S.s), 0.0)) * 2.0 ** -24 + 2.0 ** -22)
        total = w.sum(0)
        return total, off.sum(0) + total * (S.s.shape[0] + 70) * 2.0 ** -24


def evict(mass, n, n_keep, n_recent):
    """Positions of n that are kept, in order."""
    keep = min(n, n_keep)
    recent = min(n_recent, keep)
    cand = n - recent
    m = np.asarray(mass[:cand], np.float64)
    rank = np.where(np.isnan(m), -np.inf, m)
    order = sorted(range(cand), key=lambda p: (np.isnan(m[p]), -rank[p], p))[:keep - recent]
    return sorted(order) + list(range(cand, n))
