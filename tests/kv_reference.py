"""Plain 64-bit forms of the serving operators: the 8-bit cache's rows, attention over them, and the
verification of drafted tokens."""
from __future__ import annotations

import math

import numpy as np


def encode(x: np.ndarray):
    """(codes, scales) of rows of the last axis: scale = fl32(max|x| / 127), codes the nearest integers to
    x / scale (ties to even, at most 127 in size).  Quotients of 24-bit numbers in 64 bits never round onto a
    border that they do not lie on.  A row with a NaN or an infinity has the scale NaN and zero codes."""
    x = np.asarray(x, np.float32).astype(np.float64)
    with np.errstate(all="ignore"):
        bad = ~np.isfinite(x).all(-1)
        scale = (np.abs(x).max(-1) / 127.0).astype(np.float32)
        scale = np.where(bad, np.float32(np.nan), scale)
        s = scale.astype(np.float64)[..., None]
        n = np.where(s > 0, x / np.where(s > 0, s, 1.0), 0.0)
        codes = np.clip(np.rint(np.where(np.isfinite(n), n, 0.0)), -127, 127)
    return codes.astype(np.int8), scale


def held(x: np.ndarray) -> np.ndarray:
    """What the cache gives back for rows x: codes times scale, rounded once to fp32."""
    c, s = encode(x)
    with np.errstate(invalid="ignore"):
        return c.astype(np.float32) * s[..., None]


def attention(q, k, v, visible):
    """q [rows][hd], k and v [n][hd] (the values held), visible [rows][n] bool -> (out, bound) in 64 bits.

    bound: how far a row may be off.  With w the weights, out = sum w v / sum w moves by at most 2 e max|v| when
    every weight moves by e relative to itself.  e is made of: q in two fp16 parts (2^-22 of the row's
    largest, on |q| |k| summed over hd elements), the fp32 sums over hd elements (hd + 4 roundings of 2^-24 on
    the same), the exponent's rounding (2^-23 of its size), the weight's two parts and the exponential
    (2^-21 together), and the fp32 sums over the positions (a rounding for each, 2^-24)."""
    q, k, v = (np.asarray(a, np.float64) for a in (q, k, v))
    rows, hd = q.shape
    out = np.zeros((rows, hd))
    bound = np.zeros(rows)
    for r in range(rows):
        vis = visible[r]
        if not vis.any():
            continue
        kk, vv = k[vis], v[vis]
        s = kk @ q[r] / math.sqrt(hd)
        w = np.exp(s - s.max())
        out[r] = w @ vv / w.sum()
        mass = (np.abs(kk) @ np.abs(q[r])).max() / math.sqrt(hd)
        reach = np.abs(kk).sum(1).max() * np.abs(q[r]).max() / math.sqrt(hd)
        e = reach * 2.0 ** -22 + mass * (hd + 4) * 2.0 ** -24 + np.abs(s).max() * 2.0 ** -22 + 2.0 ** -21
        bound[r] = 2 * (e + (len(vv) + 64) * 2.0 ** -24) * np.abs(vv).max()
    return out, bound


def verify(target, draft, tokens, u_accept, u_draw, lens, vocab):
    """(out [n_seq][n_draft + 1], accepted [n_seq]) of smx_verify_draft, in 64 bits."""
    n_seq, n_draft = u_accept.shape
    out = np.full((n_seq, n_draft + 1), -1, np.int64)
    acc = np.zeros(n_seq, np.int64)
    for b in range(n_seq):
        n = n_draft if lens is None else min(int(lens[b]), n_draft)
        if n < 0:
            continue
        i = 0
        while i < n:
            t = int(tokens[b, i])
            if not 0 <= t < vocab:
                break
            qt = 1.0 if draft is None else float(draft[b, i, t])
            if not float(u_accept[b, i]) * qt < float(target[b, i, t]):
                break
            out[b, i] = t
            i += 1
        p = target[b, i, :vocab].astype(np.float64)
        choices = [p]
        if i < n:
            if draft is not None:
                choices.insert(0, p - draft[b, i, :vocab].astype(np.float64))
            else:
                r = p.copy()
                if 0 <= int(tokens[b, i]) < vocab:
                    r[int(tokens[b, i])] -= 1.0
                choices.insert(0, r)
        for w in choices:
            w = np.where(w > 0, w, 0.0)    # NaN: nothing
            if w.sum() > 0:
                c = np.cumsum(w)
                hit = np.nonzero((c > float(u_draw[b]) * c[-1]) & (w > 0))[0]
                out[b, i] = hit[0] if hit.size else np.nonzero(w > 0)[0][-1]
                break
        acc[b] = i
    return out, acc


def attention_by_terms(q, k, v, visible):
    """attention() with a bound for every element that goes by the row's own weighted terms p_j v_j, not by the
    largest v: (out, bound), each [rows][hd], in 64 bits.

    With p_j the weights relative to the largest (p <= 1), A = sum p |v| per element and S = sum p:
      scores    q in two fp16 parts is off by 2^-22 of each element and 2^-38 of the row's largest; the 2 hd products
                are added in fp32 (a rounding of 2^-24 of the sum of sizes for each, 2^-24 each for the scale of K and for
                K's held value); the exponent's difference and product are 3 roundings of |score| and of the largest
                one.  Weight j moves by that e_j relative to itself, and by 2^-22 for the exponential and the rounding
                of p times V's scale; numerator and S both move.
      weights   two fp16 parts: 2^-22 of each, and 2^-38 of the largest p_j max|v_j|, for each position.
      sums      the two parts' products (2 n), S (n) and the joins of waves and parts, 2^-24 of A or S each."""
    q, k, v = (np.asarray(a, np.float64) for a in (q, k, v))
    rows, hd = q.shape
    out, bound = np.zeros((rows, v.shape[1])), np.zeros((rows, v.shape[1]))
    for r in range(rows):
        vis = visible[r]
        n = int(vis.sum())
        if not n:
            continue
        kk, vv = k[vis], v[vis]
        s = kk @ q[r] / math.sqrt(hd)
        p = np.exp(s - s.max())
        S, A = p.sum(), p @ np.abs(vv)
        out[r] = p @ vv / S
        mass = (np.abs(kk) @ np.abs(q[r])) / math.sqrt(hd)
        reach = np.abs(kk).sum(1) * np.abs(q[r]).max() / math.sqrt(hd)
        e = mass * (2.0 ** -22 + (2 * hd + 2) * 2.0 ** -24) + reach * 2.0 ** -38 + 3 * (np.abs(s) + abs(s.max())) * 2.0 ** -24
        e += 2.0 ** -22
        most = (p * np.abs(vv).max(1)).max()
        bound[r] = ((p * e) @ np.abs(vv) + A * ((p @ e) / S + 2.0 ** -22 + (3 * n + 16) * 2.0 ** -24) + n * 2.0 ** -38 * most) / S
    return out, bound
