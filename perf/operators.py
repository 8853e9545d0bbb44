"""The serving operators whose speed is measured: an 8-bit KV cache, the attention of a batch that
reads it, with and without a prompt prefix that the whole batch shares, and the verification of
drafted tokens.

With `own` false, run() computes them in their plain form, elementary torch operations in 32 bits;
with `own` true it calls the framework's operators.  Heads and vocabularies are those of
synthetic.WORKLOADS (GPT-2 small, a 1.1B and a 1.7B LLaMA-style model) and generic ones.
"""
import math

import torch

own = False


def listed():
    return [
        # one new token for each of 16 served requests: a decode step's cache write, and the smallest one
        {"name": "kv decode 16", "kind": "kv", "slots": 16, "n_tok": 16, "kv_heads": 4, "hd": 64, "ctx": 256, "heads": 32},
        # an ordinary prompt, ragged, of a model with as many KV heads as query heads
        {"name": "kv prompt 511", "kind": "kv", "slots": 2, "n_tok": 511, "kv_heads": 12, "hd": 64, "ctx": 1024,
         "heads": 12},
        # 16 prompts of 2047 tokens, each written behind a preamble of odd length: the largest write
        {"name": "kv prompts 16 x 2047", "kind": "kv", "slots": 16, "n_tok": 16 * 2047, "kv_heads": 8, "hd": 128,
         "ctx": 2112, "heads": 32},
        # one chat at an ordinary context, grouped-query heads
        {"name": "cached decode 1 x 700", "kind": "cached", "n_seq": 1, "n_q": 1, "heads": 32, "kv_heads": 4, "hd": 64,
         "max_len": 700},
        # 16 requests of a 1.7B model, each with its own context of up to 1024
        {"name": "cached decode 16 x 1024", "kind": "cached", "n_seq": 16, "n_q": 1, "heads": 32, "kv_heads": 32,
         "hd": 64, "max_len": 1024},
        # five tokens of 8 requests at once: four drafted ones and the token before them
        {"name": "cached drafts 8 x 5 x 999", "kind": "cached", "n_seq": 8, "n_q": 5, "heads": 12, "kv_heads": 12,
         "hd": 64, "max_len": 999},
        # 64 requests with contexts of up to 8192 and 128-wide heads: the largest read of a cache
        {"name": "cached decode 64 x 8192", "kind": "cached", "n_seq": 64, "n_q": 1, "heads": 32, "kv_heads": 8,
         "hd": 128, "max_len": 8192},
        # 16 chats that begin with one 512-token system prompt
        {"name": "shared 16 x 512 + 130", "kind": "shared", "n_seq": 16, "n_q": 1, "heads": 32, "kv_heads": 4, "hd": 64,
         "prefix": 512, "max_len": 130},
        # drafted tokens of 32 chats over a ragged shared document
        {"name": "shared drafts 32 x 4 x 2047 + 65", "kind": "shared", "n_seq": 32, "n_q": 4, "heads": 32,
         "kv_heads": 32, "hd": 64, "prefix": 2047, "max_len": 65},
        # 128 questions about one 8192-token document: the most arithmetic
        {"name": "shared 128 x 8192 + 256", "kind": "shared", "n_seq": 128, "n_q": 1, "heads": 32, "kv_heads": 8,
         "hd": 128, "prefix": 8192, "max_len": 256},
        # four drafted tokens of one chat
        {"name": "verify 1 x 4 x 32000", "kind": "verify", "n_seq": 1, "n_draft": 4, "vocab": 32000},
        # up to seven drafted tokens of each of 64 requests, ragged, over an odd vocabulary
        {"name": "verify 64 x 7 x 50257", "kind": "verify", "n_seq": 64, "n_draft": 7, "vocab": 50257},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _heads(rng):
    """Query heads, KV heads, head width."""
    return rng.choice([(12, 12, 64), (32, 4, 64), (32, 32, 64), (32, 8, 128), (16, 2, 128), (8, 8, 80), (10, 2, 96),
                       (6, 3, 32), (8, 1, 256), (15, 5, 64)])


def _most(kind):
    w = [work(c) for c in listed() if c["kind"] == kind]
    return max(x["bytes"] for x in w), max(x["flops"] for x in w)


def draw(rng):
    kind = rng.choice(["kv", "cached", "cached", "shared", "shared", "verify"])
    heads, kv, hd = _heads(rng)
    if kind == "kv":
        slots = _log(rng, 1, 40)
        per = rng.choice([1, 1, _log(rng, 2, 2500)])
        c = {"kind": kind, "slots": slots, "n_tok": slots * per, "kv_heads": kv, "hd": hd,
             "ctx": per + rng.randrange(17, 90), "heads": heads}
    elif kind == "verify":
        return {"kind": kind, "n_seq": _log(rng, 1, 64), "n_draft": rng.randrange(1, 8), "vocab": _log(rng, 1000, 50257)}
    else:
        c = {"kind": kind, "n_seq": _log(rng, 1, 128), "n_q": rng.choice([1, 1, 2, 4, 5, 8]), "heads": heads,
             "kv_heads": kv, "hd": hd, "max_len": _log(rng, 9, 8192 if kind == "cached" else 512)}
        if kind == "shared":
            c["prefix"] = _log(rng, 64, 8192)
    most = _most(kind)
    while work(c)["bytes"] > most[0] or work(c)["flops"] > most[1]:
        if kind == "kv":
            c["n_tok"] -= c["slots"] * max(1, c["n_tok"] // c["slots"] // 4)
        else:
            c["n_seq"] = max(1, c["n_seq"] * 3 // 4)
    return c


# ---- what a case holds ---------------------------------------------------------------------------
def _gen(seed, i=0):
    return torch.Generator(device="cuda").manual_seed(seed * 100003 + i * 7919 + 11)


def _lens(c):
    """Contexts from a quarter of max_len to all of it; every 16th request has not begun (no position of its
    own) where there is a prefix, and stops at its new tokens where there is none."""
    n, L = c["n_seq"], c["max_len"]
    out = [max(min(c["n_q"], L), L - (3 * L * ((7 * b) % n)) // (4 * n)) for b in range(n)]
    return [(0 if c["kind"] == "shared" and b % 16 == 15 else v) for b, v in enumerate(out)]


def _places(c):
    """Slot and position of every token of a cache write: a run for each slot, behind what it holds already."""
    per = c["n_tok"] // c["slots"]
    first = ((c["ctx"] - per) // 2) | 1
    slots = torch.arange(c["slots"], dtype=torch.int32).repeat_interleave(per)
    pos = torch.arange(per, dtype=torch.int32).repeat(c["slots"]) + first
    if c["n_tok"] % c["slots"]:                     # what is left over goes behind the last slot's run
        rest = c["n_tok"] % c["slots"]
        slots = torch.cat([slots, torch.full((rest,), c["slots"] - 1, dtype=torch.int32)])
        pos = torch.cat([pos, first + per + torch.arange(rest, dtype=torch.int32)])
    return slots, pos


def _rows(n, kv, hd, g, key):
    """Keys (a few channels several times larger than the rest) or values of n tokens."""
    x = torch.randn(n, kv, hd, device="cuda", generator=g)
    if key:
        x[:, :, ::29] *= 4.0
    return x


def _qkv(c, seed):
    """The rows of a fused projection: queries, keys and values of every token side by side."""
    g, n, kv, hd = _gen(seed), c["n_tok"], c["kv_heads"], c["hd"]
    f = torch.randn(n, (c["heads"] + 2 * kv) * hd, device="cuda", generator=g)
    k = f[:, c["heads"] * hd:(c["heads"] + kv) * hd].unflatten(1, (kv, hd))
    v = f[:, (c["heads"] + kv) * hd:].unflatten(1, (kv, hd))
    k[:, :, ::29] *= 4.0
    return k, v


def _encode(x):
    """Codes and scales of rows of head_dim values; decisions next to a border in 64 bits."""
    scale = (x.abs().amax(-1).double() / 127.0).float()
    safe = torch.where(scale > 0, scale, torch.ones_like(scale))
    return torch.round(x.double() / safe.double()[..., None]).clamp(-127, 127).to(torch.int8), scale


class _Cache:
    """The cache that both forms attend over: its slots filled with keys and values of their own."""

    def __init__(self, c, seed, slots, ctx):
        kv, hd = c["kv_heads"], c["hd"]
        self.kc = torch.zeros(slots, kv, ctx, hd, dtype=torch.int8, device="cuda")
        self.vc = torch.zeros_like(self.kc)
        self.ks = torch.zeros(slots, kv, ctx, device="cuda")
        self.vs = torch.zeros_like(self.ks)
        self.handle = None
        if own:
            from smallmind_amd.quantization import GpuKvCache
            self.handle = GpuKvCache(slots, kv, hd, ctx)

    def fill(self, slot, k, v):
        n = k.shape[0]
        for codes, scales, x in ((self.kc, self.ks, k), (self.vc, self.vs, v)):
            q, s = _encode(x)
            codes[slot, :, :n] = q.transpose(0, 1)
            scales[slot, :, :n] = s.transpose(0, 1)
        if own:
            p = torch.arange(n, dtype=torch.int32, device="cuda")
            self.handle.append(k, v, torch.full_like(p, slot), p)


def _fills(c, seed):
    """(slot, keys, values) of every slot that a case's attention reads; the prefix is the last slot."""
    for b in range(c["n_seq"]):
        g = _gen(seed, b + 1)
        yield b, _rows(c["max_len"], c["kv_heads"], c["hd"], g, True), _rows(c["max_len"], c["kv_heads"], c["hd"], g, False)
    if c["kind"] == "shared":
        g = _gen(seed, c["n_seq"] + 1)
        yield (c["n_seq"], _rows(c["prefix"], c["kv_heads"], c["hd"], g, True),
               _rows(c["prefix"], c["kv_heads"], c["hd"], g, False))


def _queries(c, seed):
    """The queries as they lie in the rows of a fused projection."""
    width = (c["heads"] + 2 * c["kv_heads"]) * c["hd"]
    f = torch.randn(c["n_seq"], c["n_q"], width, device="cuda", generator=_gen(seed)) * 1.5
    return f[:, :, :c["heads"] * c["hd"]].unflatten(2, (c["heads"], c["hd"]))


def _drafts(c, seed):
    """Target and draft probabilities, tokens drawn from the draft, and the random numbers."""
    g = _gen(seed)
    n, d, V = c["n_seq"], c["n_draft"], c["vocab"]
    logits = torch.randn(n, d + 1, V, device="cuda", generator=g) * 3.0
    target = torch.softmax(logits, -1)
    draft = logits[:, :d]
    draft = torch.softmax(draft + 0.5 * torch.randn(n, d, V, device="cuda", generator=g), -1)
    u = torch.rand(n, d, V, device="cuda", generator=g)
    tokens = (draft.log() - (-u.clamp(1e-10, 1 - 1e-7).log()).log()).argmax(-1).to(torch.int32)
    ua = torch.rand(n, d, device="cuda", generator=g)
    ud = torch.rand(n, device="cuda", generator=g)
    lens = torch.tensor([d - (b % 3 if d > 2 else 0) for b in range(n)], dtype=torch.int32, device="cuda")
    return target, draft, tokens, ua, ud, lens


def prepare(case, seed):
    c = case
    if c["kind"] == "kv":
        k, v = _qkv(c, seed)
        slots, pos = _places(c)
        return {"case": c, "k": k, "v": v, "slots": slots.cuda(), "pos": pos.cuda(),
                "cache": _Cache(c, seed, c["slots"], c["ctx"])}
    if c["kind"] == "verify":
        target, draft, tokens, ua, ud, lens = _drafts(c, seed)
        return {"case": c, "target": target, "draft": draft, "tokens": tokens, "ua": ua, "ud": ud, "lens": lens}
    shared = c["kind"] == "shared"
    cache = _Cache(c, seed, c["n_seq"] + shared, max(c["max_len"], c.get("prefix", 0)))
    for slot, k, v in _fills(c, seed):
        cache.fill(slot, k, v)
    return {"case": c, "q": _queries(c, seed), "cache": cache,
            "slots": torch.arange(c["n_seq"], dtype=torch.int32, device="cuda"),
            "lens": torch.tensor(_lens(c), dtype=torch.int32, device="cuda")}


# ---- one pass ------------------------------------------------------------------------------------
def run(state):
    c = state["case"]
    kind = c["kind"]
    if kind == "kv":
        # the tokens' rows written, and read back as a host that forks or checks a sequence does
        h = state["cache"]
        if own:
            h.handle.append(state["k"], state["v"], state["slots"], state["pos"])
            return h.handle.read(state["slots"], state["pos"])
        slots, pos = state["slots"].long(), state["pos"].long()
        return (_store(h.kc, h.ks, state["k"], slots, pos), _store(h.vc, h.vs, state["v"], slots, pos))
    if kind == "verify":
        if own:
            from smallmind_amd.quantization import verify_draft
            return verify_draft(state["target"], state["draft"], state["tokens"], state["ua"], state["ud"], state["lens"])
        return _verify(state["target"], state["draft"], state["tokens"], state["ua"], state["ud"], state["lens"])
    if own:
        from smallmind_amd.quantization import attention_cached, attention_shared
        h = state["cache"].handle
        if kind == "cached":
            return attention_cached(state["q"], h, state["slots"], state["lens"], c["max_len"])
        return attention_shared(state["q"], h, c["n_seq"], c["prefix"], state["slots"], state["lens"], c["max_len"])
    return _attend(c, state["q"], state["cache"], state["slots"].long(), state["lens"])


def _store(codes, scales, x, slots, pos):
    q, s = _encode(x)
    codes[slots, :, pos] = q
    scales[slots, :, pos] = s
    return codes[slots, :, pos].float() * scales[slots, :, pos][..., None]


def _attend(c, q, cache, slots, lens):
    n, m, H, hd = q.shape
    kv, L = c["kv_heads"], c["max_len"]
    G = H // kv
    qt = (q.reshape(n, m, kv, G, hd) * (1.0 / math.sqrt(hd))).permute(0, 2, 4, 1, 3).reshape(n, kv, hd, m * G)
    k = cache.kc[slots, :, :L].float() * cache.ks[slots, :, :L, None]
    v = cache.vc[slots, :, :L].float() * cache.vs[slots, :, :L, None]
    s = torch.matmul(k, qt)                                             # [n][kv][L][m * G]
    seen = torch.arange(L, device=q.device)[None, :, None] < (lens[:, None] - m + 1 + torch.arange(m, device=q.device))[:, None, :]
    s = s.masked_fill(~seen.repeat_interleave(G, 2)[:, None], -math.inf)
    top = s.amax(2, keepdim=True)
    if c["kind"] == "shared":
        P = c["prefix"]
        kp = cache.kc[c["n_seq"], :, :P].float() * cache.ks[c["n_seq"], :, :P, None]
        vp = cache.vc[c["n_seq"], :, :P].float() * cache.vs[c["n_seq"], :, :P, None]
        qp = qt.permute(1, 2, 0, 3).reshape(kv, hd, n * m * G)
        sp = torch.matmul(kp, qp)                                       # [kv][P][n * m * G]: once for all
        tp = sp.amax(1).reshape(kv, n, m * G).transpose(0, 1)[:, :, None]
        top = torch.maximum(top, tp)
    safe = torch.where(top == -math.inf, torch.zeros_like(top), top)
    e = torch.exp(s - safe)
    num = torch.matmul(e.transpose(2, 3).contiguous(), v)               # [n][kv][m * G][hd]
    den = e.sum(2)
    if c["kind"] == "shared":
        ep = torch.exp(sp - safe.transpose(0, 1).reshape(kv, 1, n * m * G))
        num = num + torch.matmul(ep.transpose(1, 2).contiguous(), vp).reshape(kv, n, m * G, hd).transpose(0, 1)
        den = den + ep.sum(1).reshape(kv, n, m * G).transpose(0, 1)
    o = torch.where(den[..., None] > 0, num / den[..., None], torch.zeros_like(num))
    return o.reshape(n, kv, m, G, hd).permute(0, 2, 1, 3, 4).reshape(n, m, H, hd)


def _verify(target, draft, tokens, ua, ud, lens):
    n, d, V = draft.shape
    at = tokens.long()[..., None]
    p, q = target[:, :d].gather(2, at)[..., 0].double(), draft.gather(2, at)[..., 0].double()
    ok = (ua.double() * q < p) & (torch.arange(d, device=lens.device)[None] < lens[:, None])
    acc = ok.to(torch.int32).cumprod(1).sum(1)                          # drafts taken, up to the first refusal
    row = torch.arange(n, device=lens.device)
    w = target[row, acc].double()
    drafted = (acc < lens)[:, None]
    w = torch.where(drafted, w - draft[row, acc.clamp(max=d - 1)].double(), w).clamp(min=0)
    cum = w.cumsum(1)
    drawn = (cum <= (ud.double() * cum[:, -1])[:, None]).sum(1)
    cols = torch.arange(d + 1, device=lens.device)[None]
    out = torch.cat([tokens, tokens[:, :1]], 1).long()
    out = torch.where(cols < acc[:, None], out, torch.where(cols == acc[:, None], drawn[:, None], -1))
    return out.to(torch.int32), acc.to(torch.int32)


# ---- what a pass cannot do without ---------------------------------------------------------------
def work(case):
    c = case
    if c["kind"] == "kv":
        rows = 2 * c["n_tok"] * c["kv_heads"]
        # read 4 bytes, kept in one and read from it, given back in 4; a scale for each row
        return {"bytes": rows * (10 * c["hd"] + 8) + 16 * c["n_tok"], "flops": 6 * rows * c["hd"]}
    if c["kind"] == "verify":
        return {"bytes": 8 * c["n_seq"] * c["vocab"], "flops": 3 * c["n_seq"] * c["vocab"]}
    rows, hd = c["n_seq"] * c["n_q"] * c["heads"], c["hd"]
    own_pos, P = sum(_lens(c)), c.get("prefix", 0)
    seen = sum(max(0, n - c["n_q"] + 1 + i) for n in _lens(c) for i in range(c["n_q"]))
    return {"bytes": 2 * c["kv_heads"] * (hd + 4) * (own_pos + P) + 8 * rows * hd,
            "flops": 4 * hd * (c["heads"] * seen + rows * P)}


# ---- the same in 64 bits -------------------------------------------------------------------------
def _held(x):
    """What the cache stands for: each row's values rounded to whole multiples of its scale."""
    x = x.double()
    step = (x.abs().max(dim=-1, keepdim=True).values / 127).to(torch.float32).double()
    n = torch.where(step > 0, x / torch.where(step > 0, step, 1.0), 0.0)
    return torch.clamp(torch.round(n), -127.0, 127.0) * step


def exact(case, seed):
    c = case
    if c["kind"] == "kv":
        k, v = _qkv(c, seed)
        return _held(k), _held(v)
    if c["kind"] == "verify":
        target, draft, tokens, ua, ud, lens = _drafts(c, seed)
        toks, taken = [], []
        for b in range(c["n_seq"]):
            i, n = 0, int(lens[b])
            while i < n:
                x = int(tokens[b, i])
                if not float(ua[b, i]) * float(draft[b, i, x]) < float(target[b, i, x]):
                    break
                i += 1
            p = target[b, i].double()
            if i < n:
                p = torch.clamp(p - draft[b, i].double(), min=0.0)
            run_ = torch.cumsum(p, 0)
            t = int(torch.nonzero(run_ > float(ud[b]) * float(run_[-1]))[0])
            toks.append(tokens[b, :i].tolist() + [t] + [-1] * (c["n_draft"] - i))
            taken.append(i)
        return (torch.tensor(toks, dtype=torch.int32, device="cuda"), torch.tensor(taken, dtype=torch.int32, device="cuda"))
    q, lens = _queries(c, seed).double(), _lens(c)
    fills = _fills(c, seed)
    pre = None
    if c["kind"] == "shared":
        g = _gen(seed, c["n_seq"] + 1)
        pre = [_held(_rows(c["prefix"], c["kv_heads"], c["hd"], g, key)).transpose(0, 1) for key in (True, False)]
    out, G = torch.zeros_like(q), c["heads"] // c["kv_heads"]
    for b in range(c["n_seq"]):
        _, k, v = next(fills)
        for i in range(c["n_q"]):
            n = max(0, lens[b] - c["n_q"] + 1 + i)
            kk, vv = _held(k[:n]).transpose(0, 1), _held(v[:n]).transpose(0, 1)
            if pre is not None:
                kk, vv = torch.cat([pre[0], kk], 1), torch.cat([pre[1], vv], 1)
            if kk.shape[1] == 0:
                continue
            qb = q[b, i].reshape(c["kv_heads"], G, c["hd"])
            s = torch.matmul(qb, kk.transpose(1, 2).contiguous()) / math.sqrt(c["hd"])
            out[b, i] = torch.matmul(torch.softmax(s, 2), vv).reshape(c["heads"], c["hd"])
    return out
