"""The operators of a paged KV cache whose speed is measured: the write of a batch's tokens with the norms of
queries and keys and the rotation by position (one axis or several), the attention of ragged batches of
prompt chunks and single tokens over the pages, the attention weight that every position has received, and the eviction
of the positions that received least.

With `own` false, run() computes them in their plain form, elementary torch operations in 32 bits;
with `own` true it calls the framework's operators.  Heads are those of synthetic.WORKLOADS (GPT-2 small, a 1.1B
and a 1.7B LLaMA-style model) and generic ones.
"""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
EPS = 1e-6


def listed():
    return [
        # a decode step's write for 16 served requests, fp32 rows of a fused projection: the smallest write
        {"name": "write decode 16", "kind": "write", "n_tok": 16, "n_seq": 16, "heads": 32, "kv_heads": 4, "hd": 64, "page": 64,
         "type": "f16", "io": "f32", "norm": True, "axes": 1, "halves": False},
        # a prompt of images and text, positions of three axes, norms of queries and keys: the largest write
        {"name": "write images 16383", "kind": "write", "n_tok": 16383, "n_seq": 3, "heads": 32, "kv_heads": 8, "hd": 128, "page": 64,
         "type": "bf16", "io": "bf16", "norm": True, "axes": 3, "halves": True},
        # one chat at an ordinary context, fp32 on both sides of the attention: a call of the smallest latency
        {"name": "decode 1 x 700", "kind": "attend", "n_seq": 1, "n_long": 0, "max_q": 1, "heads": 32, "kv_heads": 4, "hd": 64, "page": 16,
         "type": "f16", "io": "f32", "max_len": 700, "cap": 0.0, "slopes": False, "window": 0, "prefix": 0},
        # 64 requests with contexts of up to 8192: the largest read of the pages
        {"name": "decode 64 x 8192", "kind": "attend", "n_seq": 64, "n_long": 0, "max_q": 1, "heads": 32, "kv_heads": 8, "hd": 128,
         "page": 64, "type": "bf16", "io": "bf16", "max_len": 8192, "cap": 0.0, "slopes": False, "window": 0, "prefix": 0},
        # a prompt chunk of 512 tokens of a 1.1B model, fp32 on both sides
        {"name": "chunk 512 over 4096", "kind": "attend", "n_seq": 1, "n_long": 1, "max_q": 512, "heads": 32, "kv_heads": 4, "hd": 64,
         "page": 64, "type": "f16", "io": "f32", "max_len": 4096, "cap": 0.0, "slopes": False, "window": 0, "prefix": 0},
        # a prompt chunk of a long document: the most arithmetic
        {"name": "chunk 2048 over 32768", "kind": "attend", "n_seq": 1, "n_long": 1, "max_q": 2048, "heads": 32, "kv_heads": 8, "hd": 128,
         "page": 64, "type": "bf16", "io": "bf16", "max_len": 32768, "cap": 0.0, "slopes": False, "window": 0, "prefix": 0},
        # a continuous batch: two prompt chunks among 30 decodes, capped scores, a sliding window with its first positions kept
        {"name": "mixed 2 x 509 + 30, window", "kind": "attend", "n_seq": 32, "n_long": 2, "max_q": 509, "heads": 16, "kv_heads": 2,
         "hd": 128, "page": 32, "type": "bf16", "io": "bf16", "max_len": 4099, "cap": 50.0, "slopes": False, "window": 1024, "prefix": 16},
        # whole prompts with a bias by distance, whose first 300 positions see one another
        {"name": "prompts 4 x 1023, slopes", "kind": "attend", "n_seq": 4, "n_long": 4, "max_q": 1023, "heads": 12, "kv_heads": 12,
         "hd": 64, "page": 16, "type": "f16", "io": "f16", "max_len": 1023, "cap": 0.0, "slopes": True, "window": 0, "prefix": 300},
        # the weight that a decode step of 16 requests gives to every position
        {"name": "mass decode 16 x 1024", "kind": "mass", "n_seq": 16, "n_long": 0, "max_q": 1, "heads": 32, "kv_heads": 32, "hd": 64,
         "page": 64, "type": "f16", "io": "f32", "max_len": 1024, "cap": 0.0, "slopes": False, "window": 0, "prefix": 0},
        # the same of a whole prompt
        {"name": "mass prompt 4095", "kind": "mass", "n_seq": 1, "n_long": 1, "max_q": 4095, "heads": 32, "kv_heads": 8, "hd": 128, "page": 64,
         "type": "bf16", "io": "bf16", "max_len": 4095, "cap": 0.0, "slopes": False, "window": 0, "prefix": 0},
        # one chat's cache shortened
        {"name": "evict 1 x 700 to 256", "kind": "evict", "n_seq": 1, "heads": 32, "kv_heads": 4, "hd": 64, "page": 16, "type": "f16",
         "max_len": 700, "keep": 256, "recent": 64},
        # the caches of 16 long requests brought to a quarter
        {"name": "evict 16 x 8192 to 2048", "kind": "evict", "n_seq": 16, "heads": 32, "kv_heads": 8, "hd": 128, "page": 64, "type": "bf16",
         "max_len": 8192, "keep": 2048, "recent": 256},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _most(kind):
    w = [work(c) for c in listed() if c["kind"] == kind]
    return max(x["bytes"] for x in w), max(x["flops"] for x in w)


def draw(rng):
    kind = rng.choice(["write", "attend", "attend", "attend", "mass", "evict"])
    heads, kv, hd = rng.choice([(12, 12, 64), (32, 4, 64), (32, 32, 64), (32, 8, 128), (16, 2, 128), (8, 8, 80), (10, 2, 96),
                                (6, 3, 32), (8, 1, 256), (15, 5, 64)])
    t, page = rng.choice(["f16", "bf16"]), rng.choice([16, 32, 64, 128])
    io = rng.choice(["f32", t])
    if kind == "write":
        c = {"kind": kind, "n_tok": _log(rng, 1, 16383), "n_seq": _log(rng, 1, 32), "heads": heads, "kv_heads": kv, "hd": hd, "page": page,
             "type": t, "io": io, "norm": rng.random() < 0.7, "axes": rng.choice([1, 1, 3]), "halves": rng.random() < 0.6}
        c["n_seq"] = min(c["n_seq"], c["n_tok"])
    elif kind == "evict":
        c = {"kind": kind, "n_seq": _log(rng, 1, 32), "heads": heads, "kv_heads": kv, "hd": hd, "page": page, "type": t,
             "max_len": _log(rng, 64, 16384)}
        c["keep"] = max(8, int(c["max_len"] * rng.uniform(0.1, 0.8)))
        c["recent"] = int(c["keep"] * rng.uniform(0.0, 0.6))
    else:
        n_seq = _log(rng, 1, 64)
        long = rng.choice([0, 0, 1, min(n_seq, 4), n_seq])
        c = {"kind": kind, "n_seq": n_seq, "n_long": long, "max_q": _log(rng, 2, 2048) if long else 1, "heads": heads, "kv_heads": kv,
             "hd": hd, "page": page, "type": t, "io": io, "max_len": _log(rng, 20, 32768), "cap": rng.choice([0.0, 0.0, 30.0]),
             "slopes": rng.random() < 0.3, "window": rng.choice([0, 0, _log(rng, 16, 4096)]), "prefix": rng.choice([0, 0, _log(rng, 4, 512)])}
        c["max_len"] = max(c["max_len"], c["max_q"])
    most = _most(kind)
    size = "n_tok" if kind == "write" else "max_len"
    while work(c)["bytes"] > most[0] or work(c)["flops"] > most[1] or _padded(c) > 2 ** 31:
        if c["n_seq"] > 1:
            c["n_seq"] = c["n_seq"] * 3 // 4
            c["n_long"] = min(c.get("n_long", 0), c["n_seq"])
        else:
            c[size] = c[size] * 3 // 4
        if kind in ("attend", "mass"):
            c["max_q"] = min(c["max_q"], c["max_len"])
        if kind == "evict":
            c["keep"] = min(c["keep"], c["max_len"])
            c["recent"] = min(c["recent"], c["keep"])
    if kind in ("write", "evict"):
        c.pop("n_long", None)
    return c


def _padded(c):
    """Scores of a batch whose sequences are all as long as the longest, as the plain form has them."""
    return c["n_seq"] * c["heads"] * c["max_q"] * c["max_len"] if "max_q" in c else 0


# ---- what a case holds ---------------------------------------------------------------------------
def _gen(seed, i=0):
    return torch.Generator(device="cuda").manual_seed(seed * 100003 + i * 7919 + 11)


def _new(c):
    """New tokens of each sequence: ragged chunks first, then single tokens."""
    return [max(1, c["max_q"] - (37 * b) % (c["max_q"] // 4 + 1)) if b < c["n_long"] else 1 for b in range(c["n_seq"])]


def _lens(c):
    """Positions of each sequence, its new tokens among them: from a quarter of max_len to all of it."""
    n, L = c["n_seq"], c["max_len"]
    new = _new(c) if "max_q" in c else [1] * n
    return [max(m, L - (3 * L * ((7 * b) % n)) // (4 * n)) for b, m in enumerate(new)]


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _tables(lens, page, g):
    """Page tables of sequences of these lengths in a shuffled pool with some spare pages: ([n_seq][pages], pages of the
    pool); places a sequence does not need are -1."""
    per = [-(-n // page) for n in lens]
    pool = sum(per) + 7
    order = torch.randperm(pool, device="cuda", generator=g).to(torch.int32)
    at, need = torch.arange(max(per), device="cuda"), torch.tensor(per, device="cuda")
    first = need.cumsum(0) - need
    t = order[(first[:, None] + at).clamp(max=pool - 1)]
    return torch.where(at < need[:, None], t, -1).to(torch.int32).contiguous(), pool


def _places(tables, seqs, pos, page):
    """Where positions `pos` of sequences `seqs` lie: page times page size, plus the place within."""
    return (tables[seqs, pos // page] * page + pos % page).to(torch.int32)


def _of_tokens(lens):
    """Sequence and position of every token of sequences of these lengths, one after another."""
    n = torch.tensor(lens, device="cuda")
    seqs = torch.arange(len(lens), device="cuda").repeat_interleave(n)
    return seqs, torch.arange(sum(lens), device="cuda") - (n.cumsum(0) - n)[seqs]


class _Pages:
    """The cache that both forms work on."""

    def __init__(self, c, pool):
        if own:
            from smallmind_amd.quantization import GpuPagedCache
            self.handle = GpuPagedCache(TYPES[c["type"]], pool, c["kv_heads"], c["hd"], c["page"])
        else:
            self.k = torch.zeros(pool * c["page"], c["kv_heads"], c["hd"], dtype=TYPES[c["type"]], device="cuda")
            self.v = torch.zeros_like(self.k)

    def fill(self, k, v, places):
        if own:
            self.handle.append(k, v, places)
        else:
            self.k[places.long()] = k
            self.v[places.long()] = v


def _rows(c, n, g, key):
    """Keys (a few channels larger than the rest) or values of n tokens."""
    x = torch.randn(n, c["kv_heads"], c["hd"], device="cuda", generator=g)
    if key:
        x[:, :, ::29] *= 3.0
    return x.to(TYPES[c["type"]])


def _cached(c, seed):
    """Keys, values and places of everything that the pages hold, the tables and the pool's size."""
    g, lens = _gen(seed, 1), _lens(c)
    tables, pool = _tables(lens, c["page"], g)
    seqs, pos = _of_tokens(lens)
    return _rows(c, len(seqs), g, True), _rows(c, len(seqs), g, False), _places(tables, seqs, pos, c["page"]), tables, pool


def _queries(c, seed):
    """The queries as they lie in the rows of a fused projection."""
    n, H, hd = sum(_new(c)), c["heads"], c["hd"]
    f = torch.randn(n, (H + 2 * c["kv_heads"]) * hd, device="cuda", generator=_gen(seed)) * 1.5
    return f.to(TYPES[c["io"]])[:, :H * hd].unflatten(1, (H, hd))


def _starts(c):
    n = torch.tensor(_new(c))
    return torch.cat([torch.zeros(1, dtype=torch.int64), n.cumsum(0)]).to(torch.int32).cuda()


def _slopes(c):
    """Slopes of a geometric series over the heads."""
    return torch.exp2(-8.0 * (torch.arange(c["heads"], device="cuda") + 1) / c["heads"]).float() if c["slopes"] else None


def _prefix(c):
    return _ints([c["prefix"]] * c["n_seq"]) if c["prefix"] else None


def _angles(c):
    """Tables of cosines and sines, and the pairs that turn by each axis (two thirds of the heights and widths)."""
    half = c["hd"] // 2
    a = torch.arange(32768, dtype=torch.float64, device="cuda")[:, None] * 10000.0 ** (-torch.arange(half, device="cuda").double() / half)
    sections = [half] if c["axes"] == 1 else [half - 2 * (half * 3 // 8), half * 3 // 8, half * 3 // 8]
    return a.cos().float(), a.sin().float(), sections


def _positions(c, seed):
    """Positions of a write's tokens on each axis, and their places in the cache: each sequence behind what it holds."""
    n = [c["n_tok"] // c["n_seq"] + (b < c["n_tok"] % c["n_seq"]) for b in range(c["n_seq"])]
    before = [(97 * b) % 211 + 1 for b in range(c["n_seq"])]
    g = _gen(seed, 2)
    tables, pool = _tables([a + m for a, m in zip(before, n)], c["page"], g)
    seqs, pos = _of_tokens(n)
    pos = pos + torch.tensor(before, device="cuda")[seqs]
    places = _places(tables, seqs, pos, c["page"])
    p = pos[None]
    if c["axes"] == 3:      # 28 x 36 patches an image: one time, rows, columns
        p = torch.stack([pos // 1008 * 36, pos // 1008 * 36 + pos % 1008 // 36, pos // 1008 * 36 + pos % 36])
    return p.to(torch.int32).contiguous(), places, pool


def _projected(c, seed):
    """Queries, keys and values of every token side by side, and the weights of the norms."""
    g, H, kv, hd = _gen(seed), c["heads"], c["kv_heads"], c["hd"]
    f = (torch.randn(c["n_tok"], (H + 2 * kv) * hd, device="cuda", generator=g) * 2.0).to(TYPES[c["io"]])
    q, k, v = f.split([H * hd, kv * hd, kv * hd], 1)
    gq, gk = (1.0 + 0.2 * torch.randn(hd, device="cuda", generator=g) for _ in range(2))
    return q.unflatten(1, (H, hd)), k.unflatten(1, (kv, hd)), v.unflatten(1, (kv, hd)), gq if c["norm"] else None, gk if c["norm"] else None


def _received(c, seed, width):
    """Weight that positions have received: most little, a few much, the same for some."""
    x = torch.exp(2.5 * torch.randn(c["n_seq"], c["kv_heads"], width, device="cuda", generator=_gen(seed, 3)) - 3.0)
    return torch.where(x < 0.005, 0.0, x)


def prepare(case, seed):
    c = case
    if c["kind"] == "write":
        q, k, v, gq, gk = _projected(c, seed)
        pos, places, pool = _positions(c, seed)
        cos, sin, sections = _angles(c)
        s = {"case": c, "q": q, "k": k, "v": v, "gq": gq, "gk": gk, "pos": pos, "places": places, "cos": cos, "sin": sin,
             "axis": torch.arange(c["axes"], device="cuda").repeat_interleave(torch.tensor(sections, device="cuda")), "pages": _Pages(c, pool)}
        if own:
            from smallmind_amd.quantization import Rotation
            s["rotation"] = Rotation(cos, sin, sections=sections, halves=c["halves"])
        return s
    k, v, places, tables, pool = _cached(c, seed)
    lens = _lens(c)
    if c["kind"] == "evict":
        new, more = _tables([min(n, c["keep"]) for n in lens], c["page"], _gen(seed, 4))
        pages = _Pages(c, pool + more)
        pages.fill(k, v, places)
        new = torch.where(new >= 0, new + pool, -1).to(torch.int32)
        seqs, pos = _of_tokens([min(n, c["keep"]) for n in lens])
        return {"case": c, "pages": pages, "tables": tables, "new": new, "lens": _ints(lens), "mass": _received(c, seed, c["max_len"]),
                "read": _places(new, seqs, pos, c["page"]), "at": (seqs, pos)}
    pages = _Pages(c, pool)
    pages.fill(k, v, places)
    s = {"case": c, "pages": pages, "tables": tables, "lens": _ints(lens), "q": _queries(c, seed), "starts": _starts(c),
         "slopes": _slopes(c), "prefix": _prefix(c)}
    if c["kind"] == "mass":
        s["lse"] = _sums(c, seed)
        s["mass"] = _received(c, seed, c["max_len"])
    return s


# ---- one pass ------------------------------------------------------------------------------------
def run(state):
    s, c = state, state["case"]
    kind, pages = c["kind"], state["pages"]
    if kind == "write":
        # the tokens' rows written, and read back as a host that forks or checks a sequence does
        if own:
            q = pages.handle.append(s["k"], s["v"], s["places"], q=s["q"], q_gamma=s["gq"], k_gamma=s["gk"], eps=EPS,
                                    rotation=s["rotation"], pos=s["pos"])
            return (q, *pages.handle.read(s["places"]))
        at = s["places"].long()
        pages.k[at] = _turned(s, s["k"], s["gk"]).to(pages.k.dtype)
        pages.v[at] = s["v"].to(pages.v.dtype)
        return _turned(s, s["q"], s["gq"]).to(s["q"].dtype), pages.k[at], pages.v[at]
    if kind == "evict":
        if own:
            kept, lens, mass = pages.handle.evict(s["mass"], s["lens"], c["keep"], c["recent"], s["tables"], s["new"])
            return (kept, lens, mass, *pages.handle.read(s["read"]))
        return _evict(s)
    if own:
        from smallmind_amd.quantization import attention_mass, attention_paged
        rules = {"cap": c["cap"], "slopes": s["slopes"], "window": c["window"], "prefix": s["prefix"]}
        if kind == "mass":
            return attention_mass(s["q"], s["lse"], pages.handle, s["starts"], s["lens"], s["tables"], c["max_q"], c["max_len"],
                                  mass=s["mass"], **rules)
        return attention_paged(s["q"], pages.handle, s["starts"], s["lens"], s["tables"], c["max_q"], c["max_len"], **rules)
    score, seen, seq, i = _scores(s)
    if kind == "mass":
        lse = s["lse"].float().unflatten(1, (c["kv_heads"], -1))                       # [tokens][kv][G]
        lse = _by_sequence(s, lse, seq, i).permute(0, 2, 1, 3).flatten(2)              # [n][kv][rows]
        e = torch.exp(score.sub_(lse[..., None])).masked_fill_(~seen, 0.0)
        beyond = torch.arange(c["max_len"], device="cuda") >= s["lens"][:, None]
        return (s["mass"] + e.sum(2)).masked_fill(beyond[:, None], 0.0)
    score.masked_fill_(~seen, -math.inf)
    top = score.amax(3, keepdim=True)
    e = score.sub_(torch.where(top == -math.inf, torch.zeros_like(top), top)).exp_()
    num, den = torch.matmul(e, _gathered(s, pages.v)), e.sum(3, keepdim=True)
    o = torch.where(den > 0, num / den, torch.zeros_like(num))                         # [n][kv][rows][hd]
    o = o.unflatten(2, (c["max_q"], -1)).permute(0, 2, 1, 3, 4).flatten(2, 3)          # [n][max_q][H][hd]
    return o[seq, i].to(s["q"].dtype)


def _turned(s, x, gamma):
    """Rows normed and turned, in 32 bits."""
    c, y = s["case"], x.float()
    if gamma is not None:
        y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + EPS) * gamma
    at, pair = s["pos"].long()[s["axis"]].t(), torch.arange(c["hd"] // 2, device="cuda")
    cos, sin = s["cos"][at, pair][:, None], s["sin"][at, pair][:, None]                # [tokens][1][pairs]
    a, b = (y[..., :c["hd"] // 2], y[..., c["hd"] // 2:]) if c["halves"] else (y[..., 0::2], y[..., 1::2])
    both = (a * cos - b * sin, a * sin + b * cos)
    return torch.cat(both, -1) if c["halves"] else torch.stack(both, -1).flatten(-2)


def _gathered(s, x):
    """Keys or values of every sequence up to max_len: [n][kv][max_len][hd], 0 where there is no page."""
    c, t = s["case"], s["tables"]
    at = (t.clamp(min=0).long()[..., None] * c["page"] + torch.arange(c["page"], device="cuda")).flatten(1)[:, :c["max_len"]]
    there = (t >= 0).repeat_interleave(c["page"], 1)[:, :c["max_len"], None, None]
    return torch.where(there, x[at].float(), 0.0).transpose(1, 2).contiguous()


def _by_sequence(s, x, seq, i):
    """x [tokens]... as [n][max_q]..., 0 where a sequence has fewer."""
    o = torch.zeros(s["case"]["n_seq"], s["case"]["max_q"], *x.shape[1:], device="cuda")
    o[seq, i] = x
    return o


def _scores(s):
    """(scores [n][kv][max_q * G][max_len], which of them are seen, sequence and place of every token)."""
    c = s["case"]
    n, m, kv, hd, L = c["n_seq"], c["max_q"], c["kv_heads"], c["hd"], c["max_len"]
    G = c["heads"] // kv
    tok, starts = torch.arange(s["q"].shape[0], device="cuda", dtype=torch.int32), s["starts"]
    seq = torch.searchsorted(starts, tok, right=True) - 1
    i = (tok - starts[seq]).long()
    q = _by_sequence(s, s["q"].float() * (1.0 / math.sqrt(hd)), seq, i)
    q = q.reshape(n, m, kv, G, hd).permute(0, 2, 1, 3, 4).reshape(n, kv, m * G, hd)
    x = torch.matmul(q, _gathered(s, s["pages"].k).transpose(2, 3).contiguous())
    if c["cap"]:
        x = x.div_(c["cap"]).tanh_().mul_(c["cap"])
    new = starts[1:] - starts[:-1]
    t = (s["lens"] - new)[:, None] + torch.arange(m, device="cuda", dtype=torch.int32)  # positions of the tokens
    p = torch.arange(L, device="cuda", dtype=torch.int32)
    away = t[:, :, None] - p                                                           # [n][m][L]
    seen = (away >= 0) & (away < (c["window"] or 1 << 30))
    if c["prefix"]:
        seen |= p < s["prefix"][:, None, None]
    seen &= (p < s["lens"][:, None])[:, None] & (torch.arange(m, device="cuda") < new[:, None])[..., None]
    if c["slopes"]:
        bias = s["slopes"].reshape(kv, 1, G, 1) * away.abs()[:, None, :, None].float()
        x = x.sub_(bias.reshape(n, kv, m * G, L))
    return x, seen[:, :, None].expand(n, m, G, L).reshape(n, 1, m * G, L), seq, i


def _evict(s):
    c, pages, L, K = s["case"], s["pages"], s["case"]["max_len"], s["case"]["keep"]
    p, lens = torch.arange(L, device="cuda"), s["lens"][:, None, None]
    rank = torch.where(p >= lens - c["recent"], math.inf, s["mass"])
    rank = torch.where(p < lens, rank, -math.inf)
    kept = torch.sort(rank, dim=2, descending=True, stable=True).indices[..., :K]
    kept = torch.where(torch.arange(K, device="cuda") < lens, kept, L).sort(2).values   # [n][kv][K], L where there is none
    there = kept < L
    mass = torch.where(there, s["mass"].gather(2, kept.clamp(max=L - 1)), 0.0)
    at = kept.clamp(max=L - 1)
    row = torch.arange(c["n_seq"], device="cuda")[:, None, None]
    src = s["tables"].long()[row, at // c["page"]] * c["page"] + at % c["page"]         # [n][kv][K]
    seqs, pos = s["at"]
    src, head, dst = src[seqs, :, pos], torch.arange(c["kv_heads"], device="cuda"), s["read"].long()
    pages.k[dst] = pages.k[src, head]
    pages.v[dst] = pages.v[src, head]
    return (torch.where(there, kept, -1).to(torch.int32), s["lens"].clamp(max=K), mass, pages.k[dst], pages.v[dst])


# ---- what a pass cannot do without ---------------------------------------------------------------
def _seen(c):
    """Pairs of a token and a position that it sees."""
    total, w, P = 0, c["window"] or 1 << 30, c["prefix"]
    for n, m in zip(_lens(c), _new(c)):
        first, last = n - m, n - 1                                        # positions of the tokens
        if w > last and not P:
            total += (first + 1 + last + 1) * m // 2
            continue
        for t in range(first, last + 1):
            lo = max(0, t - w + 1)
            total += t + 1 - lo + min(lo, P) + max(0, min(P, n) - (t + 1))
    return total


def _reached(c):
    """Positions that some token sees."""
    total, w = 0, c["window"] or 1 << 30
    for n, m in zip(_lens(c), _new(c)):
        lo = max(0, n - m - w + 1)
        total += n - lo + min(lo, c["prefix"])
    return total


def work(case):
    c = case
    H, kv, hd = c["heads"], c["kv_heads"], c["hd"]
    if c["kind"] == "write":
        io = 4 if c["io"] == "f32" else 2
        # q read and written; k, v read, kept, read and given back
        return {"bytes": c["n_tok"] * (2 * H * hd * io + 2 * kv * hd * (io + 6) + 4 + 4 * c["axes"]), "flops": 8 * c["n_tok"] * (H + kv) * hd}
    if c["kind"] == "evict":
        kept = sum(min(n, c["keep"]) for n in _lens(c)) * kv
        # what was received, and the kept rows: read, written, read and given back
        return {"bytes": 4 * kv * sum(_lens(c)) + kept * (16 * hd + 8), "flops": kv * sum(_lens(c))}
    io, rows = 4 if c["io"] == "f32" else 2, sum(_new(c)) * H
    if c["kind"] == "mass":
        return {"bytes": 2 * kv * hd * _reached(c) + rows * (hd * io + 4) + 8 * kv * sum(_lens(c)), "flops": 2 * hd * H * _seen(c)}
    return {"bytes": 4 * kv * hd * _reached(c) + 2 * rows * hd * io, "flops": 4 * hd * H * _seen(c)}


# ---- the same in 64 bits -------------------------------------------------------------------------
def _tokens(c, seed):
    """Of every sequence, 64-bit scores [kv][m][G][n] with -inf where nothing is seen, and its values [kv][n][hd]."""
    k, v, _, _, _ = _cached(c, seed)
    q, G = _queries(c, seed).double(), c["heads"] // c["kv_heads"]
    row = at = 0
    for n, m in zip(_lens(c), _new(c)):
        kk, vv = k[at:at + n].double().permute(1, 2, 0).contiguous(), v[at:at + n].double().transpose(0, 1).contiguous()
        t = torch.arange(n - m, n, device="cuda").view(m, 1, 1)
        p = torch.arange(n, device="cuda")
        see = ((p <= t) & (p > t - (c["window"] or n + 1))) | (p < c["prefix"])
        for h in range(c["kv_heads"]):
            x = torch.matmul(q[row:row + m, h * G:(h + 1) * G].reshape(m * G, -1), kk[h]).view(m, G, n) / math.sqrt(c["hd"])
            if c["cap"]:
                x = c["cap"] * torch.tanh(x / c["cap"])
            if c["slopes"]:
                x = x - _slopes(c)[h * G:(h + 1) * G].double().view(1, G, 1) * (t - p).abs()
            yield row, m, h, torch.where(see, x, -math.inf), vv[h]
        row, at = row + m, at + n


def _sums(c, seed):
    """Logarithms of the sums of the exponentials that the weights are divided by, [tokens][heads]."""
    G = c["heads"] // c["kv_heads"]
    out = torch.empty(sum(_new(c)), c["heads"], device="cuda")
    for row, m, h, x, _ in _tokens(c, seed):
        out[row:row + m, h * G:(h + 1) * G] = torch.logsumexp(x, 2).float()
    return out


def exact(case, seed):
    c = case
    if c["kind"] == "write":
        q, k, v, gq, gk = _projected(c, seed)
        pos, _, _ = _positions(c, seed)
        cos, sin, sections = _angles(c)
        half, out = c["hd"] // 2, []
        for x, gamma in ((q, gq), (k, gk)):
            x = x.double()
            if gamma is not None:
                x = x / torch.sqrt((x ** 2).sum(-1, keepdim=True) / c["hd"] + EPS) * gamma.double()
            y, first = torch.empty_like(x), 0
            for axis, n in enumerate(sections):
                for j in range(first, first + n):
                    a, b = (j, j + half) if c["halves"] else (2 * j, 2 * j + 1)
                    cj, sj = cos[pos[axis].long(), j].double()[:, None], sin[pos[axis].long(), j].double()[:, None]
                    y[..., a] = x[..., a] * cj - x[..., b] * sj
                    y[..., b] = x[..., b] * cj + x[..., a] * sj
                first += n
            out.append(y)
        return out[0], out[1], v.double()
    if c["kind"] == "evict":
        k, v, _, _, _ = _cached(c, seed)
        mass, at, lens = _received(c, seed, c["max_len"]), 0, _lens(c)
        m = mass.cpu().double().numpy()
        kept = torch.full((c["n_seq"], c["kv_heads"], c["keep"]), -1, dtype=torch.int32)
        ks, vs = [], []
        for b, n in enumerate(lens):
            last = range(max(0, n - c["recent"]), n)
            heads = []
            for h in range(c["kv_heads"]):
                best = sorted(range(n - len(last)), key=lambda p: -m[b, h, p])[:max(0, c["keep"] - len(last))]
                heads.append(sorted(best + list(last)[-c["keep"]:]))
                kept[b, h, :len(heads[-1])] = torch.tensor(heads[-1], dtype=torch.int32)
            row = (torch.tensor(heads, device="cuda") + at).t()
            ks.append(k[row, torch.arange(c["kv_heads"], device="cuda")].double())
            vs.append(v[row, torch.arange(c["kv_heads"], device="cuda")].double())
            at += n
        kept = kept.cuda()
        new = torch.where(kept >= 0, mass.double().gather(2, kept.clamp(min=0).long()), 0.0)
        return kept, _ints([min(n, c["keep"]) for n in lens]), new, torch.cat(ks), torch.cat(vs)
    G = c["heads"] // c["kv_heads"]
    if c["kind"] == "mass":
        lse = _sums(c, seed).double()
        out, b, before = torch.zeros(c["n_seq"], c["kv_heads"], c["max_len"], dtype=torch.float64, device="cuda"), 0, _received(c, seed, c["max_len"])
        for row, m, h, x, _ in _tokens(c, seed):
            n = x.shape[2]
            w = torch.exp(x - lse[row:row + m, h * G:(h + 1) * G, None])
            out[b, h, :n] = before[b, h, :n].double() + w.sum((0, 1))
            b += h == c["kv_heads"] - 1
        return out
    out = torch.zeros(sum(_new(c)), c["heads"], c["hd"], dtype=torch.float64, device="cuda")
    for row, m, h, x, v in _tokens(c, seed):
        w = torch.softmax(x, 2)
        out[row:row + m, h * G:(h + 1) * G] = torch.matmul(w.view(m * G, -1), v).view(m, G, -1)
    return out
