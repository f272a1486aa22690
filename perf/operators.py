"""The operators of a served step over a paged key / value cache, as cases that can be timed: rows are rotated and appended to the
cache, they attend to it (over a prefix that the whole batch shares, too), and the next tokens are drawn from the rows' logits.

Shapes are the benchmark's (`c3`: 16 query heads on 2 key heads of 256, 64 of them rotated, vocabulary 151,936; `tiny`: 8 on 2 of 64,
vocabulary 32,000; contexts of 3,000 / 9,600 / 15,000 / 24,576) and, beside them, a generic attention layer (`gqa`: 32 heads on 8 of 128).
`own` = False: the plain form, elementary torch operations in 32 bits (angles and the sampler's sums in 64); True: the library's calls."""
import math

import torch

own = False

HEADS = {  # query heads, key heads, head width, rotated dimensions, normed per head before the rotation, gated output
    "c3": (16, 2, 256, 64, True, True),
    "tiny": (8, 2, 64, 32, True, True),
    "gqa": (32, 8, 128, 128, False, False),
}
VOCAB = {"c3": 151936, "tiny": 32000, "odd": 32003}
DTYPE = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
THETA, EPS = 1e7, 1e-6
CUT = 18.0     # the sampler: tokens more than 18 temperatures below the largest are never drawn


def listed():
    return [
        # one conversation, one token: the smallest call of a step, all launch and latency
        {"name": "append-1", "kind": "append", "heads": "c3", "seqs": 1, "rows": 1, "ctx_lo": 24576, "ctx_hi": 24576, "page": 64, "io": "f32", "cache": "f16"},
        # a served batch's step: 64 conversations with up to 4 rows each (speculation), their contexts far apart
        {"name": "append-64", "kind": "append", "heads": "gqa", "seqs": 64, "rows": 163, "ctx_lo": 3000, "ctx_hi": 15000, "page": 16, "io": "bf16", "cache": "bf16"},
        # a prompt, of a length that is no multiple of anything
        {"name": "append-4093", "kind": "append", "heads": "c3", "seqs": 1, "rows": 4093, "ctx_lo": 4093, "ctx_hi": 4093, "page": 64, "io": "bf16", "cache": "bf16"},
        # one token early in a small model's conversation: latency
        {"name": "attend-1", "kind": "attend", "heads": "tiny", "seqs": 1, "rows": 1, "ctx_lo": 257, "ctx_hi": 257, "shared": 0, "page": 16, "io": "f32", "cache": "f16"},
        # a verify pass (K = 3 drafts) of one long conversation over the packed 8-bit cache
        {"name": "attend-verify-4", "kind": "attend", "heads": "c3", "seqs": 1, "rows": 4, "ctx_lo": 24576, "ctx_hi": 24576, "shared": 0, "page": 64, "io": "f32", "cache": "q8"},
        # a served batch's step, ragged rows and contexts
        {"name": "attend-step-64", "kind": "attend", "heads": "gqa", "seqs": 64, "rows": 163, "ctx_lo": 3000, "ctx_hi": 15000, "shared": 0, "page": 16, "io": "bf16", "cache": "bf16"},
        # 64 conversations behind one long system prompt, a token each
        {"name": "attend-shared-64", "kind": "attend", "heads": "gqa", "seqs": 64, "rows": 64, "ctx_lo": 24651, "ctx_hi": 25813, "shared": 24576, "page": 16, "io": "bf16", "cache": "bf16"},
        # the same over the packed cache with drafts, the prefix ending inside a page
        {"name": "attend-shared-32-q8", "kind": "attend", "heads": "c3", "seqs": 32, "rows": 101, "ctx_lo": 9800, "ctx_hi": 11600, "shared": 9599, "page": 64, "io": "f32", "cache": "q8"},
        # a chunk of a long prompt against what was fed before it
        {"name": "attend-prompt-2045", "kind": "attend", "heads": "c3", "seqs": 1, "rows": 2045, "ctx_lo": 9600, "ctx_hi": 9600, "shared": 0, "page": 64, "io": "bf16", "cache": "bf16"},
        # the next token of one conversation
        {"name": "sample-1", "kind": "sample", "vocab": "c3", "rows": 1, "logits": "f32", "mix": "chat"},
        # of a served batch, every request with settings of its own
        {"name": "sample-64", "kind": "sample", "vocab": "c3", "rows": 64, "logits": "f32", "mix": "mixed"},
        # many draws from whole distributions (several answers to a prompt)
        {"name": "sample-250-whole", "kind": "sample", "vocab": "c3", "rows": 250, "logits": "bf16", "mix": "whole"},
    ]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm."""
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    kind = rng.choice(["append", "append", "attend", "attend", "attend", "sample", "sample"])
    if kind == "sample":
        return {"kind": kind, "vocab": rng.choice(["c3", "c3", "tiny", "odd"]), "rows": _spread(rng, 1, 250), "logits": rng.choice(["f32", "f32", "bf16", "f16"]),
                "mix": rng.choice(["chat", "mixed", "whole"])}
    heads = rng.choice(["c3", "gqa", "tiny"])
    page = rng.choice([8, 16, 32, 64, 128])
    if kind == "append":
        seqs = _spread(rng, 1, 64)
        rows = _spread(rng, 1, 4093) if seqs == 1 else rng.randint(seqs, 4 * seqs)
        lo = _spread(rng, max(200, rows), 24576)
        io = rng.choice(["f32", "bf16", "f16"])
        return {"kind": kind, "heads": heads, "seqs": seqs, "rows": rows, "ctx_lo": lo, "ctx_hi": _spread(rng, lo, 24576), "page": page, "io": io,
                "cache": rng.choice(["f16", "bf16"])}
    form = rng.choice(["step", "step", "shared", "prompt"])
    io = rng.choice(["f32", "bf16", "bf16", "f16"])
    cache = rng.choice({"f32": ["q8", "q8", "f16", "bf16"], "bf16": ["bf16", "bf16", "q8", "f16"], "f16": ["f16", "q8", "bf16"]}[io])
    c = {"kind": kind, "heads": heads, "seqs": 1, "rows": 1, "ctx_lo": 0, "ctx_hi": 0, "shared": 0, "page": page, "io": io, "cache": cache}
    if form == "prompt":
        c["rows"] = _spread(rng, 30, 1000)
        c["ctx_lo"] = c["ctx_hi"] = c["rows"] + _spread(rng, 1, 8000)
        return c
    c["seqs"] = _spread(rng, 1 if form == "step" else 4, 48)
    c["rows"] = rng.randint(c["seqs"], 4 * c["seqs"])
    if form == "shared":
        c["shared"] = _spread(rng, 500, 15000)
        c["ctx_lo"] = c["shared"] + rng.randint(10, 300)
        c["ctx_hi"] = c["ctx_lo"] + rng.randint(1, 1000)
    else:
        c["ctx_lo"] = _spread(rng, 200, 6000)
        c["ctx_hi"] = _spread(rng, c["ctx_lo"], 12000)
    return c


# ---- what a case is made of -----------------------------------------------------------------------------------------------------------
def _lengths(case):
    """Positions and rows of every sequence: contexts over [ctx_lo, ctx_hi], rows shared out unevenly."""
    n = case["seqs"]
    lens = [int(round(case["ctx_lo"] + (case["ctx_hi"] - case["ctx_lo"]) * ((i * 0.6180339887) % 1.0))) for i in range(n)]
    rows = [1] * n
    left = case["rows"] - n
    for i in range(n):                                   # the first sequences bring more
        take = min(left, 3 if n > 1 else left)
        rows[i] += take
        left -= take
    return lens, rows


def _head_bytes(cache, hd):
    return hd + (((hd // 32) * 2 + 15) & ~15) if cache == "q8" else 2 * hd


def _q8(x):
    """Packed heads of x [..., hd]: hd codes, then the groups' f16 scales (of 32 values each), zero-padded to 16 bytes."""
    hd = x.shape[-1]
    g = x.float().reshape(*x.shape[:-1], hd // 32, 32)
    sc = (g.abs().amax(-1) / 127).half()
    inv = torch.where(sc > 0, 1 / sc.float(), torch.zeros_like(sc, dtype=torch.float32))
    q = torch.round(g * inv[..., None]).clamp(-127, 127).to(torch.int8).reshape(x.shape).view(torch.uint8)
    out = torch.zeros(*x.shape[:-1], _head_bytes("q8", hd), dtype=torch.uint8, device=x.device)
    out[..., :hd] = q
    out[..., hd:hd + hd // 16] = sc.view(torch.uint8)
    return out


def _from_q8(b, hd, dtype):
    sc = b[..., hd:hd + hd // 16].contiguous().view(torch.float16).to(dtype)
    q = b[..., :hd].view(torch.int8).to(dtype).reshape(*b.shape[:-1], hd // 32, 32)
    return (q * sc[..., None]).reshape(*b.shape[:-1], hd)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    rnd = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    if case["kind"] == "sample":
        return _prepare_sample(case, g, rnd)
    nh, nkv, hd, rope, norm, gate = HEADS[case["heads"]]
    lens, rows = _lengths(case)
    n, R, ps, shared, io = case["seqs"], case["rows"], case["page"], case.get("shared", 0), DTYPE[case["io"]]
    st = {"case": dict(case), "lens_list": lens, "rows_list": rows, "heads": (nh, nkv, hd)}
    st["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    starts = [0]
    for m in rows:
        starts.append(starts[-1] + m)
    st["row_start"] = torch.tensor(starts, dtype=torch.int32, device="cuda")
    own_pages = [-(-(x - shared) // ps) for x in lens]
    width = max(own_pages)
    if case["kind"] == "append":
        # the appended rows' pages are their own; what lies before them is not read, so the pool holds a few pages for it
        first = [(x - m) // ps for x, m in zip(lens, rows)]
        used = [w - f for w, f in zip(own_pages, first)]
    else:
        first, used = [0] * n, own_pages
    spare = 8
    total = sum(used) + -(-shared // ps) + spare
    order = torch.randperm(total, device="cuda", generator=g).to(torch.int32)          # pages are handed out in no order
    at = torch.arange(width, device="cuda")[None, :] - torch.tensor(first, device="cuda")[:, None]
    base = torch.tensor([sum(used[:i]) for i in range(n)], device="cuda")[:, None]
    mine = (at >= 0) & (at < torch.tensor(used, device="cuda")[:, None])
    st["pages"] = order[torch.where(mine, base + at, total - spare + at % spare)].contiguous()
    st["shared_pages"] = order[sum(used):sum(used) + -(-shared // ps)].contiguous()
    if case["cache"] == "q8":
        st["k"], st["v"] = _q8(rnd(total, nkv, ps, hd)), _q8(rnd(total, nkv, ps, hd))
    else:
        st["k"], st["v"] = (rnd(total, nkv, ps, hd).to(DTYPE[case["cache"]]) for _ in range(2))
    if case["kind"] == "append":
        st["kin"], st["vin"], st["q"] = rnd(R, nkv, hd).to(io), rnd(R, nkv, hd).to(io), rnd(R, nh, hd).to(io)
        st["q_norm"], st["k_norm"] = ((1 + 0.1 * rnd(hd), 1 + 0.1 * rnd(hd)) if norm else (None, None))
        st["rope"], st["q_out"] = rope, torch.empty(R, nh, hd, dtype=io, device="cuda")
    else:
        st["q"] = (1.5 * rnd(R, nh, hd)).to(io)
        st["gate"] = rnd(R, nh, hd).to(io) if gate else None
        st["out"] = torch.empty(R, nh, hd, dtype=io, device="cuda")
    return st


def _prepare_sample(case, g, rnd):
    R, V = case["rows"], VOCAB[case["vocab"]]
    lg = 2.5 * rnd(R, V)
    lg.scatter_add_(1, torch.randint(0, V, (R, 40), device="cuda", generator=g), 6 + 4 * rnd(R, 40).abs())   # a few dozen likely tokens a row
    u = lambda: torch.rand(R, device="cuda", generator=g)  # noqa: E731
    full = lambda x, t=torch.float32: torch.full((R,), x, dtype=t, device="cuda")  # noqa: E731
    st = {"case": dict(case), "logits": lg.to(DTYPE[case["logits"]]), "u": torch.rand(R, dtype=torch.float64, device="cuda", generator=g)}
    if case["mix"] == "chat":
        st["temperature"], st["top_k"], st["top_p"], st["min_p"] = full(0.7), full(20, torch.int32), full(0.9), full(0.0)
    elif case["mix"] == "whole":
        st["temperature"], st["top_k"], st["top_p"], st["min_p"] = full(1.0), full(V, torch.int32), full(1.0), full(0.0)
    else:
        st["temperature"] = 0.2 + 1.2 * u()
        k = (2 ** (1 + 8 * u())).to(torch.int32)
        st["top_k"] = torch.where(u() < 0.5, k, torch.full_like(k, V))
        st["top_p"] = torch.where(u() < 0.7, 0.5 + 0.5 * u(), torch.ones(R, device="cuda"))
        st["min_p"] = torch.where(u() < 0.3, 0.1 * u(), torch.zeros(R, device="cuda"))
    st["token"], st["prob"] = torch.empty(R, dtype=torch.int32, device="cuda"), torch.empty(R, dtype=torch.float32, device="cuda")
    return st


# ---- one pass ---------------------------------------------------------------------------------------------------------------------------
def run(st):
    kind = st["case"]["kind"]
    if own:
        return _own(st, kind)
    return {"append": _append, "attend": _attend, "sample": _sample}[kind](st)


def _own(st, kind):
    if "pkg" not in st:
        import __graft_entry__ as graft
        st["pkg"] = graft.load_package()
    pkg = st["pkg"]
    if kind == "sample":
        pkg.sampling.sample_rows(st["logits"], st["u"], temperature=st["temperature"], top_k=st["top_k"], top_p=st["top_p"], min_p=st["min_p"],
                                 out=st["token"], prob=st["prob"])
        return {"token": st["token"], "prob": st["prob"]}
    if "step" not in st:      # what a server keeps from step to step: the cache, its tables, a scratch
        cache = pkg.paged.Cache(st["k"], st["v"], st["heads"][2])
        st["step"] = pkg.paged.Step(cache, st["pages"], st["row_start"], st["lens"], st["case"]["rows"], st["heads"][0],
                                    shared_pages=st["shared_pages"], shared_len=st["case"].get("shared", 0))
    if kind == "append":
        st["step"].append(st["kin"], st["vin"], q=st["q"], q_out=st["q_out"], rope_dims=st["rope"], theta=THETA, q_norm=st["q_norm"], k_norm=st["k_norm"], eps=EPS)
        return {"k": st["k"], "v": st["v"], "q": st["q_out"]}
    st["step"].attend(st["q"], out=st["out"], gate=st["gate"])
    return {"out": st["out"]}


def _row_places(st):
    """Of every row: its sequence and its position in it."""
    rs = st["row_start"].long()
    r = torch.arange(st["case"]["rows"], device="cuda")
    b = torch.searchsorted(rs, r, right=True) - 1
    return b, st["lens"].long()[b] - (rs[b + 1] - r)


def _rotated(x, w, pos, rope):
    """x [rows, heads, hd] in 32 bits: normed by its own length where w is given, then its first `rope` dimensions turned, i with i + rope / 2."""
    x = x.float()
    if w is not None:
        x = x * torch.rsqrt(x.double().square().mean(-1, keepdim=True) + EPS).float() * w
    h = rope // 2
    angle = pos.double()[:, None] / THETA ** (2 * torch.arange(h, dtype=torch.float64, device="cuda") / rope)
    cs, sn = angle.cos().float()[:, None, :], angle.sin().float()[:, None, :]
    a, b = x[..., :h], x[..., h:rope]
    return torch.cat([a * cs - b * sn, b * cs + a * sn, x[..., rope:]], -1)


def _append(st):
    ps, shared = st["case"]["page"], st["case"].get("shared", 0)
    b, pos = _row_places(st)
    page = st["pages"][b, (pos - shared) // ps].long()
    slot = (pos - shared) % ps
    st["k"][page, :, slot] = _rotated(st["kin"], st["k_norm"], pos, st["rope"]).to(st["k"].dtype)
    st["v"][page, :, slot] = st["vin"].to(st["v"].dtype)
    st["q_out"].copy_(_rotated(st["q"], st["q_norm"], pos, st["rope"]))
    return {"k": st["k"], "v": st["v"], "q": st["q_out"]}


def _values(st, pool, pages):
    """[.., positions, kv head, hd] in 32 bits of the pages of a table."""
    x = pool[pages.long()]                                   # [.., page, kv head, slot, bytes or values]
    x = _from_q8(x, st["heads"][2], torch.float32) if st["case"]["cache"] == "q8" else x.float()
    x = x.transpose(-3, -2)
    return x.reshape(*pages.shape[:-1], -1, *x.shape[-2:])


def _attend(st):
    nh, nkv, hd = st["heads"]
    G, R, n, shared = nh // nkv, st["case"]["rows"], st["case"]["seqs"], st["case"]["shared"]
    b, pos = _row_places(st)
    place = torch.arange(R, device="cuda") - st["row_start"].long()[b]
    M = max(st["rows_list"])
    q = st["q"].float() / math.sqrt(hd)
    # every sequence's own positions, padded to the longest one's rows and positions
    qp = torch.zeros(n, M, nh, hd, device="cuda")
    qp[b, place] = q
    qp = qp.view(n, M, nkv, G, hd).permute(0, 2, 1, 3, 4).reshape(n, nkv, M * G, hd)
    last = torch.full((n, M), -1, dtype=torch.int64, device="cuda")
    last[b, place] = pos - shared                                        # the last own position a row attends to
    k = _values(st, st["k"], st["pages"])                                # [n, L, key heads, hd]
    s = torch.matmul(qp, k.permute(0, 2, 3, 1)).view(n, nkv, M, G, -1)
    del k
    s.masked_fill_(torch.arange(s.shape[-1], device="cuda") > last[:, None, :, None, None], -math.inf)
    v = _values(st, st["v"], st["pages"])
    parts = [[x.view(n, nkv, M, G, -1).permute(0, 2, 1, 3, 4)[b, place] for x in _part(s, v.transpose(1, 2))]]
    if shared:
        ks, vs = (_values(st, st[x], st["shared_pages"])[:shared].transpose(0, 1) for x in "kv")     # [key heads, S, hd]
        s = torch.matmul(q.view(R, nkv, G, hd).transpose(0, 1).reshape(nkv, R * G, hd), ks.transpose(1, 2)).view(nkv, R, G, -1)
        s.masked_fill_(torch.arange(shared, device="cuda") > pos[:, None, None], -math.inf)
        parts.append([x.view(nkv, R, G, -1).transpose(0, 1) for x in _part(s, vs)])
    top = torch.stack([p[0] for p in parts]).amax(0)
    share = [torch.exp(p[0] - torch.where(top > -math.inf, top, 0.0)) for p in parts]
    total = sum(w * p[1] for w, p in zip(share, parts))
    o = sum(w * p[2] for w, p in zip(share, parts)) / torch.where(total > 0, total, 1.0)
    o = o.reshape(R, nh, hd)
    if st["gate"] is not None:
        o = o * torch.sigmoid(st["gate"].float())
    st["out"].copy_(o)
    return {"out": st["out"]}


def _part(s, v):
    """Largest score, sum of the weights and weighted values of scores s [.., positions] (masked ones -inf)."""
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top > -math.inf, top, 0.0))
    return top, p.sum(-1, keepdim=True), torch.matmul(p.flatten(-3, -2), v)


def _sample(st):
    lg = st["logits"].float()
    lg = torch.where(torch.isnan(lg), -math.inf, lg)
    v, ids = torch.sort(lg, dim=1, descending=True, stable=True)         # equal ones: the lowest id first
    T = st["temperature"][:, None]
    at = torch.arange(v.shape[1], device="cuda")[None, :]
    may = (v >= v[:, :1] - CUT * T) & (at < st["top_k"].clamp(min=1)[:, None])
    w = torch.where(may, torch.exp(((v - v[:, :1]) * (1 / T)).double()), 0.0)            # the largest has weight 1
    total = w.sum(1, keepdim=True)
    keep = may & (w >= st["min_p"].double()[:, None])
    w = torch.where(keep, w, 0.0)
    run_ = w.cumsum(1)
    p = st["top_p"].double()[:, None]
    keep &= (run_ - w < p * total) | (p >= 1)                            # up to the one that reaches top_p
    w = torch.where(keep, w, 0.0)
    run_ = w.cumsum(1)
    mass = w.sum(1, keepdim=True)
    place = torch.minimum((run_ <= st["u"][:, None] * mass).sum(1), keep.sum(1) - 1)
    st["token"].copy_(ids.gather(1, place[:, None])[:, 0])
    st["prob"].copy_((w.gather(1, place[:, None]) / mass)[:, 0])
    return {"token": st["token"], "prob": st["prob"]}


# ---- the work a pass cannot do without, and its values in 64 bits -------------------------------------------------------------------
def work(case):
    if case["kind"] == "sample":
        n = case["rows"] * VOCAB[case["vocab"]]
        return {"bytes": n * DTYPE[case["logits"]].itemsize + case["rows"] * 32, "flops": 4 * n}
    nh, nkv, hd, rope, norm, gate = HEADS[case["heads"]]
    lens, rows = _lengths(case)
    io, R, hb = DTYPE[case["io"]].itemsize, case["rows"], _head_bytes(case["cache"], hd)
    if case["kind"] == "append":
        return {"bytes": R * ((2 * nkv + 2 * nh) * hd * io + 2 * nkv * hb + 8), "flops": R * (nh + nkv) * (3 * rope + (4 * hd if norm else 0))}
    positions = case["shared"] + sum(x - case["shared"] for x in lens)
    pairs = sum(m * (x - m) + m * (m + 1) // 2 for x, m in zip(lens, rows))
    return {"bytes": 2 * nkv * hb * positions + (3 if gate else 2) * R * nh * hd * io + 4 * sum(-(-x // case["page"]) for x in lens), "flops": 4 * nh * hd * pairs}


def exact(case, seed):
    st = prepare(case, seed)
    if case["kind"] == "sample":
        return _exact_sample(st)
    nh, nkv, hd, rope, norm, gate = HEADS[case["heads"]]
    lens, rows = _lengths(case)
    shared, ps = case.get("shared", 0), case["page"]

    def of_row(b, t):       # page and slot of position t of sequence b
        return (int(st["shared_pages"][t // ps]), t % ps) if t < shared else (int(st["pages"][b, (t - shared) // ps]), (t - shared) % ps)

    if case["kind"] == "append":
        k, v = st["k"].double(), st["v"].double()
        pos = torch.cat([torch.arange(x - m, x, dtype=torch.float64, device="cuda") for x, m in zip(lens, rows)])
        at = [of_row(b, t) for b, (x, m) in enumerate(zip(lens, rows)) for t in range(x - m, x)]
        page, slot = (torch.tensor(x, device="cuda") for x in zip(*at))
        k[page, :, slot] = _exact_rotated(st["kin"], st["k_norm"], pos, rope)
        v[page, :, slot] = st["vin"].double()
        return {"k": k, "v": v, "q": _exact_rotated(st["q"], st["q_norm"], pos, rope)}
    of = (lambda x: _from_q8(x, hd, torch.float64)) if case["cache"] == "q8" else (lambda x: x.double())
    table = lambda pool, ids, length: of(pool[ids.long()]).transpose(1, 2).reshape(-1, nkv, hd)[:length]  # noqa: E731
    front = [table(st[x], st["shared_pages"], shared) if shared else None for x in "kv"]
    out, r = [], 0
    for b, (x, m) in enumerate(zip(lens, rows)):
        k, v = (table(st[n], st["pages"][b, :-(-(x - shared) // ps)], x - shared) for n in "kv")
        if shared:
            k, v = torch.cat([front[0], k]), torch.cat([front[1], v])
        q = st["q"][r:r + m].double()
        later = torch.arange(x, device="cuda")[None, :] > torch.arange(x - m, x, device="cuda")[:, None]
        heads = []
        for h in range(nh):
            s = (q[:, h] @ k[:, h // (nh // nkv)].T) * hd ** -0.5
            heads.append(torch.softmax(s.masked_fill(later, -math.inf), -1) @ v[:, h // (nh // nkv)])
        out.append(torch.stack(heads, 1))
        r += m
    out = torch.cat(out)
    return {"out": out / (1 + torch.exp(-st["gate"].double())) if gate else out}


def _exact_rotated(x, w, pos, rope):
    x = x.double()
    if w is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * w.double()
    z = torch.complex(x[..., :rope // 2], x[..., rope // 2:rope])
    turn = torch.outer(pos, THETA ** (-torch.arange(0, rope, 2, dtype=torch.float64, device="cuda") / rope))
    z = z * torch.polar(torch.ones_like(turn), turn)[:, None, :]
    return torch.cat([z.real, z.imag, x[..., rope:]], -1)


def _exact_sample(st):
    tokens, probs = [], []
    for r in range(st["case"]["rows"]):
        lg, T = st["logits"][r].double(), st["temperature"][r].double()
        order = torch.argsort(lg, descending=True, stable=True)[:max(1, int(st["top_k"][r]))]
        x = (lg[order] - lg[order[0]]) / T
        w = torch.exp(x[x >= -CUT])
        total, n = w.sum(), int((w >= st["min_p"][r].double()).sum())
        if float(st["top_p"][r]) < 1:
            n = min(n, int((w[:n].cumsum(0) < st["top_p"][r].double() * total).sum()) + 1)
        w = w[:n]
        i = min(int(torch.searchsorted(w.cumsum(0), st["u"][r] * w.sum(), right=True)), n - 1)
        tokens.append(order[i].to(torch.int32))
        probs.append(w[i] / w.sum())
    return {"token": torch.stack(tokens), "prob": torch.stack(probs)}
