"""More operators of a served step, as cases that can be timed: the DeltaNet layer of a batch of sequences whose states lie in slots of a pool - the
causal convolution with its carried rows, the gated delta rule for single tokens, drafts and whole prompts - and the log probabilities of given
tokens with the distribution's entropy and its best alternatives.

Shapes are the benchmark's (`c3`: 16 key and 32 value heads of 128, convolution over 4 rows, vocabulary 151,936; `tiny`: 4 and 4 of 64, vocabulary
32,000) and, beside them, a generic layer (`gen`: 16 value heads of 64, two beside each other on one of 8 key heads, convolution over 3 rows, neither norm nor gate).
`own` = False: the plain form, elementary torch operations in 32 bits (the softmax's sums and the gates' exponents in 64); True: the library's calls."""
import math

import torch

own = False

HEADS = {  # key heads, value heads, width, rows of the convolution, value heads of a key head side by side (or tiled), outputs normed and gated
    "c3": (16, 32, 128, 4, False, True),
    "tiny": (4, 4, 64, 4, False, True),
    "gen": (8, 16, 64, 3, True, False),
}
VOCAB = {"c3": 151936, "tiny": 32000, "odd": 32003}
DTYPE = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
EPS = 1e-6


def listed():
    return [
        # one conversation, one token: the smallest call, all launch and latency
        {"name": "conv-1", "kind": "conv", "heads": "c3", "seqs": 1, "lo": 1, "hi": 1, "new": False, "fork": False, "io": "f32"},
        # a served batch's step: 64 conversations with up to 4 rows each (speculation); states go to other slots, so that a refused draft costs nothing
        {"name": "conv-64", "kind": "conv", "heads": "c3", "seqs": 64, "lo": 1, "hi": 4, "new": False, "fork": True, "io": "bf16"},
        # a prompt, of a length that is no multiple of anything
        {"name": "conv-4093", "kind": "conv", "heads": "c3", "seqs": 1, "lo": 4093, "hi": 4093, "new": True, "fork": False, "io": "bf16"},
        # the rule for one token of one conversation
        {"name": "rule-1", "kind": "rule", "heads": "c3", "seqs": 1, "lo": 1, "hi": 1, "new": False, "fork": False, "replay": False, "io": "f32"},
        # the same batch's step: every state is read and written once
        {"name": "rule-64", "kind": "rule", "heads": "c3", "seqs": 64, "lo": 1, "hi": 4, "new": False, "fork": True, "replay": False, "io": "bf16"},
        # drafts were refused: the states again, after the rows that are kept, without outputs
        {"name": "rule-replay-32", "kind": "rule", "heads": "c3", "seqs": 32, "lo": 1, "hi": 8, "new": False, "fork": False, "replay": True, "io": "f32"},
        # the prompt of above
        {"name": "rule-4093", "kind": "rule", "heads": "c3", "seqs": 1, "lo": 4093, "hi": 4093, "new": True, "fork": False, "replay": False, "io": "bf16"},
        # several prompts' chunks at once, each behind what was fed before it
        {"name": "rule-prompts-9", "kind": "rule", "heads": "c3", "seqs": 9, "lo": 203, "hi": 1811, "new": False, "fork": False, "replay": False, "io": "bf16"},
        # a prompt of a small model in 32 bits
        {"name": "rule-tiny-700", "kind": "rule", "heads": "tiny", "seqs": 1, "lo": 701, "hi": 701, "new": True, "fork": False, "replay": False, "io": "f32"},
        # what an answer's next token weighed, and five others
        {"name": "logprob-1", "kind": "logprob", "vocab": "c3", "rows": 1, "logits": "f32", "top": 5, "temperature": False},
        # a served batch's tokens
        {"name": "logprob-64", "kind": "logprob", "vocab": "c3", "rows": 64, "logits": "f32", "top": 20, "temperature": True},
        # a prompt scored token by token
        {"name": "logprob-1021", "kind": "logprob", "vocab": "c3", "rows": 1021, "logits": "bf16", "top": 1, "temperature": False},
    ]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm."""
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    kind = rng.choice(["conv", "conv", "rule", "rule", "rule", "logprob", "logprob"])
    if kind == "logprob":
        return {"kind": kind, "vocab": rng.choice(["c3", "c3", "tiny", "odd"]), "rows": _spread(rng, 1, 500), "logits": rng.choice(["f32", "f32", "bf16", "f16"]),
                "top": rng.choice([0, 1, 5, 8, 20, 64]), "temperature": rng.random() < 0.4}
    form = rng.choice(["step", "step", "prompt", "prompts"])
    c = {"kind": kind, "heads": rng.choice(["c3", "tiny", "gen"]), "seqs": 1, "lo": 1, "hi": 1, "new": form != "step" and rng.random() < 0.5,
         "fork": rng.random() < 0.4, "io": rng.choice(["f32", "bf16", "bf16", "f16"])}
    if kind == "rule":
        c["replay"] = form == "step" and rng.random() < 0.2
    if form == "step":
        c["seqs"] = _spread(rng, 1, 64)
        c["hi"] = rng.randint(1, 8)
    elif form == "prompt":
        c["lo"] = c["hi"] = _spread(rng, 9, 4093)
    else:
        c["seqs"] = rng.randint(2, 9)
        c["lo"] = _spread(rng, 5, 400)
        c["hi"] = _spread(rng, c["lo"], 1500)
    return c


# ---- what a case is made of -----------------------------------------------------------------------------------------------------------
def _rows(case):
    """Rows of every sequence, spread over [lo, hi]."""
    return [case["lo"] + int((case["hi"] - case["lo"] + 1) * (((i + 1) * 0.6180339887) % 1.0)) for i in range(case["seqs"])]


def _kept(case):
    """Of every sequence the rows that a replay keeps."""
    return [1 + i % m for i, m in enumerate(_rows(case))]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    rnd = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    if case["kind"] == "logprob":
        return _prepare_logprob(case, g, rnd)
    kh, vh, d, conv_k, grouped, normed = HEADS[case["heads"]]
    counts, n, io = _rows(case), case["seqs"], DTYPE[case["io"]]
    R, ch = sum(counts), (2 * kh + vh) * d
    st = {"case": dict(case), "counts": counts, "rows": R, "conv_k": conv_k}
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    starts = [0]
    for m in counts:
        starts.append(starts[-1] + m)
    st["row_start"] = ints(starts)
    st["lens"] = ints([m + (0 if case["new"] else 300 + 7 * i) for i, m in enumerate(counts)])
    slots = (2 if case["fork"] else 1) * n + 2
    order = torch.randperm(slots, device="cuda", generator=g).to(torch.int32)               # slots are handed out in no order
    st["slots"] = order[:n].contiguous()
    st["to"] = order[n:2 * n].contiguous() if case["fork"] else None
    if case["kind"] == "conv":
        st["conv"] = rnd(slots, conv_k - 1, ch).to(io)
        st["x"], st["w"] = rnd(R, ch).to(io), 0.3 * rnd(ch, conv_k)
        st["out"] = torch.zeros(R, ch, dtype=io, device="cuda")
        return st
    st["state"] = 0.2 * rnd(slots, vh, d, d)
    y = torch.nn.functional.silu(rnd(R, ch)).to(io)                                         # what the convolution gives: queries, keys and values side by side
    st["q"], st["k"], st["v"] = (t.unflatten(1, (-1, d)) for t in y.split([kh * d, kh * d, vh * d], 1))
    st["alpha"], st["beta"] = rnd(R, vh).to(io), rnd(R, vh).to(io)
    st["a"] = -torch.exp(math.log(0.002) + (math.log(1.5) - math.log(0.002)) * torch.rand(vh, device="cuda", generator=g))      # heads that forget in two rows to a thousand
    st["dt"] = 0.1 * rnd(vh)
    st["take"] = ints(_kept(case)) if case["replay"] else None
    st["z"], st["norm"] = (rnd(R, vh, d).to(io), 1 + 0.1 * rnd(d)) if normed and not case["replay"] else (None, None)
    st["out"] = None if case["replay"] else torch.zeros(R, vh, d, dtype=io, device="cuda")
    return st


def _prepare_logprob(case, g, rnd):
    R, V = case["rows"], VOCAB[case["vocab"]]
    lg = 2.5 * rnd(R, V)
    lg.scatter_add_(1, torch.randint(0, V, (R, 40), device="cuda", generator=g), 6 + 4 * rnd(R, 40).abs())   # a few dozen likely tokens a row
    u = lambda *s: torch.rand(*s, device="cuda", generator=g)  # noqa: E731
    drawn = torch.cat([(x - (-u(*x.shape).clamp_min(1e-20).log()).log()).argmax(1) for x in lg.split(64)])   # a token of the distribution, or (unlikely text) any
    some = torch.randint(0, V, (R,), device="cuda", generator=g)
    st = {"case": dict(case), "logits": lg.to(DTYPE[case["logits"]]), "tokens": torch.where(u(R) < 0.8, drawn, some).to(torch.int32)}
    st["temperature"] = 0.2 + 1.2 * u(R) if case["temperature"] else None
    return st


# ---- one pass ---------------------------------------------------------------------------------------------------------------------------
def run(st):
    kind = st["case"]["kind"]
    if own:
        return _own(st, kind)
    return {"conv": _conv, "rule": _rule, "logprob": _logprob}[kind](st)


def _own(st, kind):
    if "pkg" not in st:
        import __graft_entry__ as graft
        st["pkg"] = graft.load_package()
    pkg, case = st["pkg"], st["case"]
    if kind == "logprob":
        st["res"] = pkg.sampling.logprob_rows(st["logits"], st["tokens"], top=case["top"], temperature=st["temperature"], out=st.get("res"))
        return dict(st["res"]._asdict())
    kh, vh, d, conv_k, grouped, _ = HEADS[case["heads"]]
    if "step" not in st:      # what a server keeps from step to step: the pool, its tables, a scratch
        pool = pkg.delta.States(kh, vh, d, state=st.get("state"), conv=st.get("conv"), grouped=grouped)
        st["step"] = pkg.delta.Step(pool, st["row_start"], st["lens"], st["slots"], st["rows"], to=st["to"], take=st.get("take"), max_rows=max(st["counts"]))
    if kind == "conv":
        st["step"].conv(st["x"], st["w"], out=st["out"])
        return {"y": st["out"], "conv": st["conv"]}
    if case["replay"]:
        st["step"].replay(st["k"], st["v"], st["alpha"], st["beta"], st["a"], st["dt"])
        return {"state": st["state"]}
    st["step"].rule(st["q"], st["k"], st["v"], st["alpha"], st["beta"], st["a"], st["dt"], z=st["z"], norm=st["norm"], eps=EPS, out=st["out"])
    return {"out": st["out"], "state": st["state"]}


def _conv(st):
    """Every sequence's carried rows before its own; the sum over the shifted rows; the last rows are carried on."""
    k, counts, slots = st["conv_k"], st["counts"], st["slots"].long()
    to = slots if st["to"] is None else st["to"].long()
    rs = st["row_start"].long()
    n, most = len(counts), max(counts)
    at = torch.arange(most, device="cuda")
    mine = at[None, :] < (rs[1:] - rs[:-1])[:, None]                              # [sequences, rows]: rows of shorter ones are empty
    x = torch.zeros(n, k - 1 + most, st["x"].shape[1], device="cuda")
    old = st["conv"][slots].float()
    new = st["lens"].long() <= rs[1:] - rs[:-1]
    x[:, :k - 1] = torch.where(new[:, None, None], torch.zeros_like(old), old)
    x[:, k - 1:][mine] = st["x"].float()
    y = sum(x[:, t:t + most] * st["w"][:, t] for t in range(k))
    y = y * torch.sigmoid(y)
    st["out"].copy_(y[mine])
    last = (rs[1:] - rs[:-1])[:, None] + torch.arange(k - 1, device="cuda")       # the k - 1 rows before the next one
    st["conv"][to] = x[torch.arange(n, device="cuda")[:, None], last].to(st["conv"].dtype)
    return {"y": st["out"], "conv": st["conv"]}


def _rule(st):
    """Row after row, all sequences and heads at once."""
    kh, vh, d, _, grouped, _ = HEADS[st["case"]["heads"]]
    rs = st["row_start"].long()
    counts = rs[1:] - rs[:-1]
    take = counts if st["take"] is None else torch.minimum(st["take"].long(), counts)
    to = (st["slots"] if st["to"] is None else st["to"]).long()
    S = st["state"][st["slots"].long()]
    S = torch.where((st["lens"].long() <= counts)[:, None, None, None], torch.zeros_like(S), S)
    of = torch.arange(vh, device="cuda") // (vh // kh) if grouped else torch.arange(vh, device="cuda") % kh      # the key head of a value head
    unit = lambda x: x.float() * torch.rsqrt(x.float().square().sum(-1, keepdim=True) + 1e-6)  # noqa: E731
    k, q = unit(st["k"]), unit(st["q"]) / math.sqrt(d)
    v, beta = st["v"].float(), torch.sigmoid(st["beta"].float())
    decay = torch.exp(st["a"].double() * torch.nn.functional.softplus(st["alpha"].double() + st["dt"].double())).float()
    o = torch.zeros(st["rows"], vh, d, device="cuda")
    for t in range(max(st["counts"])):
        live = take > t
        r = torch.where(live, rs[:-1] + t, 0)
        kt, qt = k[r][:, of], q[r][:, of]
        new = S * decay[r][:, :, None, None]
        delta = (v[r] - torch.einsum("bhij,bhi->bhj", new, kt)) * beta[r][:, :, None]
        new = new + kt[..., :, None] * delta[..., None, :]
        S = torch.where(live[:, None, None, None], new, S)
        if st["out"] is not None:
            o.index_add_(0, r, torch.where(live[:, None, None], torch.einsum("bhij,bhi->bhj", S, qt), 0.0))
    st["state"][to] = S
    if st["out"] is None:
        return {"state": st["state"]}
    if st["norm"] is not None:
        o = o * torch.rsqrt(o.square().mean(-1, keepdim=True) + EPS) * st["norm"] * torch.sigmoid(st["z"].float())
    st["out"].copy_(o)
    return {"out": st["out"], "state": st["state"]}


def _logprob(st):
    lg, n = st["logits"].float(), st["case"]["top"]
    V = lg.shape[1]
    lg = torch.where(torch.isnan(lg), -math.inf, lg)
    top, best = lg.max(1, keepdim=True)
    best = (lg == top).int().argmax(1, keepdim=True)                                # the lowest of equal ones
    inv = 1.0 if st["temperature"] is None else 1 / st["temperature"][:, None]
    x = (lg - top) * inv
    w = torch.exp(x.double()).scatter_(1, best, 0.0)                                # all but the largest, which weighs 1
    s = w.sum(1)
    log_z = torch.log1p(s)
    token = st["tokens"].long()[:, None]
    own_x = x.gather(1, token)
    v = lg.gather(1, token)
    before = (lg > v) | ((lg == v) & (torch.arange(V, device="cuda")[None, :] < token))      # (by the logits: their product with 1 / T may round to equal ones)
    res = {"logprob": (own_x[:, 0].double() - log_z).float(), "rank": before.sum(1).to(torch.int32),
           "entropy": (log_z - torch.where(w > 0, w * x, 0.0).sum(1) / (1 + s)).float()}
    ids = torch.sort(lg, dim=1, descending=True, stable=True)[1][:, :n]             # equal ones: the lowest id first
    res["top_ids"], res["top_logprobs"] = ids.to(torch.int32), (x.gather(1, ids).double() - log_z[:, None]).float()
    return res


# ---- the work a pass cannot do without, and its values in 64 bits -------------------------------------------------------------------
def work(case):
    if case["kind"] == "logprob":
        n = case["rows"] * VOCAB[case["vocab"]]
        return {"bytes": n * DTYPE[case["logits"]].itemsize + case["rows"] * (16 + 8 * case["top"]), "flops": 4 * n}
    kh, vh, d, conv_k, _, normed = HEADS[case["heads"]]
    io, n, counts, ch = DTYPE[case["io"]].itemsize, case["seqs"], _rows(case), (2 * kh + vh) * d
    states = n * (1 if case["new"] else 2)
    if case["kind"] == "conv":
        R = sum(counts)
        return {"bytes": 2 * R * ch * io + states * (conv_k - 1) * ch * io + 4 * ch * conv_k, "flops": R * ch * (2 * conv_k + 4)}
    if case["replay"]:
        R = sum(_kept(case))
        return {"bytes": R * ((kh + vh) * d + 2 * vh) * io + states * 4 * vh * d * d, "flops": R * vh * 4 * d * d}
    R = sum(counts)
    return {"bytes": R * ((2 * kh + (3 if normed else 2) * vh) * d + 2 * vh) * io + states * 4 * vh * d * d, "flops": R * vh * 6 * d * d}


def exact(case, seed):
    st = prepare(case, seed)
    return {"conv": _exact_conv, "rule": _exact_rule, "logprob": _exact_logprob}[case["kind"]](st)


def _exact_conv(st):
    k, pool = st["conv_k"], st["conv"].double()
    to = (st["slots"] if st["to"] is None else st["to"]).tolist()
    out, r = [], 0
    for b, m in enumerate(st["counts"]):
        past = st["conv"][int(st["slots"][b])].double() * (int(st["lens"][b]) > m)
        seq = torch.cat([past, st["x"][r:r + m].double()])
        y = torch.einsum("mck,ck->mc", seq.unfold(0, k, 1), st["w"].double())
        out.append(y / (1 + torch.exp(-y)))
        pool[to[b]] = seq[m:]
        r += m
    return {"y": torch.cat(out), "conv": pool}


def _exact_rule(st):
    """Blocks of rows: with the decays' logarithms summed up, the rows' changes solve a triangular system."""
    kh, vh, d, _, grouped, _ = HEADS[st["case"]["heads"]]
    pool = st["state"].double()
    to = (st["slots"] if st["to"] is None else st["to"]).tolist()
    gate = st["a"].double() * torch.log1p(torch.exp(st["alpha"].double() + st["dt"].double()))
    beta = 1 / (1 + torch.exp(-st["beta"].double()))
    heads = [h // (vh // kh) if grouped else h % kh for h in range(vh)]
    out = torch.zeros(st["rows"], vh, d, dtype=torch.float64, device="cuda")
    r0 = 0
    for b, m in enumerate(st["counts"]):
        S = st["state"][int(st["slots"][b])].double() * (int(st["lens"][b]) > m)
        upto = r0 + (m if st["take"] is None else min(m, int(st["take"][b])))
        for r in range(r0, upto, 32):
            e = min(r + 32, upto)
            k = st["k"][r:e, heads].double().transpose(0, 1)                        # [heads, rows, d]
            k = k / torch.sqrt((k * k).sum(-1, keepdim=True) + 1e-6)
            q = st["q"][r:e, heads].double().transpose(0, 1)
            q = q / torch.sqrt((q * q).sum(-1, keepdim=True) + 1e-6) * d ** -0.5
            G = gate[r:e].T.cumsum(1)                                               # [heads, rows]
            ratio = torch.exp((G[:, :, None] - G[:, None, :]).clamp(max=0.0)).tril()
            bt = beta[r:e].T[:, :, None]
            A = torch.tril(bt * ratio * (k @ k.transpose(1, 2)), -1) + torch.eye(e - r, dtype=torch.float64, device="cuda")
            rhs = bt * (st["v"][r:e].double().transpose(0, 1) - torch.exp(G)[:, :, None] * (k @ S))
            D = torch.linalg.solve_triangular(A, rhs, upper=False)
            out[r:e] = (torch.exp(G)[:, :, None] * (q @ S) + (ratio * (q @ k.transpose(1, 2))) @ D).transpose(0, 1)
            S = torch.exp(G[:, -1])[:, None, None] * S + k.transpose(1, 2) @ (torch.exp(G[:, -1:] - G)[:, :, None] * D)
        pool[to[b]] = S
        r0 += m
    if st["out"] is None:
        return {"state": pool}
    if st["norm"] is not None:
        z = st["z"].double()
        out = out / torch.sqrt((out * out).mean(-1, keepdim=True) + EPS) * st["norm"].double() / (1 + torch.exp(-z))
    return {"out": out, "state": pool}


def _exact_logprob(st):
    res = {"logprob": [], "rank": [], "entropy": [], "top_ids": [], "top_logprobs": []}
    n = st["case"]["top"]
    for r, token in enumerate(st["tokens"].tolist()):
        lg = st["logits"][r].double()
        T = 1.0 if st["temperature"] is None else st["temperature"][r].double()
        order = torch.argsort(lg, descending=True, stable=True)
        x = (lg[order] - lg[order[0]]) / T
        s = torch.exp(x[1:]).flip(0).sum()                                          # (smallest first)
        lp = x - torch.log1p(s)
        place = int((order == token).nonzero()[0, 0])
        res["logprob"].append(lp[place])
        res["rank"].append(torch.tensor(place, dtype=torch.int32, device="cuda"))
        res["entropy"].append(-(torch.exp(lp) * lp).sum())
        res["top_ids"].append(order[:n].to(torch.int32))
        res["top_logprobs"].append(lp[:n])
    return {k: torch.stack(v) for k, v in res.items()}
