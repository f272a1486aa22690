"""Draws over whole rows of logits against the oracle's Sampler::sample (a full sort in 64 bits) and against a plain restatement, and where they can go
wrong: ties, one candidate, thousands of equal logits, infinities and NaN, every row with its own settings, odd widths and strides."""
import ctypes as C
import math

import numpy as np
import pytest
import torch

from oracle import binding as ob
from tests.util import pkg

szlib, sampling = pkg.lib, pkg.sampling
pytestmark = pytest.mark.gpu


def plain(v, T, k, p, mp, u):
    """One row by the definition; returns (token, its probability, how near u was to another token's range, relative)."""
    v = np.where(np.isnan(v), -np.inf, v).astype(np.float32)
    top = v.max()
    if not np.isfinite(top) or not T > 0:
        return int(np.argmax(v == top)), 1.0, 1.0
    ids = np.argsort(-v, kind="stable")
    s = v[ids]
    n = min(int((s >= top - np.float32(18) * np.float32(T)).sum()), max(int(k), 1))
    w = np.exp(((s[:n] - top) * (np.float32(1) / np.float32(T))).astype(np.float64))
    Z = w.sum()
    keep = max(1, int((w >= np.float64(np.float32(mp))).sum()))
    if p < 1:
        keep = min(keep, int((np.cumsum(w) < np.float64(np.float32(p)) * Z).sum()) + 1)
    w = w[:keep]
    c = np.cumsum(w)
    i = min(int((c <= u * c[-1]).sum()), keep - 1)
    return int(ids[i]), float(w[i] / c[-1]), float(np.min(np.abs(c - u * c[-1])) / c[-1])


def check(lg, T, k, p, mp, u, **kw):
    rows = lg.shape[0]
    d = lambda x, t: torch.as_tensor(np.asarray(x), dtype=t).cuda()  # noqa: E731
    prob = torch.zeros(rows, device="cuda")
    x = lg.cuda()
    tok = sampling.sample_rows(x, d(u, torch.float64), temperature=d(T, torch.float32), top_k=d(k, torch.int32), top_p=d(p, torch.float32), min_p=d(mp, torch.float32), prob=prob, **kw)
    tok, prob = tok.cpu().numpy(), prob.cpu().numpy()
    host = lg.float().numpy()
    for r in range(rows):
        want, wp, near = plain(host[r], T[r], k[r], p[r], mp[r], u[r])
        # (weights are held to 2^-45 of the largest: a draw within 2^-30 of a border is not decided by the definition's own rounding)
        assert tok[r] == want or near < 2.0 ** -30, "row %d: %d, not %d" % (r, tok[r], want)
        # (a weight is 1.5e-8 of the largest at least: 2^-46 of it is 2e-6 of that)
        assert tok[r] != want or abs(prob[r] - wp) <= (2.0 ** -23 + 2e-6) * wp, (r, prob[r], wp)
    return tok


def settings(rng, rows, vocab):
    T = rng.uniform(0.1, 1.6, rows)
    k = np.where(rng.random(rows) < 0.5, (2 ** rng.uniform(0, 14, rows)).astype(np.int64), vocab)
    p = np.where(rng.random(rows) < 0.6, rng.uniform(0.05, 1.0, rows), 1.0)
    mp = np.where(rng.random(rows) < 0.4, rng.uniform(0.0, 0.3, rows), 0.0)
    return T, k, p, mp, rng.random(rows)


@pytest.mark.parametrize("vocab", [1, 2, 31, 1000, 1025, 4097, 16385, 32003, 151936, 262144])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_rows_with_settings_of_their_own(vocab, dtype):
    rng = np.random.default_rng(vocab)
    rows = 24
    lg = torch.from_numpy(rng.normal(size=(rows, vocab)).astype(np.float32) * 2.5).to(dtype)
    check(lg, *settings(rng, rows, vocab))


@pytest.mark.parametrize("rows", [1, 7, 200])
def test_numbers_of_rows(rows):
    rng = np.random.default_rng(rows)
    lg = torch.from_numpy(rng.normal(size=(rows, 20011)).astype(np.float32) * 3)
    check(lg, *settings(rng, rows, 20011))


@pytest.mark.parametrize("u", [0.0, 1e-300, 0.25, 0.5, 1 - 2.0 ** -53])
def test_ends_of_the_unit_interval(u):
    rng = np.random.default_rng(5)
    lg = torch.from_numpy(rng.normal(size=(6, 5000)).astype(np.float32))
    T, k, p, mp, _ = settings(rng, 6, 5000)
    check(lg, T, k, p, mp, np.full(6, u))


@pytest.mark.parametrize("vocab", [700, 5000, 151936])
def test_equal_logits(vocab):
    """Thousands of candidates of one weight: the ids decide, lowest first."""
    rng = np.random.default_rng(vocab)
    rows = 16
    lg = torch.zeros(rows, vocab)
    lg[4:8] = torch.from_numpy(rng.integers(0, 3, (4, vocab)).astype(np.float32))
    lg[8:12] = torch.from_numpy(rng.integers(0, 40, (4, vocab)).astype(np.float32) * 2.0 ** -12)       # thousands in a bin, forty values
    lg[12:] = torch.from_numpy(rng.random((4, vocab)).astype(np.float32) * 2.0 ** -9)                   # thousands in a bin, all different
    T, k, p, mp, u = settings(rng, rows, vocab)
    check(lg, T, k, p, mp, u)
    k = np.full(rows, vocab)
    tok = check(lg, np.ones(rows), k, np.ones(rows), np.zeros(rows), u)
    assert list(tok[:4]) == [int(u[r] * vocab) for r in range(4)]
    check(lg, np.ones(rows), np.minimum(k, 3000), np.full(rows, 0.7), np.zeros(rows), u)
    check(lg, np.ones(rows), k, np.full(rows, 0.7), np.ones(rows), u)


def test_top_k_alone():
    rng = np.random.default_rng(3)
    lg = torch.from_numpy(rng.normal(size=(40, 9000)).astype(np.float32) * 4)
    k = np.array([-5, 0, 1, 2, 3, 5, 8, 64, 1000, 1023, 1024, 1025, 4000, 8999, 9000, 9001, 2 ** 31 - 1] + [17] * 23)
    check(lg, np.full(40, 0.8), k, np.ones(40), np.zeros(40), rng.random(40))


def test_infinities_nan_and_no_temperature():
    rng = np.random.default_rng(4)
    lg = torch.from_numpy(rng.normal(size=(12, 3001)).astype(np.float32))
    lg[0, 5] = lg[0, 9] = math.inf
    lg[1] = -math.inf
    lg[2] = math.nan
    lg[3, ::2] = math.nan
    lg[4, 100:] = -math.inf
    lg[5, :] = -math.inf
    lg[5, 2999] = -3.0
    lg[6] = -3e38
    lg[6, 17] = 3e38
    T, k, p, mp, u = settings(rng, 12, 3001)
    T[7], T[8], T[9], T[10], T[11] = 0.0, -1.0, 1e-42, 1e30, 3e38
    k[10:] = 3001
    p[10:] = 1
    d = lambda x, t: torch.as_tensor(x, dtype=t).cuda()  # noqa: E731
    prob = torch.zeros(12, device="cuda")
    tok = sampling.sample_rows(lg.cuda(), d(u, torch.float64), temperature=d(T, torch.float32), top_k=d(k, torch.int32), top_p=d(p, torch.float32), min_p=d(mp, torch.float32), prob=prob).cpu().numpy()
    host = lg.numpy()
    assert tok[0] == 5 and tok[1] == 0 and tok[2] == 0 and tok[5] == 2999 and tok[6] == 17
    assert tok[3] % 2 == 1 and tok[4] < 100
    for r in (7, 8, 9):
        assert tok[r] == int(host[r].argmax()) and float(prob[r]) == 1.0
    for r in (10, 11):                                   # so hot that all weigh the same: the order is that of the logits, still
        order = np.argsort(-host[r], kind="stable")
        assert tok[r] == order[int(u[r] * 3001)]
    check(lg[[3, 4, 5, 6]], T[[3, 4, 5, 6]], k[[3, 4, 5, 6]], p[[3, 4, 5, 6]], mp[[3, 4, 5, 6]], u[[3, 4, 5, 6]])


def test_defaults_and_strides():
    rng = np.random.default_rng(6)
    wide = torch.from_numpy(rng.normal(size=(9, 2049)).astype(np.float32)).cuda()
    u = torch.from_numpy(rng.random(9)).cuda()
    for a, b in ((0, 2048), (1, 2049), (3, 1777)):       # rows that begin anywhere
        x = wide[:, a:b]
        tok = sampling.sample_rows(x, u)
        assert torch.equal(tok, sampling.sample_rows(x.contiguous(), u))
        host = x.cpu().numpy()
        for r in range(9):
            want, _, near = plain(host[r], 1.0, 2 ** 30, 1.0, 0.0, float(u[r]))
            assert int(tok[r]) == want or near < 2.0 ** -30


def test_the_host_samplers_draw():
    """Where 64 candidates are all there are, the token is sz_sample_top's for the same seed and position."""
    rng = np.random.default_rng(7)
    L = szlib.load()
    rows, vocab = 50, 32000
    lg = torch.from_numpy(rng.normal(size=(rows, vocab)).astype(np.float32) * 2).cuda()
    for T, k, p, mp in ((0.7, 40, 0.9, 0.0), (1.2, 64, 1.0, 0.05), (0.3, 5, 0.5, 0.0)):
        raw = (C.c_uint8 * 24)()
        np.frombuffer(raw, dtype=np.uint8)[:] = np.frombuffer(np.float32(T).tobytes() + np.int32(k).tobytes() + np.float32(p).tobytes() + np.float32(mp).tobytes() + np.uint64(99).tobytes(), dtype=np.uint8)
        u = torch.tensor([L.sz_uniform(99, r) for r in range(rows)], dtype=torch.float64).cuda()
        full = lambda x, t=torch.float32: torch.full((rows,), x, dtype=t, device="cuda")  # noqa: E731
        tok = sampling.sample_rows(lg, u, temperature=full(T), top_k=full(k, torch.int32), top_p=full(p), min_p=full(mp)).cpu().numpy()
        v, i = torch.sort(lg, dim=1, descending=True, stable=True)
        top = np.concatenate([v[:, :64].cpu().numpy().view(np.uint32), i[:, :64].cpu().numpy().astype(np.uint32)], 1)
        for r in range(rows):
            row = np.ascontiguousarray(top[r])
            assert int(tok[r]) == L.sz_sample_top(C.cast(raw, C.c_void_p), row.ctypes.data_as(C.POINTER(C.c_uint32)), r)


def test_distribution():
    """A million draws from six tokens: each count within five deviations of its expectation."""
    p = np.array([0.5, 0.2, 0.15, 0.1, 0.04, 0.01])
    n = 1 << 20
    lg = torch.from_numpy(np.log(p).astype(np.float32)).cuda().expand(n, 6).contiguous()
    u = (torch.arange(n, dtype=torch.float64, device="cuda") + 0.5) / n
    tok = sampling.sample_rows(lg, u)
    got = torch.bincount(tok.long(), minlength=6).cpu().numpy()
    assert np.abs(got - p * n).max() < 5 * math.sqrt(n * 0.25)


def test_a_captured_call():
    rng = np.random.default_rng(8)
    lg, u = torch.from_numpy(rng.normal(size=(5, 40000)).astype(np.float32)).cuda(), torch.from_numpy(rng.random(5)).cuda()
    out = torch.zeros(5, dtype=torch.int32, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        sampling.sample_rows(lg, u, out=out)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        sampling.sample_rows(lg, u, out=out)
    for _ in range(3):
        lg.copy_(torch.from_numpy(rng.normal(size=(5, 40000)).astype(np.float32)))
        u.copy_(torch.from_numpy(rng.random(5)))
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, sampling.sample_rows(lg, u))


@pytest.mark.parametrize("rows,vocab,dtype", [(300, 40001, torch.bfloat16), (100, 100003, torch.float32), (64, 70002, torch.float16), (37, 262143, torch.float32)])
def test_rows_in_fewer_blocks(rows, vocab, dtype):
    """Many rows: one to four blocks a row, whose parts do not fit shared memory and begin at any element."""
    rng = np.random.default_rng(rows + vocab)
    lg = torch.from_numpy(rng.normal(size=(rows, vocab)).astype(np.float32) * 2.5).to(dtype)
    T, k, p, mp, u = settings(rng, rows, vocab)
    lg[3] = -math.inf
    lg[4, 5:] = math.nan
    check(lg, T, k, p, mp, u)


def test_most_equal_logits_in_one_block():
    """262,144 members of one bin in one block: its count and its sum fill their bits."""
    rows, vocab = 300, 262144
    lg = torch.zeros(rows, vocab, dtype=torch.float16, device="cuda")
    u = torch.rand(rows, dtype=torch.float64, generator=torch.Generator().manual_seed(8))
    u[0], u[1] = 0.0, 1 - 2.0 ** -53
    assert torch.equal(sampling.sample_rows(lg, u.cuda()).cpu(), (u * vocab).to(torch.int32))
    lg[:, ::2] = -2.0 ** -9                      # (less than half a bin: two weights in one)
    tok = sampling.sample_rows(lg, u.cuda()).cpu().numpy()
    w = np.where(np.arange(vocab) % 2 == 1, 1.0, math.exp(-2.0 ** -9))
    order = np.concatenate([np.arange(1, vocab, 2), np.arange(0, vocab, 2)])
    c = np.cumsum(w[order])
    for r in range(rows):
        goal = float(u[r]) * c[-1]
        assert tok[r] == order[min(int((c <= goal).sum()), vocab - 1)] or np.abs(c - goal).min() < 2.0 ** -30 * c[-1], r


def test_zeros_of_both_signs_are_equal():
    """0 and -0 are one logit: the lower id first, whichever it is; a reading of the bits would put every 0 before every -0."""
    tok = check(torch.tensor([[-0.0, 0.0]]), np.ones(1), np.ones(1, dtype=np.int64), np.ones(1), np.zeros(1), np.array([0.5]))
    assert tok[0] == 0
    for vocab, dtype in ((7, torch.float32), (700, torch.bfloat16), (5000, torch.float16), (40001, torch.float32)):
        rng = np.random.default_rng(vocab)
        rows = 12
        lg = torch.from_numpy(np.where(rng.random((rows, vocab)) < 0.5, np.float32(-0.0), np.float32(0.0))).to(dtype)
        lg[6:] = torch.where(torch.from_numpy(rng.random((6, vocab)) < 0.3), torch.tensor(-1.0, dtype=dtype), lg[6:])
        u = rng.random(rows)
        tok = check(lg, np.ones(rows), np.full(rows, vocab), np.ones(rows), np.zeros(rows), u)
        assert list(tok[:6]) == [int(u[r] * vocab) for r in range(6)]
        T, k, p, mp, u = settings(rng, rows, vocab)
        check(lg, T, k, p, mp, u)


@pytest.mark.parametrize("vocab", [3, 1000, 32003, 151936])
def test_the_oracles_draws(vocab):
    """The oracle's Sampler::sample over whole rows, from the same seed and position.  Its sums are f64 one after the other: vocab 2^-53 of them, far below the
    2^-30 from a border that check() allows."""
    oracle = ob.lib()
    rng = np.random.default_rng(vocab + 1)
    rows = 32
    lg = torch.from_numpy(rng.normal(size=(rows, vocab)).astype(np.float32) * 2.5)
    lg[5] = torch.round(lg[5])                                     # many equal ones, both zeros among them
    T, k, p, mp, _ = settings(rng, rows, vocab)
    k = np.minimum(k, vocab)
    u = np.array([oracle.szo_uniform(7, r) for r in range(rows)])
    tok = check(lg, T, k, p, mp, u)
    host = lg.numpy()
    for r in range(rows):
        raw = (np.float32(T[r]).tobytes() + np.int32(k[r]).tobytes() + np.float32(p[r]).tobytes() + np.float32(mp[r]).tobytes() + np.uint64(7).tobytes())
        row = np.ascontiguousarray(host[r])
        want = oracle.szo_sample(C.cast(C.create_string_buffer(raw, 24), C.c_void_p), row.ctypes.data_as(C.c_void_p), vocab, r)
        assert int(tok[r]) == int(want) or plain(host[r], T[r], k[r], p[r], mp[r], u[r])[2] < 2.0 ** -30, r


@pytest.mark.parametrize("rows,vocab,dtype", [(250, 60001, torch.bfloat16), (64, 151936, torch.float32), (3, 40000, torch.float32)])
def test_logits_that_change_underneath(rows, vocab, dtype):
    """Another stream writes the rows while they are drawn from, values far above the largest that the call has seen among them: every call ends, with tokens of
    the vocabulary, and the next one over logits at rest is right."""
    g = torch.Generator(device="cuda").manual_seed(rows)
    rest = (2.5 * torch.randn(rows, vocab, device="cuda", generator=g)).to(dtype)
    other = [(rest.float() * 10 + 100).to(dtype), torch.full_like(rest, math.inf), torch.full_like(rest, math.nan), (rest.float() * 1e30).to(dtype), torch.full_like(rest, -math.inf), rest]
    u = torch.rand(rows, dtype=torch.float64, device="cuda", generator=g)
    p = torch.full((rows,), 0.9, device="cuda")
    want = sampling.sample_rows(rest, u, top_p=p)
    lg, side, got = rest.clone(), torch.cuda.Stream(), []
    side.wait_stream(torch.cuda.current_stream())
    for i in range(40):
        with torch.cuda.stream(side):
            for x in other:
                lg.copy_(x)
        got.append(sampling.sample_rows(lg, u, top_p=p))
        got.append(sampling.sample_rows(lg, u))
    torch.cuda.synchronize()
    for t in got:
        assert bool(((t >= 0) & (t < vocab)).all())
    lg.copy_(rest)
    assert torch.equal(sampling.sample_rows(lg, u, top_p=p), want)
