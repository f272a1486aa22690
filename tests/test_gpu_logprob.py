"""Log probabilities of given tokens, entropies and best alternatives against 64-bit arithmetic, at the sizes, types and rows where they can go wrong."""
import ctypes as C
import math

import numpy as np
import pytest
import torch

from tests.util import pkg

szlib, sampling = pkg.lib, pkg.sampling
pytestmark = pytest.mark.gpu


def plain(lg, tokens, top, T):
    """By the definition, 64 bits: (logprob, rank, entropy, top ids, top logprobs, the largest |x| that weighs anything)."""
    out = []
    for r in range(lg.shape[0]):
        v = lg[r].double().numpy()
        v = np.where(np.isnan(v), -np.inf, v)
        order = np.argsort(-v, kind="stable")
        t, tok = float(T[r]), int(tokens[r])
        inside = 0 <= tok < len(v)
        place = int((v > v[tok]).sum() + ((v == v[tok]) & (np.arange(len(v)) < tok)).sum()) if inside else -1
        if not t > 0 or not np.isfinite(1 / np.float32(t)) or not np.isfinite(v[order[0]]):
            lp = np.where(np.arange(len(v)) == 0, 0.0, -np.inf)
            ent = 0.0
        else:
            x = (v[order] - v[order[0]]) / t
            w = np.exp(x)
            lp = x - np.log1p(w[1:][::-1].sum())
            ent = float(-(w[w > 0] / w.sum() * lp[w > 0]).sum())
        n = min(top, len(v))
        ids = np.concatenate([order[:n], np.full(top - n, -1)])
        best = np.concatenate([lp[:n], np.full(top - n, -np.inf)])
        out.append((lp[place] if inside else -np.inf, place, ent, ids, best))
    return out


def close(got, want):
    """x is a difference and a product in f32 (3 half steps), the sum s of up to 2^18 weights has terms off by 2^-21 of themselves (exponential 2^-22, exponent 3 half
    steps of up to 16 that matter: a weight e^-16 of 2^18 is the most that counts) and partial sums of at most 1,024 terms a thread: below 2^-14
    relative in the worst order, 2^-18 with roundings either way; log1p(s) is off by as much at most, and 2^-22 of itself."""
    if not math.isfinite(np.float32(want)):
        return got == np.float32(want)
    return abs(got - want) <= 2.0 ** -17 * min(1.0, abs(want)) + 2.0 ** -21 * abs(want) + 2.0 ** -30


def check(lg, tokens, top=5, T=None, out=None, **kw):
    rows = lg.shape[0]
    x = lg if lg.is_cuda else lg.cuda()
    tok = torch.as_tensor(np.asarray(tokens), dtype=torch.int32).cuda()
    t = None if T is None else torch.as_tensor(np.asarray(T), dtype=torch.float32).cuda()
    res = sampling.logprob_rows(x, tok, top=top, temperature=t, out=out)
    lp, rank, ent, ids, best = (y.cpu().numpy() for y in res)
    for r, (wl, wr, we, wi, wb) in enumerate(plain(x.cpu(), np.asarray(tokens), top, np.ones(rows) if T is None else np.asarray(T, dtype=np.float32))):
        assert rank[r] == wr, (r, rank[r], wr)
        assert close(lp[r], wl), (r, lp[r], wl)
        assert close(ent[r], we), (r, ent[r], we)
        assert list(ids[r]) == list(wi), (r, ids[r], wi)
        assert all(close(a, b) for a, b in zip(best[r], wb)), (r, best[r], wb)
    return res


@pytest.mark.parametrize("vocab", [1, 2, 31, 1000, 1025, 4097, 16385, 32003, 151936, 262144])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_sizes_and_types(vocab, dtype):
    rng = np.random.default_rng(vocab)
    rows = 9
    lg = torch.from_numpy(rng.normal(size=(rows, vocab)).astype(np.float32) * 2.5).to(dtype)
    tokens = rng.integers(0, vocab, rows)
    tokens[0], tokens[1], tokens[2], tokens[3] = 0, vocab - 1, -1, vocab
    tokens[4] = int(lg[4].float().argmax())
    check(lg, tokens, top=20, T=rng.uniform(0.2, 1.6, rows))
    check(lg, tokens, top=5)


@pytest.mark.parametrize("top", [0, 1, 2, 17, 63, 64])
@pytest.mark.parametrize("vocab", [40, 5000, 151936])
def test_numbers_of_alternatives(top, vocab):
    rng = np.random.default_rng(top)
    lg = torch.from_numpy(rng.normal(size=(5, vocab)).astype(np.float32))
    check(lg, rng.integers(0, vocab, 5), top=top)


@pytest.mark.parametrize("rows", [1, 3, 150, 700])
def test_numbers_of_rows(rows):
    """.. and so of blocks a row."""
    rng = np.random.default_rng(rows)
    lg = torch.from_numpy(rng.normal(size=(rows, 20011)).astype(np.float32) * 3)
    check(lg, rng.integers(0, 20011, rows), top=3)


@pytest.mark.parametrize("vocab", [90, 700, 5000, 151936])
@pytest.mark.parametrize("rows", [1, 8, 400])
def test_equal_logits_and_masked_rows(vocab, rows):
    """The ids decide, lowest first, however many are equal; a mask may leave fewer than are asked for."""
    rng = np.random.default_rng(vocab)
    lg = torch.zeros(rows, vocab)
    for r in range(rows):
        k = r % 6
        if k == 1:
            lg[r] = torch.from_numpy(rng.integers(0, 3, vocab).astype(np.float32))
        if k == 2:
            lg[r] = -math.inf
            lg[r, rng.integers(0, vocab, 3)] = torch.tensor([1.0, 2.0, 2.0])
        if k == 3:
            lg[r] = torch.finfo(torch.float32).min
            lg[r, vocab // 2] = 5.0
        if k == 4:
            lg[r] = torch.from_numpy(np.sort(rng.normal(size=vocab)).astype(np.float32)) * (1 if r % 12 == 4 else -1)
        if k == 5:
            lg[r, ::2] = -0.0
    if rows == 400:
        lg = lg[:, :min(vocab, 5000)].contiguous()
    tokens = rng.integers(0, lg.shape[1], rows)
    check(lg, tokens, top=30)
    check(lg.bfloat16(), tokens, top=1)


def test_infinities_nan_and_no_temperature():
    rng = np.random.default_rng(4)
    lg = torch.from_numpy(rng.normal(size=(14, 3001)).astype(np.float32))
    lg[0, 5] = lg[0, 9] = math.inf
    lg[1] = -math.inf
    lg[2] = math.nan
    lg[3, ::2] = math.nan
    lg[4, 100:] = -math.inf
    lg[5, :] = -math.inf
    lg[5, 2999] = -3.0
    lg[6] = -3e38
    lg[6, 17] = 3e38
    lg[11, 7] = 40.0                                     # a token that weighs all but 10^-14
    lg[12, 7] = math.nan
    T = np.ones(14)
    T[7], T[8], T[9], T[10], T[13] = 0.0, -1.0, math.nan, 1e30, 1e-42
    tokens = np.array([9, 0, 3, 2, 50, 2999, 17, 1, 2, 3, 4, 7, 7, 5])
    check(lg, tokens, top=5, T=T)
    check(lg, np.array([5, 7, 0, 1, 100, 1, 16, int(lg[7].argmax()), 0, 0, 0, 8, 8, int(lg[13].argmax())]), top=64, T=T)


def test_a_probability_next_to_one_keeps_its_distance():
    """The largest is not in the sum of the others: log p = -log1p(s) with s to 2^-17 of itself, whatever its size."""
    for dtype in (torch.float32, torch.bfloat16):
        lg = torch.zeros(4, 50000, dtype=dtype)
        for r, top in enumerate((20.0, 28.0, 36.0, 44.0)):
            lg[r, 31 + 9000 * r] = top
        res = sampling.logprob_rows(lg.cuda(), torch.tensor([31, 9031, 18031, 27031], dtype=torch.int32).cuda())
        s = 49999 * np.exp(-np.array([20.0, 28.0, 36.0, 44.0]))
        assert np.all(np.abs(res.logprob.cpu().numpy() + np.log1p(s)) <= 2.0 ** -17 * s)
        want = np.log1p(s) + s * np.array([20.0, 28.0, 36.0, 44.0]) / (1 + s)
        assert np.all(np.abs(res.entropy.cpu().numpy() - want) <= 2.0 ** -16 * want)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("offset", [0, 1, 3])
def test_rows_that_begin_anywhere(dtype, offset):
    """Odd strides and starts: rows begin and end inside 16 bytes, and what lies beside them is not theirs."""
    rng = np.random.default_rng(offset)
    wide = torch.full((6, 5003 + 11), 1e4, dtype=dtype)
    wide[:, offset:offset + 5003] = torch.from_numpy(rng.normal(size=(6, 5003)).astype(np.float32)).to(dtype)
    view = wide.cuda()[:, offset:offset + 5003]
    tokens = torch.from_numpy(rng.integers(0, 5003, 6)).int()
    check(view, tokens.numpy(), top=8)


def test_a_row_alone_and_in_a_batch():
    """Ranks and alternatives do not depend on the other rows, and what is not wanted is not needed."""
    rng = np.random.default_rng(0)
    lg = torch.from_numpy(rng.normal(size=(300, 32003)).astype(np.float32)).cuda()
    tok = torch.from_numpy(rng.integers(0, 32003, 300)).int().cuda()
    all_ = sampling.logprob_rows(lg, tok, top=10)
    again = sampling.logprob_rows(lg, tok, top=10)
    for a, b in zip(all_, again):
        assert torch.equal(a, b)
    one = sampling.logprob_rows(lg[7:8], tok[7:8], top=10)
    assert torch.equal(one.rank, all_.rank[7:8]) and torch.equal(one.top_ids, all_.top_ids[7:8])
    none = sampling.logprob_rows(lg, top=10)
    assert none.logprob is None and none.rank is None and torch.equal(none.top_ids, all_.top_ids) and torch.equal(none.entropy, all_.entropy)
    only = sampling.logprob_rows(lg, tok, out=sampling.LogProbs(torch.zeros(300, device="cuda"), None, None, None, None))
    assert torch.equal(only.logprob, all_.logprob)


def test_the_sampler_and_the_score_agree():
    """The probability that a draw from the whole distribution reports is the one that its token scores, but for the candidates that a sampler drops."""
    rng = np.random.default_rng(1)
    lg = torch.from_numpy(rng.normal(size=(40, 32003)).astype(np.float32)).cuda()
    T = torch.full((40,), 0.9, device="cuda")
    prob = torch.zeros(40, device="cuda")
    tok = sampling.sample_rows(lg, torch.rand(40, dtype=torch.float64, device="cuda"), temperature=T, prob=prob)
    res = sampling.logprob_rows(lg, tok, temperature=T)
    # dropped: at most 32,003 candidates of e^-18 of the largest, 5e-4 of the sum at most; normal logits of T 0.9 reach 9 below, so none here
    assert float((res.logprob - prob.log()).abs().max()) < 2.0 ** -16


def test_capture_and_other_streams():
    rng = np.random.default_rng(2)
    lg = torch.from_numpy(rng.normal(size=(20, 151936)).astype(np.float32)).cuda()
    tok = torch.from_numpy(rng.integers(0, 151936, 20)).int().cuda()
    want = sampling.logprob_rows(lg, tok, top=20)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = sampling.logprob_rows(lg, tok, top=20)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            sampling.logprob_rows(lg, tok, top=20, out=got)
        other = torch.from_numpy(rng.normal(size=(20, 151936)).astype(np.float32)).cuda()
        lg.copy_(other)
        graph.replay()
    side.synchronize()
    again = sampling.logprob_rows(lg, tok, top=20)
    assert all(torch.equal(a, b) for a, b in zip(got, again)) and not torch.equal(got.logprob, want.logprob)
