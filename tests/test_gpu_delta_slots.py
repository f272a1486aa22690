"""The convolution of a served step in place: a sequence's carried rows are read and written in one slot, whatever blocks its rows belong to and whatever else runs."""
import pytest
import torch

from tests.test_gpu_delta import Case

pytestmark = pytest.mark.gpu


def in_place(counts, past, times=12, **kw):
    """Results against 64 bits; then, with the multiprocessors kept busy from a second stream, the same bits every time."""
    c, busy = Case(counts, past, **kw), torch.cuda.Stream()
    before = c.carried.clone()
    want = c.check_conv()
    after = c.carried.clone()
    a = torch.randn(2048, 2048, device="cuda", dtype=torch.bfloat16)
    b = torch.empty_like(a)
    torch.cuda.synchronize()
    for i in range(times):
        c.carried.copy_(before)
        y = torch.full_like(c.x, 77.0)
        busy.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(busy):
            for _ in range(1 + i % 3):
                torch.matmul(a, a, out=b)
        c.step.conv(c.x, c.w, bias=c.bias, out=y)
        assert torch.equal(y, want) and torch.equal(c.carried, after), i
    torch.cuda.synchronize()
    assert c.step.status() == 0


@pytest.mark.parametrize("conv_k", [2, 3, 4, 5, 6, 7, 8])
def test_few_rows_of_one_sequence(conv_k):
    for rows in range(2, 2 * conv_k + 1):
        in_place([rows], [9], kh=16, vh=32, d=128, io="bf16", conv_k=conv_k, times=4, seed=rows)


@pytest.mark.parametrize("conv_k", [2, 3, 4, 8])
@pytest.mark.parametrize("rows, n", [(3, 20), (9, 15), (33, 40)])
def test_a_sequence_begins_at_every_place_of_a_tile(conv_k, rows, n):
    """(Tiles of 1, 2 and 32 rows of these channels; sequences of one row more than a power of two begin at each of their places.)"""
    in_place([rows] * n, [5 * (i % 3) for i in range(n)], kh=16, vh=32, d=128, io="bf16", conv_k=conv_k, pad=3)


@pytest.mark.parametrize("io", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("max_rows", [None, 9])
def test_drafts_of_a_batch(io, max_rows):
    """64 conversations of up to 4 rows, of which nothing was said, or too much; and what is kept of them, again."""
    counts, past = [1 + (i * 7) % 4 for i in range(64)], [3 + i for i in range(64)]
    in_place(counts, past, kh=16, vh=32, d=128, io=io, max_rows=max_rows)
    in_place(counts, past, kh=16, vh=32, d=128, io=io, max_rows=max_rows, take=[1 + i % m for i, m in enumerate(counts)])


def test_prompts_that_go_on():
    in_place([1, 30, 1, 700, 2, 63, 64, 3, 400], [7] * 9, kh=16, vh=32, d=128, io="bf16")


@pytest.mark.parametrize("rows", [3, 80])
@pytest.mark.parametrize("slots, to, past, starts, out", [
    ((1, 2, 3), (-1, 2, 3), (5, 0, 5), None, (0,)),                  # goes nowhere; the next one is new and comes from nowhere
    ((-1, 2, 3), (-1, 2, 3), (5, 0, 0), None, (0,)),
    ((1, 2, 1), (2, 99, 1), (0, 5, 5), None, (1,)),                  # reads what the first writes, besides
    ((99, 4, 2), (4, 4, 2), (5, 5, 5), None, (0,)),                  # would write where the next one goes on
    ((1, 2, 1), (1, 2, 1), (5, 5, 5), -4, (0,)),                     # rows out of range, in the slot of another
])
def test_a_sequence_that_does_not_fit_takes_no_other_with_it(rows, slots, to, past, starts, out):
    """The others' results are those beside a sequence that fits."""
    for call in ("conv", "rule"):
        c = Case([rows] * 3, list(past), d=64, io="f32", slots=list(slots), to=list(to), n_slots=6, seed=4)
        ref = Case([rows] * 3, list(past), d=64, io="f32",
                   slots=[5 if b in out else x for b, x in enumerate(slots)], to=[5 if b in out else x for b, x in enumerate(to)], n_slots=6, seed=4)
        if starts is not None:
            c.row_start[0] = starts
        wrong = 1 if starts is None else 2
        got, want = (torch.full((s.rows, s.ch) if call == "conv" else (s.rows, s.vh, s.d), 77.0, device="cuda") for s in (c, ref))
        for s, y in ((c, got), (ref, want)):
            if call == "conv":
                s.step.conv(s.x, s.w, out=y)
            else:
                s.run(y)
        assert c.step.status() == wrong and ref.step.status() == 0
        for b in range(3):
            cut = slice(rows * b, rows * b + rows)
            if b in out:
                assert bool((got[cut] == 77).all())
            else:
                assert torch.equal(got[cut], want[cut]) and bool((got[cut] != 77).any())
                assert torch.equal(c.state[c.to[b]], ref.state[ref.to[b]]) and torch.equal(c.carried[c.to[b]], ref.carried[ref.to[b]])


def test_weights_that_the_kernel_before_writes():
    """`conv(x, weight.float(), ..)`, again and again: weights, bias and rows are those that are there when the call's turn comes."""
    c = Case([3, 1], [9, 4], kh=16, vh=32, d=128, io="bf16", fork=True)
    half, bias = c.w.bfloat16(), c.bias.bfloat16()
    w, b = torch.zeros_like(c.w), torch.zeros_like(c.bias)
    got = []
    for i in range(40):
        w.copy_(half * (i + 1))
        b.copy_(bias * (i - 7))
        got.append(c.step.conv(c.x, w, bias=b))
    for i, y in enumerate(got):
        w, b = (half * (i + 1)).float(), (bias * (i - 7)).float()
        torch.cuda.synchronize()
        assert torch.equal(y, c.step.conv(c.x, w, bias=b)), i
    assert c.step.status() == 0


@pytest.mark.parametrize("dtype", [torch.float64, torch.int32])
def test_rows_of_other_types_are_refused(dtype):
    """By a ValueError, as everything that does not fit, and before anything runs."""
    c = Case([3], [0], d=64, io="f32")
    state, carried = c.state.clone(), c.carried.clone()
    to = lambda *ts: [t.to(dtype) for t in ts]  # noqa: E731
    with pytest.raises(ValueError, match="float32, float16 or bfloat16"):
        c.step.conv(c.x.to(dtype), c.w)
    with pytest.raises(ValueError, match="float32, float16 or bfloat16"):
        c.step.rule(*to(c.q, c.k, c.v, c.alpha, c.beta), c.a, c.dt)
    with pytest.raises(ValueError, match="float32, float16 or bfloat16"):
        c.step.replay(*to(c.k, c.v, c.alpha, c.beta), c.a, c.dt)
    with pytest.raises(ValueError, match="float32, float16 or bfloat16"):
        c.step.rule(c.q, c.k, c.v.to(dtype), c.alpha, c.beta, c.a, c.dt)
    assert torch.equal(c.state, state) and torch.equal(c.carried, carried) and c.step.status() == 0
