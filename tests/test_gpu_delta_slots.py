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
