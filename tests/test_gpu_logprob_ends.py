"""Log probabilities at the ends of what a temperature may be."""
import math

import pytest
import torch

from tests.util import pkg

sampling = pkg.sampling
pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [2, 300])
def test_an_infinite_temperature_leaves_masked_tokens_out(rows):
    """All that is not masked weighs the same."""
    lg = torch.full((rows, 3001), -math.inf, device="cuda")
    ids = [7, 100, 1500, 2999, 3000]
    lg[:, ids] = torch.tensor([1.0, -5.0, 300.0, 0.0, 2.0], device="cuda")
    tok = torch.tensor([100, 8] * (rows // 2), dtype=torch.int32, device="cuda")
    res = sampling.logprob_rows(lg, tok, top=8, temperature=torch.full((rows,), math.inf, device="cuda"))
    want = -math.log(5)
    assert bool(((res.logprob[::2] - want).abs() < 2.0 ** -20).all()) and bool((res.logprob[1::2] == -math.inf).all())
    assert bool(((res.entropy + want).abs() < 2.0 ** -20).all())
    assert res.top_ids[0].tolist()[:5] == [1500, 3000, 7, 2999, 100]
    assert bool(((res.top_logprobs[:, :5] - want).abs() < 2.0 ** -20).all()) and bool((res.top_logprobs[:, 5:] == -math.inf).all())


@pytest.mark.parametrize("rows", [2, 300])
@pytest.mark.parametrize("temperature", [2e-38, 5e-39, 3e-39])
def test_equal_ones_share_at_the_smallest_temperatures(rows, temperature):
    """The reciprocal is a number still, its product with log2(e) may not be one."""
    lg = torch.randn(rows, 20011, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)).clamp_max(3.0)
    ids = [3, 4, 5000, 12345, 20010]
    lg[:, ids] = 6.5
    tok = torch.tensor([12345, 6] * (rows // 2), dtype=torch.int32, device="cuda")
    res = sampling.logprob_rows(lg, tok, top=5, temperature=torch.full((rows,), temperature, device="cuda"))
    want = -math.log(5)
    assert bool(((res.logprob[::2] - want).abs() < 2.0 ** -20).all()) and bool((res.logprob[1::2] < -1e37).all())
    assert bool(((res.entropy + want).abs() < 2.0 ** -20).all())
    assert res.top_ids[0].tolist() == ids and bool(((res.top_logprobs - want).abs() < 2.0 ** -20).all())


@pytest.mark.parametrize("dtype, vocab", [(torch.float32, 90112), (torch.float32, 90113), (torch.float32, 262144), (torch.bfloat16, 180224), (torch.bfloat16, 180225), (torch.float16, 262144)])
def test_both_sides_of_the_border_between_sizes_of_blocks(dtype, vocab):
    """More rows than multiprocessors; against 64 bits, by the bound of the other sizes' test."""
    g = torch.Generator(device="cuda").manual_seed(vocab)
    lg = (3 * torch.randn(152, vocab, device="cuda", generator=g)).to(dtype)
    tok = torch.randint(0, vocab, (152,), device="cuda", generator=g).to(torch.int32)
    res = sampling.logprob_rows(lg, tok, top=20)
    order = torch.sort(lg.float(), dim=1, descending=True, stable=True)[1]
    lp = torch.log_softmax(lg.double(), 1)
    close = lambda a, b: bool(((a.double() - b).abs() <= 2.0 ** -17 * b.abs().clamp_max(1) + 2.0 ** -21 * b.abs() + 2.0 ** -30).all())  # noqa: E731
    assert torch.equal(res.top_ids, order[:, :20].int()) and torch.equal(res.rank.long(), (order == tok[:, None]).int().argmax(1))
    assert close(res.logprob, lp.gather(1, tok.long()[:, None])[:, 0]) and close(res.top_logprobs, lp.gather(1, order[:, :20])) and close(res.entropy, -(lp.exp() * lp).sum(1))
