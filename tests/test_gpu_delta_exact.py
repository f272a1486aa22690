"""What the DeltaNet layer of a served step keeps of its numbers: errors in relation to the results' own size, against plain 64-bit arithmetic."""
import math

import pytest
import torch

from tests.test_gpu_delta import Case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [20, 449])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("io", ["bf16", "f16"])
def test_outputs_of_16_bits_are_those_of_32_rounded(io, d, rows):
    """Some eight stages with roundings of 2^-22 each, of numbers up to 4 times an output: 2^-18.5 of it, root mean square.  A number that is off by e rounds to the neighbour
    of its nearest one, which is a step u away, with a probability of 2 e / u: root mean square sqrt(2 e u), u = 2^-7 (bf16) or 2^-10 at most: below 2^-12 and 2^-13.5."""
    c = Case([rows], [5], d=d, io=io, gate=False, seed=rows + d)
    want, _, _, _ = c.want_rule()
    got = c.run()
    assert c.step.status() == 0
    near = want.to(c.io).double()
    off = float((got.double() - near).square().sum().sqrt() / want.square().sum().sqrt())
    assert off <= (2.0 ** -12 if io == "bf16" else 2.0 ** -13.5), off


@pytest.mark.parametrize("io", ["bf16", "f16"])
def test_a_prompt_past_the_slab_of_heads_whose_f32_chunks_fill_it_worse(io):
    """A whole number of f32 chunks may take less of the scratch's slab than one of 16-bit chunks: the step's scratch holds either."""
    Case([16400], [3], kh=8, vh=16, d=64, io=io, grouped=True, gate=False, v_scale=0.5).check_rule()


@pytest.mark.parametrize("io", ["f32", "bf16"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("rows", [20, 300])
@pytest.mark.parametrize("gate", [-8.0, -12.0, -16.0, -40.0])
def test_changes_behind_gates_that_are_all_but_closed(io, d, rows, gate):
    """A new sequence's state is its small changes alone.  An element is a sum over rows of k (2^-23 off by its length), a change (R and T as two f16 numbers, 2^-21 in all; beta's
    exponential and quotient 2^-22; sums of 64 products 2^-22) and a decay, the exponential of a sum of up to 16 that matters (16 half steps, 2^-20): below 2^-18.5 of the column's length, sums over rows
    and chunks of errors of either sign not above that of one times 2^0.5."""
    c = Case([rows], [0], d=d, io=io, gate=False, seed=rows + d)
    c.beta.fill_(gate)
    _, _, pool, _ = c.want_rule()
    want = pool[c.to[0]]
    c.run()
    assert c.step.status() == 0
    off = (c.state[c.to[0]].double() - want).square().sum(1).sqrt() / want.square().sum(1).sqrt()
    assert float(off.max()) <= 2.0 ** -18, float(off.max())


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("rows", [20, 300])
@pytest.mark.parametrize("size", [1e-3, 1e-6, 1e-9, 1e-12])
def test_short_keys(d, rows, size):
    """Keys far below the 1e-3 that the norm adds in: states of a new sequence are as small, and as exact.  (The bound of above, and one bit for the sums of several chunks.)"""
    c = Case([rows], [0], d=d, io="f32", gate=False, seed=rows + d)
    c.k.mul_(size)
    _, _, pool, _ = c.want_rule()
    want = pool[c.to[0]]
    c.run()
    assert c.step.status() == 0
    off = (c.state[c.to[0]].double() - want).square().sum(1).sqrt() / want.square().sum(1).sqrt()
    assert float(off.max()) <= 2.0 ** -17, float(off.max())


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("rows", [20, 300])
@pytest.mark.parametrize("size", [1.0, 1e-3, 1e-6, 1e-9, 1e-12])
def test_short_queries(d, rows, size):
    """Queries as short: a row of outputs is a product of them with the state, whose columns it may turn away from.  (Errors of the above against outputs of 2^-1.5 and more of what their rows could
    be at most: 2^-15.5.)"""
    c = Case([rows], [0], d=d, io="f32", gate=False, seed=rows + d)
    c.q.mul_(size)
    want, _, _, _ = c.want_rule()
    got = c.run()
    assert c.step.status() == 0
    off = (got.double() - want).square().sum(2).sqrt() / want.square().sum(2).sqrt()
    assert float(off.max()) <= 2.0 ** -15.5, float(off.max())


ENDS = [math.inf, 3e38, 1e30, 200.0, 88.0, 87.0, 86.0, 0.0, -86.0, -87.0, -88.0, -200.0, -1e30, -3e38]


@pytest.mark.parametrize("io", ["f32", "bf16", "f16"])
def test_gates_at_the_ends_of_the_exponential(io):
    """A gate of +inf is open, of -inf shut; a NaN is one.  (Below -87 a sigmoid is less than 2^-125: 0.)"""
    for rows in (20, 200):
        c, ref = (Case([rows], [3], d=64, io=io, seed=1) for _ in range(2))
        gates = torch.tensor(ENDS + [-math.inf], dtype=torch.float64, device="cuda")
        for s in (c, ref):
            s.z[:len(gates)] = gates.to(s.io)[:, None, None]
        ref.z[:len(gates)] = 0
        half, out = ref.run().double(), c.run()
        want = half[:len(gates)] * 2 * torch.sigmoid(c.z[:len(gates), :1, :1].double())
        step = {"f32": 2.0 ** -20, "bf16": 2.0 ** -7, "f16": 2.0 ** -10}[io]           # (half a step of each of the two, and of the gates)
        assert bool(((out[:len(gates)].double() - want).abs() <= step * want.abs() + 2.0 ** -24).all())
        c.z[5] = math.nan
        out = c.run()
        assert bool(out[5].isnan().all()) and not bool(out[:5].isnan().any())


@pytest.mark.parametrize("io", ["f32", "bf16"])
@pytest.mark.parametrize("ends", [ENDS, ENDS[1:]])
def test_convolution_sums_at_the_ends_of_the_exponential(io, ends):
    """x sigmoid(x) of x: x itself, or nothing.  (An infinite row times a weight of 0 is a NaN, in the sums of the rows behind it, too.)"""
    n = len(ends)
    c = Case([n, 1], [0, 0], kh=1, vh=1, d=64, io=io)
    x = torch.tensor(ends, dtype=torch.float64, device="cuda").to(c.io)
    c.x[:n] = x[:, None]
    c.x[n] = math.nan
    c.w.fill_(0)
    c.w[:, -1] = 1
    y = c.step.conv(c.x, c.w).double()
    s = (torch.cat([torch.zeros(3, dtype=torch.float64, device="cuda"), x.double()]).unfold(0, 4, 1) * c.w[0].double()).sum(1)
    want = (s * torch.sigmoid(s))[:, None].expand(n, c.ch)
    assert bool(y[n].isnan().all()) and torch.equal(y[:n].isnan(), want.isnan()) and torch.equal(y[:n].isinf(), want.isinf())
    fine = want.isfinite()
    off = (y[:n] - want).abs()
    assert bool((off <= (2.0 ** -20 if io == "f32" else 2.0 ** -8) * want.abs() + 2.0 ** -118)[fine].all()), off.max(1)


@pytest.mark.parametrize("n, rows", [(1, 39), (1, 40), (2, 47), (2, 48), (3, 59), (3, 60), (4, 95), (4, 96), (19, 127), (19, 128)])
def test_both_sides_of_the_borders_between_rows_and_chunks(n, rows):
    Case([rows] * n, [4 * (i % 2) for i in range(n)], kh=16, vh=32, d=128, io="bf16", seed=n).check_rule()
    if n == 2:
        Case([rows] * n, [4 * (i % 2) for i in range(n)], kh=8, vh=16, d=64, io="f16", grouped=True, seed=n).check_rule()


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("size", [1.0, 3e-3, 1e-4])
def test_the_largest_changes_there_can_be(d, size):
    """Every gate open, no decay, keys that are all alike, or one direction and its opposite in turn, values that alternate: changes are sums of values of one sign, as large as they become."""
    for flip in (False, True):
        c = Case([320], [0], d=d, kh=1, vh=2, io="f32", gate=False, seed=d)
        c.a.zero_()
        c.beta.fill_(60.0)
        key = torch.zeros(d, device="cuda")
        key[3] = size
        c.k.copy_(key.expand_as(c.k))
        if flip:
            c.k[1::2].mul_(-1)
        c.v.fill_(1.999)
        c.v[1::2].mul_(-1)
        c.check_rule()
