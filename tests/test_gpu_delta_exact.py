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
