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
