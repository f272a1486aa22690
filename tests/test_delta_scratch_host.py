"""The scratch of the DeltaNet layer's calls without a GPU: what a step allocates is enough for rows of every type."""
import ctypes as C

import pytest

from tests.test_delta_host import batch, pool, rule
from tests.util import pkg

szlib = pkg.lib
ROWS = [1, 39, 40, 64, 128, 700, 2048, 4093, 4096, 6500, 8192, 12300, 16384, 16400, 40000, 1 << 17, 1 << 20]


def need(io, kh, vh, d, n_seq, rows, max_rows):
    n = C.c_int64()
    p = pool(k_heads=kh, v_heads=vh, head_dim=d, state_stride=4 * vh * d * d)
    assert szlib.load().sz_delta_scratch_bytes(C.byref(p), C.byref(batch(n_seq=n_seq, rows=rows, max_rows=max_rows)), io, C.byref(n)) == szlib.OK
    return n.value


@pytest.mark.parametrize("kh, vh", [(1, 1), (4, 4), (8, 16), (8, 32), (16, 16), (16, 32), (16, 48), (32, 32), (5, 35), (64, 64), (128, 1024)])
@pytest.mark.parametrize("d", [64, 128])
def test_no_type_of_rows_needs_more_than_f32(kh, vh, d):
    """On both sides of the slab's size."""
    for n_seq in (1, 9, 64, 4096):
        for rows in ROWS:
            for max_rows in (0, 4, 300):
                f32, f16, bf16 = (need(t, kh, vh, d, n_seq, rows, max_rows) for t in (szlib.TYPE_F32, szlib.TYPE_F16, szlib.TYPE_BF16))
                assert f32 >= f16 and f32 >= bf16, (n_seq, rows, max_rows, f32, f16, bf16)
                assert f32 <= 256 + max(96 << 20, 8 * (256 + need(szlib.TYPE_F32, kh, vh, d, 1, 128, 0)))


@pytest.mark.parametrize("io", [szlib.TYPE_F16, szlib.TYPE_BF16])
def test_long_prompts_of_16_bits(io):
    """What f32 asks for holds them; a byte less than they need is refused."""
    for kh, vh, d, rows in ((16, 48, 128, 6500), (32, 32, 128, 4096), (8, 32, 128, 8192), (8, 16, 64, 16400), (16, 16, 128, 8192)):
        size = need(io, kh, vh, d, 1, rows, 0)
        assert size <= need(szlib.TYPE_F32, kh, vh, d, 1, rows, 0)
        p, b = pool(k_heads=kh, v_heads=vh, head_dim=d, state_stride=4 * vh * d * d), batch(n_seq=1, rows=rows)
        assert rule(szlib.load(), p=p, b=b, io=io, qs=kh * d, ks=kh * d, vs=vh * d, als=vh, bes=vh, out=1 << 40, outs=vh * d, size=size - 1) == szlib.E_SCRATCH
