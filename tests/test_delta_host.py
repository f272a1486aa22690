"""The DeltaNet layer of a served step and the log probabilities without a GPU: what the entry points refuse before anything is launched, and what the Python side checks."""
import ctypes as C

import pytest
import torch

from tests.util import pkg

szlib, delta, sampling = pkg.lib, pkg.delta, pkg.sampling


def pool(**kw):
    d = dict(n_slots=4, k_heads=2, v_heads=4, head_dim=64, grouped=0, conv_k=3, conv_type=szlib.TYPE_BF16, state=4096, conv=8192, state_stride=4 * 64 * 64 * 4, conv_stride=2 * 512 * 2)
    d.update(kw)
    return delta.DeltaPoolC(**d)


def batch(**kw):
    d = dict(n_seq=2, rows=4, max_rows=0, row_start=4096, lens=4096, from_=4096, to=0, take=0)
    d.update(kw)
    return delta.DeltaBatchC(**d)


def gates(**kw):
    d = dict(a=4096, dt=4096, norm=0, eps=1e-6)
    d.update(kw)
    return delta.DeltaGatesC(**d)


def conv(L, p=None, b=None, io=szlib.TYPE_BF16, x=1 << 20, xs=512, w=4096, bias=0, y=1 << 21, ys=512, scratch=4096, size=1 << 40):
    return L.sz_delta_conv(C.byref(p or pool()), C.byref(b or batch()), io, x, xs, w, bias, y, ys, scratch, size, 0)


def rule(L, p=None, b=None, g=None, io=szlib.TYPE_BF16, q=4096, qs=128, k=4096, ks=128, v=4096, vs=256, al=4096, als=4, be=4096, bes=4, z=0, zs=0, out=1 << 20, outs=256, scratch=4096, size=1 << 40):
    return L.sz_delta_rows(C.byref(p or pool()), C.byref(b or batch()), C.byref(g or gates()), io, q, qs, k, ks, v, vs, al, als, be, bes, z, zs, out, outs, scratch, size, 0)


BAD_POOL = [dict(head_dim=96), dict(k_heads=0), dict(v_heads=3), dict(v_heads=1), dict(v_heads=2048), dict(n_slots=0), dict(grouped=2)]
BAD_BATCH = [dict(n_seq=0), dict(n_seq=4097), dict(rows=0), dict(rows=(1 << 20) + 1), dict(max_rows=-1)]
BAD_TABLES = [dict(row_start=0), dict(lens=0), dict(from_=0), dict(lens=4098), dict(to=4097), dict(take=4099)]


def test_scratch_query_is_pure_and_checks_arguments():
    L, n = szlib.load(), C.c_int64()
    for io in (szlib.TYPE_F32, szlib.TYPE_F16, szlib.TYPE_BF16):
        assert L.sz_delta_scratch_bytes(C.byref(pool()), C.byref(batch()), io, C.byref(n)) == szlib.OK and n.value >= 256
    assert L.sz_delta_scratch_bytes(C.byref(pool()), C.byref(batch()), szlib.TYPE_Q8_0, C.byref(n)) == szlib.E_TYPE
    for bad in BAD_POOL:
        assert L.sz_delta_scratch_bytes(C.byref(pool(**bad)), C.byref(batch()), szlib.TYPE_F32, C.byref(n)) == szlib.E_ARG, bad
        assert len(L.sz_last_error()) > 0
    for bad in BAD_BATCH:
        assert L.sz_delta_scratch_bytes(C.byref(pool()), C.byref(batch(**bad)), szlib.TYPE_F32, C.byref(n)) == szlib.E_ARG, bad
    assert L.sz_delta_scratch_bytes(C.byref(pool()), C.byref(batch()), szlib.TYPE_F32, None) == szlib.E_ARG


@pytest.mark.parametrize("call", [conv, rule])
def test_calls_refuse_bad_tables_and_pools(call):
    L = szlib.load()
    for bad in BAD_POOL:
        assert call(L, p=pool(**bad)) == szlib.E_ARG, bad
    for bad in BAD_BATCH + BAD_TABLES:
        assert call(L, b=batch(**bad)) == szlib.E_ARG, bad
    assert call(L, io=szlib.TYPE_Q8_0) == szlib.E_TYPE
    for bad in (dict(scratch=0), dict(scratch=4100), dict(size=100)):
        assert call(L, **bad) == szlib.E_SCRATCH, bad


def test_conv_refuses():
    L = szlib.load()
    for bad in (dict(conv=0), dict(conv=4104), dict(conv_stride=2 * 512 * 2 - 16), dict(conv_stride=2 * 512 * 2 + 8), dict(conv_k=1), dict(conv_k=9)):
        assert conv(L, p=pool(**bad)) == szlib.E_ARG, bad
    assert conv(L, p=pool(conv_type=szlib.TYPE_Q8_0)) == szlib.E_TYPE
    for bad in (dict(x=0), dict(y=0), dict(x=(1 << 20) + 8), dict(xs=511), dict(xs=516), dict(ys=500), dict(w=0), dict(w=4100), dict(bias=4104), dict(y=1 << 20), dict(y=(1 << 20) + 512)):
        assert conv(L, **bad) == szlib.E_ARG, bad


def test_rule_refuses():
    L = szlib.load()
    for bad in (dict(state=0), dict(state=4104), dict(state_stride=4 * 64 * 64 * 4 - 16), dict(state_stride=4 * 64 * 64 * 4 + 4)):
        assert rule(L, p=pool(**bad)) == szlib.E_ARG, bad
    for bad in (dict(a=0), dict(dt=0), dict(a=4098), dict(norm=4096), dict(norm=4104)):
        assert rule(L, g=gates(**bad)) == szlib.E_ARG, bad
    for e in (-1.0, float("nan")):
        assert rule(L, g=gates(norm=4096, eps=e), z=4096, zs=256) == szlib.E_ARG
    for bad in (dict(q=0), dict(out=0), dict(k=0), dict(v=0), dict(al=0), dict(be=0), dict(q=4104), dict(k=4100), dict(vs=128), dict(ks=130), dict(qs=100), dict(al=4097), dict(als=3), dict(bes=2),
                dict(z=4096, zs=256), dict(outs=252)):
        assert rule(L, **bad) == szlib.E_ARG, bad
    assert rule(L, g=gates(norm=4096), z=4096, zs=256, q=0, out=0) == szlib.E_ARG


def test_outputs_over_inputs_are_refused():
    """Other blocks read what one writes; rows side by side in one buffer are apart."""
    L = szlib.load()
    for bad in (dict(out=4096), dict(out=4096 + 256 * 2), dict(out=4096 - 2 * 256), dict(v=1 << 20), dict(k=(1 << 20) + 1024), dict(al=(1 << 20) + 8), dict(be=(1 << 20) + 2046)):
        assert rule(L, **bad) == szlib.E_ARG, bad
        assert b"over an input" in L.sz_last_error()
    assert rule(L, g=gates(norm=4096), z=1 << 20, zs=256) == szlib.E_ARG
    assert conv(L, x=1 << 20, xs=1024, y=(1 << 20) + 512, ys=1024) == szlib.E_ARG and b"over x" in L.sz_last_error()
    assert conv(L, b=batch(rows=1), x=1 << 20, y=1 << 20) == szlib.E_ARG and b"over x" in L.sz_last_error()
    # side by side: past this check (and refused for the scratch)
    assert conv(L, x=1 << 20, xs=1024, y=(1 << 20) + 1024, ys=1024, scratch=0) == szlib.E_SCRATCH
    assert conv(L, x=(1 << 20) + 1024, xs=1024, y=1 << 20, ys=1024, scratch=0) == szlib.E_SCRATCH
    assert rule(L, v=(1 << 20) + 512, vs=512, out=1 << 20, outs=512, scratch=0) == szlib.E_SCRATCH


def test_status_refuses():
    L = szlib.load()
    assert L.sz_delta_status(0, 1, None, 0) == szlib.E_ARG and L.sz_delta_status(4100, 1, None, 0) == szlib.E_ARG and L.sz_delta_status(4096, 0, None, 0) == szlib.E_ARG


def test_logprob_rows_refuses():
    L = szlib.load()

    def call(ty=szlib.TYPE_F32, lg=4096, st=1000, rows=2, vocab=1000, tok=4096, T=0, top=2, lp=4096, rank=4096, ent=4096, ids=4096, best=4096):
        return L.sz_logprob_rows(ty, lg, st, rows, vocab, tok, T, top, lp, rank, ent, ids, best, 0)
    assert call(ty=szlib.TYPE_Q8_0) == szlib.E_TYPE
    for bad in (dict(lg=0), dict(lg=4097), dict(tok=0), dict(tok=4098), dict(T=4097), dict(top=-1), dict(top=65), dict(ids=0), dict(best=0), dict(ids=4097), dict(best=4098), dict(lp=4097), dict(rank=4099),
                dict(ent=4098), dict(rows=0), dict(vocab=0), dict(vocab=262145), dict(st=999), dict(rows=(1 << 20) + 1), dict(top=0, lp=0, rank=0, ent=0), dict(tok=0, rank=0)):
        assert call(**bad) == szlib.E_ARG, bad
        assert len(L.sz_last_error()) > 0


def ints(*s):
    return torch.zeros(*s, dtype=torch.int32)


def test_the_python_side_checks_shapes():
    state, carried = torch.zeros(5, 4, 64, 64), torch.zeros(5, 2, 512, dtype=torch.bfloat16)
    p = delta.States(2, 4, 64, state, carried)
    assert (p.conv_k, p.channels, p.c.state_stride, p.c.conv_stride) == (3, 512, 65536, 2048)
    apart = delta.States(2, 4, 64, state=torch.zeros(5, 2, 4, 64, 64)[:, 1])
    assert apart.c.state_stride == 131072
    for args, kw in (((2, 4, 64), {}), ((2, 4, 64, state.half()), {}), ((2, 4, 64, state[:, :3]), {}), ((2, 4, 64, state.transpose(2, 3)), {}), ((2, 4, 64, state, carried[:4]), {}),
                     ((2, 4, 64, state, carried[:, :, :500]), {}), ((2, 4, 64, state[:1].expand(5, 4, 64, 64)), {}), ((2, 4, 64), dict(conv=carried.double())), ((2, 4, 64), dict(conv=carried[:, 0]))):
        with pytest.raises(ValueError):
            delta.States(*args, **kw)
    for args, kw in (((ints(3).long(), ints(2), ints(2)), {}), ((ints(2), ints(2), ints(2)), {}), ((ints(3), ints(2), ints(3)), {}), ((ints(3), ints(2), ints(2)), dict(to=ints(1))),
                     ((ints(3), ints(2), ints(2)), dict(take=ints(4)[::2])), ((ints(3), ints(2), None), {})):
        with pytest.raises(ValueError):
            delta.Step(p, *args, 4, **kw)
    with pytest.raises(ValueError, match="GPU"):
        delta.Step(p, ints(3), ints(2), ints(2), 4)


def test_the_log_probabilities_python_side_checks_shapes():
    lg, tok = torch.zeros(3, 10), ints(3)
    for kw in (dict(tokens=tok.long()), dict(tokens=ints(2)), dict(tokens=tok, temperature=torch.zeros(3, dtype=torch.float64)), dict(tokens=ints(6)[::2]),
               dict(tokens=tok, top=2, out=sampling.LogProbs(None, None, None, ints(3, 2), None)), dict(tokens=tok, out=sampling.LogProbs(torch.zeros(4), None, None, None, None)),
               dict(out=sampling.LogProbs(torch.zeros(3), None, None, None, None))):
        with pytest.raises(ValueError):
            sampling.logprob_rows(lg, **kw)
    for bad in (lg.double(), lg[0], torch.zeros(1, 10).expand(3, 10), torch.zeros(3, 20)[:, ::2]):
        with pytest.raises(ValueError):
            sampling.logprob_rows(bad, tok)
    with pytest.raises(ValueError, match="GPU"):
        sampling.logprob_rows(lg, tok)
