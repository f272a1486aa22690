"""The paged cache and the row sampler without a GPU: what the entry points refuse, before anything is launched, and what the Python side checks."""
import ctypes as C

import pytest
import torch

from tests.util import pkg

szlib, paged, sampling = pkg.lib, pkg.paged, pkg.sampling


def cache(**kw):
    d = dict(type=szlib.TYPE_BF16, n_kv_head=2, head_dim=128, page_size=16, n_pages=10, k=4096, v=8192, page_stride=2 * 16 * 256, head_stride=16 * 256, pos_stride=256)
    d.update(kw)
    return paged.PagedCacheC(**d)


def batch(**kw):
    d = dict(n_seq=2, rows=4, max_pages=8, shared_len=0, pages=4096, row_start=4096, lens=4096, shared_pages=0)
    d.update(kw)
    return paged.PagedBatchC(**d)


BAD_CACHE = [(dict(type=szlib.TYPE_F32), szlib.E_TYPE), (dict(type=szlib.TYPE_Q8_0), szlib.E_TYPE), (dict(head_dim=96), szlib.E_ARG), (dict(n_kv_head=0), szlib.E_ARG),
             (dict(n_kv_head=3), szlib.E_ARG), (dict(page_size=12), szlib.E_ARG), (dict(page_size=4), szlib.E_ARG), (dict(page_size=2048), szlib.E_ARG), (dict(n_pages=0), szlib.E_ARG),
             (dict(pos_stride=250), szlib.E_ARG), (dict(pos_stride=128), szlib.E_ARG), (dict(page_stride=0), szlib.E_ARG), (dict(head_stride=-16), szlib.E_ARG)]
BAD_BATCH = [dict(n_seq=0), dict(n_seq=4097), dict(rows=0), dict(rows=(1 << 20) + 1), dict(max_pages=0), dict(shared_len=-1)]
BAD_TABLES = [dict(pages=0), dict(row_start=0), dict(lens=0), dict(lens=4098), dict(shared_len=5)]


def append(L, c=None, b=None, rope=None, io=szlib.TYPE_BF16, nh=8, k=4096, ks=256, v=4096, vs=256, q=4096, qs=1024, qh=128, qo=8192, qos=1024, scratch=4096, size=1 << 40):
    rope = paged.PagedRopeC(64, 1e-6, 1e4, 0, 0) if rope is None else rope
    return L.sz_paged_append(C.byref(c or cache()), C.byref(b or batch()), C.byref(rope), io, nh, k, ks, v, vs, q, qs, qh, qo, qos, scratch, size, 0)


def attend(L, c=None, b=None, io=szlib.TYPE_BF16, nh=8, scale=0.1, q=4096, qs=1024, gate=0, gs=0, gh=0, out=4096, os_=1024, lse=0, scratch=4096, size=1 << 40):
    return L.sz_paged_attend(C.byref(c or cache()), C.byref(b or batch()), io, nh, scale, q, qs, gate, gs, gh, out, os_, lse, scratch, size, 0)


def test_scratch_query_is_pure_and_checks_arguments():
    L, n = szlib.load(), C.c_int64()
    assert L.sz_paged_scratch_bytes(C.byref(cache()), C.byref(batch()), 8, C.byref(n)) == szlib.OK
    few = n.value
    assert L.sz_paged_scratch_bytes(C.byref(cache()), C.byref(batch(rows=64, n_seq=64, shared_len=100)), 8, C.byref(n)) == szlib.OK and n.value > few > 0
    for bad, code in BAD_CACHE:
        assert L.sz_paged_scratch_bytes(C.byref(cache(**bad)), C.byref(batch()), 8, C.byref(n)) == code, bad
        assert len(L.sz_last_error()) > 0
    for bad in BAD_BATCH:
        assert L.sz_paged_scratch_bytes(C.byref(cache()), C.byref(batch(**bad)), 8, C.byref(n)) == szlib.E_ARG, bad
    for nh in (0, 1, 7, 8192):
        assert L.sz_paged_scratch_bytes(C.byref(cache()), C.byref(batch()), nh, C.byref(n)) == szlib.E_ARG
    assert L.sz_paged_scratch_bytes(C.byref(cache()), C.byref(batch()), 8, None) == szlib.E_ARG


@pytest.mark.parametrize("call", [append, attend])
def test_calls_refuse_bad_tables_and_caches(call):
    L = szlib.load()
    for bad, code in BAD_CACHE:
        assert call(L, c=cache(**bad)) == code, bad
    for bad in BAD_BATCH + BAD_TABLES:
        assert call(L, b=batch(**bad)) == szlib.E_ARG, bad
    assert call(L, c=cache(k=0)) == szlib.E_ARG and call(L, c=cache(v=8200)) == szlib.E_ARG
    assert call(L, io=szlib.TYPE_Q8_0) == szlib.E_TYPE
    for bad in (dict(scratch=0), dict(scratch=4100), dict(size=100)):
        assert call(L, **bad) == szlib.E_SCRATCH, bad
    for bad in (dict(q=4100), dict(qs=1020), dict(qs=512), dict(nh=9)):
        assert call(L, **bad) == szlib.E_ARG, bad


def test_append_refuses():
    L = szlib.load()
    for bad in (dict(k=0), dict(v=0), dict(ks=100), dict(vs=4), dict(k=4104), dict(qo=0), dict(qos=512), dict(qh=64), dict(qh=132), dict(q=4096, qo=4096, qh=256, qs=2048)):
        assert append(L, **bad) == szlib.E_ARG, bad
    for r in ((63, 1e-6, 1e4), (130, 1e-6, 1e4), (-2, 1e-6, 1e4), (64, 1e-6, 0.0), (64, 1e-6, float("inf")), (64, -1.0, 1e4), (64, float("nan"), 1e4)):
        assert append(L, rope=paged.PagedRopeC(r[0], r[1], r[2], 0, 0)) == szlib.E_ARG, r
    assert append(L, rope=paged.PagedRopeC(64, 1e-6, 1e4, 4100, 0)) == szlib.E_ARG


def test_attend_refuses():
    L = szlib.load()
    for bad in (dict(q=0), dict(out=0), dict(out=4104), dict(os_=1000), dict(scale=float("nan")), dict(scale=float("inf")), dict(lse=4098),
                dict(gate=4100, gs=1024, gh=128), dict(gate=4096, gs=512, gh=128), dict(gate=4096, gs=1024, gh=64)):
        assert attend(L, **bad) == szlib.E_ARG, bad


def test_status_refuses():
    L, n = szlib.load(), C.c_int()
    assert L.sz_paged_status(0, 1, None, 0) == szlib.E_ARG and L.sz_paged_status(4100, 1, None, 0) == szlib.E_ARG and L.sz_paged_status(4096, 0, None, 0) == szlib.E_ARG


def test_sample_rows_refuses():
    L = szlib.load()

    def call(ty=szlib.TYPE_F32, lg=4096, st=1000, rows=2, vocab=1000, T=0, k=0, p=0, mp=0, u=4096, tok=4096, prob=0):
        return L.sz_sample_rows(ty, lg, st, rows, vocab, T, k, p, mp, u, tok, prob, 0)
    assert call(ty=szlib.TYPE_Q8_0) == szlib.E_TYPE
    for bad in (dict(lg=0), dict(lg=4097), dict(u=0), dict(u=4100), dict(tok=0), dict(tok=4098), dict(prob=4098), dict(T=4097), dict(k=4098), dict(p=4099), dict(mp=4097), dict(rows=0),
                dict(vocab=0), dict(vocab=262145), dict(st=999), dict(rows=(1 << 20) + 1)):
        assert call(**bad) == szlib.E_ARG, bad
        assert len(L.sz_last_error()) > 0


def test_the_python_side_checks_shapes():
    k = torch.zeros(4, 2, 16, 64, dtype=torch.bfloat16)
    paged.Cache(k, k.clone(), 64)
    assert paged.Cache(k.transpose(1, 2).contiguous().transpose(1, 2), k.transpose(1, 2).contiguous().transpose(1, 2), 64).c.pos_stride == 2 * 64 * 2
    for a, b, hd in ((k, k[:3], 64), (k, k.half(), 64), (k.float(), k.float(), 64), (k, k, 128), (k[0], k[0], 64), (k.to(torch.uint8), k.to(torch.uint8), 64)):
        with pytest.raises(ValueError):
            paged.Cache(a, b, hd)
    c = paged.Cache(k, k.clone(), 64)
    i = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731
    for args, kw in (((i(2, 3).long(), i(3), i(2)), {}), ((i(2, 3), i(2), i(2)), {}), ((i(1, 3), i(3), i(2)), {}), ((i(2, 3), i(3), i(2)), dict(shared_len=17, shared_pages=i(1))),
                     ((i(2, 3), i(3), i(2)), dict(shared_len=17)), ((i(2, 6)[:, ::2], i(3), i(2)), {})):
        with pytest.raises(ValueError):
            paged.Step(c, *args, 4, 4, **kw)
    lg = torch.zeros(3, 10)
    for kw in (dict(uniform=torch.zeros(3)), dict(uniform=torch.zeros(2, dtype=torch.float64)), dict(uniform=torch.zeros(3, dtype=torch.float64), top_k=torch.zeros(3)),
               dict(uniform=torch.zeros(3, dtype=torch.float64), temperature=torch.zeros(6)[::2]), dict(uniform=torch.zeros(3, dtype=torch.float64), out=torch.zeros(3))):
        with pytest.raises(ValueError):
            sampling.sample_rows(lg, **kw)
    with pytest.raises(ValueError):
        sampling.sample_rows(lg.double(), torch.zeros(3, dtype=torch.float64))


def test_the_python_side_refuses_overlapping_rows():
    """A stride below a row's own size (an expanded tensor) would be read at other places than the tensor has."""
    one = torch.zeros(1, 2, 16, 64, dtype=torch.bfloat16)
    for bad in (one.expand(4, 2, 16, 64), one[:, :1].expand(1, 2, 16, 64), one[:, :, :1].expand(1, 2, 16, 64)):
        with pytest.raises(ValueError):
            paged.Cache(bad, bad, 64)
    u = torch.zeros(3, dtype=torch.float64)
    for bad in (torch.zeros(1, 10).expand(3, 10), torch.zeros(12).as_strided((3, 10), (1, 1)), torch.zeros(3, 1).expand(3, 10)):
        with pytest.raises(ValueError):
            sampling.sample_rows(bad, u)


def test_more_work_than_a_call_takes_is_refused():
    """Units of work are counted in 32 bits: a million rows of 128 heads over a table of four million positions are not a call."""
    L = szlib.load()
    c = cache(n_kv_head=8, page_size=1024, n_pages=1 << 20, page_stride=8 * 1024 * 256, head_stride=1024 * 256)
    assert attend(L, c=c, b=batch(n_seq=1, rows=1 << 20, max_pages=4096), nh=128, qs=128 * 128, os_=128 * 128, size=1 << 62) == szlib.E_ARG
    assert b"more work" in L.sz_last_error()


def test_the_python_side_refuses_tensors_that_are_not_on_a_gpu():
    """Everything else about these calls is right: the kernels would read host addresses."""
    lg, u = torch.zeros(3, 10), torch.zeros(3, dtype=torch.float64)
    out = torch.full((3,), 7, dtype=torch.int32)
    for kw in (dict(), dict(out=out), dict(temperature=torch.ones(3), prob=torch.zeros(3))):
        with pytest.raises(ValueError, match="GPU"):
            sampling.sample_rows(lg, u, **kw)
    assert bool((out == 7).all())
    k = torch.zeros(4, 2, 16, 64, dtype=torch.bfloat16)
    i = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731
    with pytest.raises(ValueError, match="GPU"):
        paged.Step(paged.Cache(k, k.clone(), 64), i(2, 3), i(3), i(2), 4, 4)


def test_a_dimension_of_one_has_any_stride():
    """One page, or one key head: what a view's stride there is says nothing about the pool."""
    base = torch.zeros(4096, dtype=torch.bfloat16)
    one = base.as_strided((1, 1, 16, 64), (3, 5, 64, 1))
    c = paged.Cache(one, base[2048:].as_strided((1, 1, 16, 64), (3, 5, 64, 1)), 64).c
    n, L = C.c_int64(), szlib.load()
    assert L.sz_paged_scratch_bytes(C.byref(c), C.byref(batch()), 4, C.byref(n)) == szlib.OK
    packed = torch.zeros(4096, dtype=torch.uint8).as_strided((2, 1, 16, 80), (1280, 7, 80, 1))
    c = paged.Cache(packed, packed, 64).c
    assert c.page_stride == 1280 and L.sz_paged_scratch_bytes(C.byref(c), C.byref(batch()), 4, C.byref(n)) == szlib.OK
