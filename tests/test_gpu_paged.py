"""The paged cache on the GPU: append and attention against plain 64-bit arithmetic, at the sizes, types, layouts and masks where they can go wrong."""
import math

import numpy as np
import pytest
import torch

from tests.util import pkg

paged, szlib = pkg.paged, pkg.lib
pytestmark = pytest.mark.gpu

IO = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


# ---- the plain side ---------------------------------------------------------------------------------------------------------------------
def q8_pack(x):
    """The session's packed heads (per-32 symmetric int8, f16 scales), the oracle's arithmetic in torch."""
    hd = x.shape[-1]
    g = x.float().reshape(*x.shape[:-1], hd // 32, 32)
    sc = (g.abs().amax(-1) * np.float32(1 / 127)).half()
    inv = torch.where(sc > 0, 1 / sc.float(), torch.zeros_like(sc, dtype=torch.float32))
    codes = torch.round(g * inv[..., None]).clamp(-127, 127).to(torch.int8).reshape(x.shape).view(torch.uint8)
    out = torch.zeros(*x.shape[:-1], paged.head_bytes(hd), dtype=torch.uint8, device=x.device)
    out[..., :hd] = codes
    out[..., hd:hd + hd // 16] = sc.view(torch.uint8)
    return out


def values(pool, hd):
    if pool.dtype != torch.uint8:
        return pool.double()
    sc = pool[..., hd:hd + hd // 16].contiguous().view(torch.float16).double()
    return (pool[..., :hd].view(torch.int8).double().reshape(*pool.shape[:-1], hd // 32, 32) * sc[..., None]).reshape(*pool.shape[:-1], hd)


class Case:
    """A batch over a paged cache.  lens: positions of the sequences, ms: their rows; `pad` rows follow the last sequence."""

    def __init__(self, lens, ms, nh=4, nkv=2, hd=64, page=16, io="f32", cache="f16", shared=0, pad=0, layout="hnd", seed=0, scale_kv=1.0, extra_pages=0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.rnd = lambda *s: torch.randn(*s, device="cuda", generator=g)
        self.lens, self.ms, self.nh, self.nkv, self.hd, self.ps, self.shared, self.cache_type = lens, ms, nh, nkv, hd, page, shared, cache
        self.io = IO[io]
        n = len(lens)
        own = [max(0, -(-(x - shared) // page)) for x in lens]
        width, nsh = max(own + [1]) + extra_pages, -(-shared // page)
        total = sum(own) + nsh + 3
        order = torch.randperm(total, device="cuda", generator=g).to(torch.int32)
        pages = torch.full((n, width), -7, dtype=torch.int32, device="cuda")          # entries that no position needs are no pages
        at = 0
        for b in range(n):
            pages[b, :own[b]] = order[at:at + own[b]]
            at += own[b]
        self.pages, self.shared_pages = pages, order[at:at + nsh].contiguous()
        self.rows = sum(ms) + pad
        starts = np.concatenate([[0], np.cumsum(ms)]).astype(np.int32)
        self.row_start = torch.from_numpy(starts).cuda()
        self.len_t = torch.tensor(lens, dtype=torch.int32, device="cuda")
        shape = (total, nkv, page, hd) if layout == "hnd" else (total, page, nkv, hd)
        k, v = scale_kv * self.rnd(*shape), scale_kv * self.rnd(*shape)
        k, v = (q8_pack(k), q8_pack(v)) if cache == "q8" else (k.to(IO[cache]), v.to(IO[cache]))
        if layout == "nhd":
            k, v = k.transpose(1, 2), v.transpose(1, 2)
        self.k, self.v = k, v
        self.q = (1.5 * self.rnd(self.rows, nh, hd)).to(self.io)
        self.make_step()

    def make_step(self):
        self.cache = paged.Cache(self.k, self.v, self.hd)
        self.step = paged.Step(self.cache, self.pages, self.row_start, self.len_t, self.rows, self.nh, shared_pages=self.shared_pages, shared_len=self.shared)

    def positions(self, pool, b):
        """[positions of sequence b, kv heads, hd] in 64 bits."""
        of = lambda ids, n: values(pool[ids.long()], self.hd).transpose(1, 2).reshape(-1, self.nkv, self.hd)[:n]  # noqa: E731
        own = max(0, self.lens[b] - self.shared)
        parts = [of(self.shared_pages, self.shared)] if self.shared else []
        if own:
            parts.append(of(self.pages[b, :-(-own // self.ps)], own))
        return torch.cat(parts) if parts else torch.zeros(0, self.nkv, self.hd, dtype=torch.float64, device="cuda")

    def want(self, gate=None, scale=None):
        """(outputs, the sum of weights times |values|, log of the denominators), 64-bit; rows behind the sequences are not set."""
        out = torch.zeros(self.rows, self.nh, self.hd, dtype=torch.float64, device="cuda")
        mag, lse = torch.zeros_like(out), torch.full((self.rows, self.nh), -math.inf, dtype=torch.float64, device="cuda")
        scale = 1 / math.sqrt(self.hd) if scale is None else scale
        r = 0
        for b, m in enumerate(self.ms):
            k, v = self.positions(self.k, b), self.positions(self.v, b)
            for j in range(m):
                p = self.lens[b] - m + j
                if p >= self.shared:
                    for h in range(self.nh):
                        s = scale * (k[:p + 1, h // (self.nh // self.nkv)] @ self.q[r, h].double())
                        w = torch.softmax(s, 0)
                        out[r, h], mag[r, h] = w @ v[:p + 1, h // (self.nh // self.nkv)], w @ v[:p + 1, h // (self.nh // self.nkv)].abs()
                        lse[r, h] = torch.logsumexp(s, 0)
                r += 1
        if gate is not None:
            z = torch.sigmoid(gate.double())
            out, mag = out * z, mag * z
        return out, mag, lse

    def tolerance(self, want, mag):
        """Half a step of the result's type; before it, f32 arithmetic: a score is a sum of hd products (hd 2^-23 of their magnitudes, |q||k| scale below 12
        sigma = 30 here, in units of its own exponent), which moves every weight by that much, and sums of up to 64 partial sums - 2^-13 of the
        weighted magnitudes holds f32's part with a wide margin; 16-bit results carry weights of 11 bits and more: 2^-10 of the magnitudes.
        Where many rows share positions (tcgen05: 16-bit queries over their own type) weights are rounded to the result's type: half a step of
        every weight, of the magnitudes in sum."""
        many = self.io != torch.float32 and self.k.dtype == self.io and self.rows * self.nh // self.nkv >= 96
        return HALF_STEP[self.io] * (want.abs() + (mag if many else 0)) + (2.0 ** -13 if self.io == torch.float32 else 2.0 ** -10) * mag + 1e-30

    def check(self, gate=None, **kw):
        out = torch.full_like(self.q, 77.0)
        lse = torch.full((self.rows, self.nh), 77.0, device="cuda")
        self.step.attend(self.q, out=out, gate=gate, lse=lse, **kw)
        assert self.step.status() == 0
        want, mag, wl = self.want(gate, **kw)
        n = sum(self.ms)
        off = (out.double() - want).abs() / self.tolerance(want, mag)
        assert float(off[:n].max()) < 1.0, "%.3g of the tolerance at %s" % (float(off[:n].max()), np.unravel_index(int(off[:n].argmax()), off[:n].shape))
        assert bool((out[n:] == 77.0).all()) and bool((lse[n:] == 77.0).all())          # a padded batch's rows are left as they were
        seen = torch.isfinite(wl[:n])
        assert bool(((lse[:n].double() - wl[:n]).abs()[seen] < 2e-4).all()) and bool((lse[:n][~seen] == -math.inf).all())
        return out


# ---- attention ---------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("cache", ["f16", "bf16", "q8"])
@pytest.mark.parametrize("io", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_every_type_and_width(io, cache, hd):
    Case([1, 77, 130], [1, 2, 5], nh=8, nkv=2, hd=hd, io=io, cache=cache, seed=hd).check()


@pytest.mark.parametrize("lens", [[1], [2], [63], [64], [65], [16 * 64], [1000, 1, 64, 129], [0, 5, 0], [3, 0, 0, 700]])
def test_lengths_from_nothing_on(lens):
    c = Case(lens, [1] * len(lens), io="bf16", cache="bf16")
    out = c.check()
    for b, x in enumerate(lens):
        if x == 0:
            assert bool((out[b] == 0).all())


@pytest.mark.parametrize("nh,nkv", [(1, 1), (5, 5), (6, 2), (7, 1), (16, 2), (64, 1), (3, 1)])
@pytest.mark.parametrize("m", [1, 3, 9])
def test_head_groups(nh, nkv, m):
    Case([150, 40 + m], [m, m], nh=nh, nkv=nkv, hd=64, seed=nh * 10 + m).check()


@pytest.mark.parametrize("page", [8, 16, 64, 128, 1024])
@pytest.mark.parametrize("layout", ["hnd", "nhd"])
def test_pages_and_layouts(page, layout):
    Case([300, 17, page + 1], [2, 1, 4], page=page, layout=layout, cache="q8", hd=128, seed=page).check()


@pytest.mark.parametrize("ms", [[17], [100], [1, 60, 3], [33, 0, 2]])
@pytest.mark.parametrize("before", [0, 1, 200])
def test_prompts(ms, before):
    Case([m + before for m in ms], ms, nh=4, nkv=1, hd=128, io="bf16", cache="bf16", seed=before).check()


@pytest.mark.parametrize("shared", [1, 16, 63, 64, 500, 1037])
@pytest.mark.parametrize("io,cache", [("f32", "q8"), ("bf16", "bf16"), ("f16", "f16")])
def test_a_shared_prefix(shared, io, cache):
    Case([shared + x for x in (1, 40, 3, 130, 2)], [1, 4, 3, 2, 1], nh=8, nkv=2, hd=64, io=io, cache=cache, shared=shared, pad=2, seed=shared).check()


def test_a_shared_prefix_of_many_rows():
    Case([700 + 5 * i for i in range(40)], [1 + i % 4 for i in range(40)], nh=16, nkv=2, hd=128, io="bf16", cache="bf16", shared=641, seed=3).check()


def test_sequences_in_front_of_the_shared_positions_attend_to_nothing():
    c = Case([70, 64, 10, 0], [2, 1, 1, 1], shared=64, seed=5)
    out = c.check()
    assert bool((out[2:] == 0).all())


def test_rows_before_the_first_position():
    c = Case([3, 200], [5, 2], seed=6)              # two rows of a padded sequence lie before position 0
    out = c.check()
    assert bool((out[:2] == 0).all())


@pytest.mark.parametrize("cache", ["f16", "bf16", "q8"])
def test_a_long_sequence_beside_short_ones(cache):
    Case([20000, 3, 900], [1, 2, 1], nh=8, nkv=1, hd=128, io="f32", cache=cache, page=64, seed=8).check()


def test_more_sequences_than_a_block_plans_for():
    Case([1 + (7 * i) % 50 for i in range(600)], [1] * 600, nh=2, nkv=1, hd=64, io="bf16", cache="bf16", seed=9).check()


def test_more_tiles_than_a_block_plans_for():
    Case([2600], [2600], nh=16, nkv=1, hd=64, io="bf16", cache="bf16", seed=10, page=128).check()


def test_gate_scale_and_strides():
    c = Case([90, 300], [3, 1], nh=8, nkv=2, hd=64, io="bf16", cache="bf16", seed=11)
    both = c.rnd(c.rows, c.nh, 2 * c.hd).to(c.io)      # queries and gates alternate
    c.check(gate=both[:, :, c.hd:])
    c.check(scale=0.3)
    wide = torch.zeros(c.rows, c.nh * c.hd + 64, dtype=c.io, device="cuda")
    wide[:, :c.nh * c.hd] = c.q.reshape(c.rows, -1)
    out = torch.full_like(wide, 5.0)
    c.step.attend(wide[:, :c.nh * c.hd].view(c.rows, c.nh, c.hd), out=out[:, :c.nh * c.hd].view(c.rows, c.nh, c.hd))
    assert torch.equal(out[:, :c.nh * c.hd].reshape(c.q.shape), c.check()) and bool((out[:, c.nh * c.hd:] == 5.0).all())


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("cache", ["f16", "bf16"])
def test_what_hidden_positions_hold_does_not_matter(cache, bad):
    """Behind a sequence's end in its last page, and at positions later than a row's own, keys and values may be anything."""
    c = Case([70, 33], [4, 2], cache=cache, io="f32", nh=8, nkv=2, seed=12)
    before = c.check()
    last = c.pages[0, (70 - 1) // 16]
    c.k[last, :, 70 % 16:] = bad
    c.v[last, :, 70 % 16:] = bad
    out = torch.empty_like(c.q)
    c.step.attend(c.q, out=out)
    assert torch.equal(out, before)
    c.v[last, :, 69 % 16, 5] = bad                     # the last row's own value: its output, and no other row's
    c.step.attend(c.q, out=out)
    rel = (out[:3].double() - before[:3].double()).abs().max() / before.abs().max()
    assert float(rel) < 2.0 ** -13 and torch.equal(out[4:], before[4:])
    hit = out[3, :, 5]
    assert not bool(torch.isfinite(hit).any()) and bool(torch.isfinite(out[3, :, :5]).all())


@pytest.mark.parametrize("io,cache,m", [("f32", "f16", 3), ("f32", "q8", 2), ("bf16", "bf16", 3), ("bf16", "bf16", 70)])
def test_nan_queries_and_keys(io, cache, m):
    """A row with a NaN in its query, or in a key that it sees, is NaN - and no other row."""
    c = Case([300, 200], [m, m], nh=4, nkv=2, hd=64, io=io, cache=cache, seed=20, page=16)
    before = c.check()
    c.q[1, 2, 5] = math.nan
    out = c.step.attend(c.q)
    assert bool(torch.isnan(out[1, 2]).all())
    keep = torch.ones(c.rows, 4, dtype=torch.bool, device="cuda")
    keep[1, 2] = False
    assert torch.equal(out[keep], before[keep])
    if cache != "q8":
        c.q[1, 2, 5] = 0
        page = c.pages[1, (200 - 1) // 16]
        c.k[page, 1, 199 % 16, 0] = math.nan            # the second sequence's last position: its last row's heads of the second key head
        out = c.step.attend(c.q)
        assert bool(torch.isnan(out[-1, 2:]).all()) and bool(torch.isfinite(out[-1, :2]).all()) and bool(torch.isfinite(out[:-1]).all())


@pytest.mark.parametrize("io,cache", [("f32", "f16"), ("f32", "q8"), ("bf16", "bf16"), ("f32", "bf16")])
def test_large_and_small_magnitudes(io, cache):
    for kv, q in ((1e-3, 100.0), (100.0, 0.01), (300.0, 0.003)):
        c = Case([130, 64], [2, 1], io=io, cache=cache, nh=8, nkv=2, seed=13, scale_kv=kv)
        c.q.mul_(q)
        c.check()


def test_far_apart_scores():
    """One position takes all the weight; the largest comes first, and last."""
    for at in (0, 199):
        c = Case([200], [1], io="f32", cache="f16", nh=2, nkv=1, hd=64, seed=14)
        page, slot = int(c.pages[0, at // 16]), at % 16
        c.k[page, 0, slot] = (c.q[0, 0] * 30).half()
        c.check()


def test_bad_pages_are_left_out_and_reported():
    c = Case([100, 50], [1, 1], nh=4, nkv=2, hd=64, seed=15)
    keep = c.pages.clone()
    for bad in (-1, c.k.shape[0], 2 ** 31 - 1):
        c.pages.copy_(keep)
        c.pages[0, 2] = bad                            # positions 32 .. 47
        c.step.attend(c.q)
        assert c.step.status() == 1
        szlib.check(c.step.lib.sz_paged_status(c.step.scratch, 1, None, 0))
        torch.cuda.synchronize()
        out = c.step.attend(c.q)
        c.pages.copy_(keep)
        k, v = c.positions(c.k, 0), c.positions(c.v, 0)
        seen = torch.cat([torch.arange(32), torch.arange(48, 100)]).cuda()
        for h in range(4):
            w = torch.softmax(k[seen, h // 2] @ c.q[0, h].double() / 8, 0)
            assert float((w @ v[seen, h // 2] - out[0, h].double()).abs().max()) < 1e-4
        szlib.check(c.step.lib.sz_paged_status(c.step.scratch, 1, None, 0))


def test_lengths_behind_the_table_and_row_starts_behind_the_rows():
    c = Case([40, 20], [1, 1], seed=16)
    c.len_t[1] = 16 * c.pages.shape[1] + 1
    c.pages[1] = c.pages[0]
    c.step.attend(c.q)
    assert c.step.status() == 2
    c = Case([40, 20], [1, 1], seed=16)
    c.row_start[2] = 9
    c.step.attend(c.q)
    assert c.step.status() == 8


def test_a_row_is_the_same_whoever_shares_the_step():
    """16-bit caches: nothing but the cuts between blocks depends on the other sequences - within f32 rounding of each other."""
    a = Case([333], [2], nh=8, nkv=2, hd=128, io="f32", cache="f16", seed=17)
    out = a.step.attend(a.q)
    again = a.step.attend(a.q)
    assert torch.equal(out, again)


def test_a_captured_step_serves_a_growing_batch():
    c = Case([100, 37, 64], [1, 1, 1], nh=8, nkv=2, hd=128, io="bf16", cache="bf16", seed=18, extra_pages=2)
    new = torch.randperm(c.k.shape[0], device="cuda").to(torch.int32)
    out, kin, vin = torch.empty_like(c.q), c.rnd(3, 2, 128).bfloat16(), c.rnd(3, 2, 128).bfloat16()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        c.step.append(kin, vin, rope_dims=64)
        c.step.attend(c.q, out=out)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.step.append(kin, vin, rope_dims=64)
        c.step.attend(c.q, out=out)
    for grow in range(3):
        c.lens = [x + (5 if grow else 0) for x in c.lens]
        for b, x in enumerate(c.lens):                 # sequences go on into further pages (any: what is checked is what they then hold)
            need = -(-x // 16)
            c.pages[b, need - 1] = new[(grow * 3 + b) % len(new)] if int(c.pages[b, need - 1]) < 0 else c.pages[b, need - 1]
        c.len_t.copy_(torch.tensor(c.lens, dtype=torch.int32))
        c.q.copy_(c.rnd(*c.q.shape))
        graph.replay()
        torch.cuda.synchronize()
        want, mag, _ = c.want()
        assert float(((out.double() - want).abs() / c.tolerance(want, mag)).max()) < 1.0
    assert c.step.status() == 0


def test_another_stream():
    c = Case([500, 70], [2, 3], nh=8, nkv=2, hd=64, io="bf16", cache="bf16", seed=19)
    want = c.check()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = c.step.attend(c.q)
    side.synchronize()
    assert torch.equal(out, want)


# ---- many rows over the same positions (whole units of 128 on tcgen05, the rest as above) --------------------------------------------------
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("lens,ms,shared", [([200], [100], 0), ([1300], [129], 0), ([3000, 260, 128], [40, 200, 128], 0), ([600 + i for i in range(24)], [1 + i % 3 for i in range(24)], 512),
                                            ([1500 + i for i in range(16)], [2] * 16, 1441), ([10000], [16], 0)])
def test_many_rows(hd, kind, lens, ms, shared):
    Case(lens, ms, nh=8, nkv=1, hd=hd, io=kind, cache=kind, shared=shared, seed=hd, page=32).check()


@pytest.mark.parametrize("page,layout", [(8, "hnd"), (16, "nhd"), (64, "nhd"), (128, "hnd"), (1024, "nhd")])
def test_many_rows_pages_and_layouts(page, layout):
    Case([2900, 300], [60, 111], nh=10, nkv=2, hd=128, io="bf16", cache="bf16", page=page, layout=layout, seed=page, pad=3).check()


@pytest.mark.parametrize("nh,nkv", [(3, 3), (14, 2), (48, 1), (200, 1)])
def test_many_rows_head_groups(nh, nkv):
    Case([700, 1000], [100, 37], nh=nh, nkv=nkv, hd=64, io="bf16", cache="bf16", seed=nh).check()


def test_many_rows_scores_that_climb():
    """Every unit's largest score is far above the one's before: the sums are scaled again and again; and the other way round."""
    for way in (1, -1):
        c = Case([1280], [130], nh=4, nkv=2, hd=128, io="bf16", cache="bf16", seed=3, page=128)
        for p in range(10):
            c.k[int(c.pages[0, p])] *= (0.2 + 0.4 * p) if way > 0 else (4.0 - 0.4 * p)
        c.check()


def test_many_rows_bad_pages_are_left_out_and_reported():
    c = Case([900], [130], nh=4, nkv=1, hd=64, io="bf16", cache="bf16", page=16, seed=4)
    keep = c.pages.clone()
    c.pages[0, 3] = -5
    c.pages[0, 20] = c.k.shape[0]
    out = c.step.attend(c.q)
    assert c.step.status() == 1
    c.pages.copy_(keep)
    k, v = c.positions(c.k, 0), c.positions(c.v, 0)
    for j in (0, 64, 129):
        seen = torch.tensor([t for t in range(900 - 130 + j + 1) if t // 16 not in (3, 20)], device="cuda")
        for h in range(4):
            w = torch.softmax(k[seen, 0] @ c.q[j, h].double() / 8, 0)
            want, mag = w @ v[seen, 0], w @ v[seen, 0].abs()
            assert bool(((out[j, h].double() - want).abs() < c.tolerance(want, mag)).all())


def test_many_rows_hidden_positions_do_not_matter():
    for bad in (math.nan, math.inf):
        c = Case([700], [130], nh=4, nkv=1, hd=128, io="bf16", cache="bf16", page=16, seed=5)
        before = c.check()
        last = c.pages[0, 699 // 16]
        c.k[last, :, 700 % 16:] = bad
        c.v[last, :, 700 % 16:] = bad
        out = c.step.attend(c.q)
        assert torch.equal(out, before)
        c.v[last, :, 699 % 16, 7] = bad                # the last row's own
        out = c.step.attend(c.q)
        assert float((out[:129].double() - before[:129].double()).abs().max()) < 2.0 ** -7 * float(before.abs().max())
        assert not bool(torch.isfinite(out[129, :, 7]).any()) and bool(torch.isfinite(out[129, :, :7]).all())


# ---- append ------------------------------------------------------------------------------------------------------------------------------
def rotated(x, w, pos, dims, theta, eps):
    x = x.double()
    if w is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w.double()
    if not dims:
        return x
    h = dims // 2
    a = torch.outer(pos.double(), theta ** (-torch.arange(0, dims, 2, dtype=torch.float64, device=x.device) / dims))[:, None, :]
    u, v = x[..., :h], x[..., h:dims]
    return torch.cat([u * a.cos() - v * a.sin(), v * a.cos() + u * a.sin(), x[..., dims:]], -1)


def check_append(c, dims, norm, theta=1e7, with_q=True, q=None, q_out=None):
    nkv, hd, n = c.nkv, c.hd, sum(c.ms)
    kin, vin = c.rnd(c.rows, nkv, hd).to(c.io), c.rnd(c.rows, nkv, hd).to(c.io)
    q = c.q if q is None else q
    qn, kn = (1 + 0.1 * c.rnd(hd), 1 + 0.1 * c.rnd(hd)) if norm else (None, None)
    k0, v0 = c.k.clone(), c.v.clone()
    if with_q and q_out is None:
        q_out = torch.full((c.rows, c.nh, hd), 55.0, dtype=c.io, device="cuda")
    qin = q.clone()
    got = c.step.append(kin, vin, q=q if with_q else None, q_out=q_out if with_q else None, rope_dims=dims, theta=theta, q_norm=qn, k_norm=kn, eps=1e-6)
    assert c.step.status() == 0
    pos = torch.cat([torch.arange(x - m, x) for x, m in zip(c.lens, c.ms)]).cuda()
    kw, vw = rotated(kin[:n], kn, pos, dims, theta, 1e-6), vin[:n].double()
    touched = torch.zeros(c.k.shape[0], c.ps, dtype=torch.bool, device="cuda")
    r = 0
    for b, (x, m) in enumerate(zip(c.lens, c.ms)):
        for p in range(x - m, x):
            if p >= 0:
                o = p - c.shared
                page, slot = int(c.pages[b, o // c.ps]), o % c.ps
                touched[page, slot] = True
                for pool, want in ((c.k, kw[r]), (c.v, vw[r])):
                    have = values(pool[page, :, slot], hd)
                    if pool.dtype == torch.uint8:      # half a code, and f16's rounding of the scale over 127 codes of it, and f32's before
                        big = want.reshape(nkv, hd // 32, 32).abs().amax(-1, keepdim=True).expand(-1, -1, 32).reshape(nkv, hd)
                        tol = big / 127 * (0.5 + 127 * 2.0 ** -11 + 127 * 2.0 ** -21) + 2.0 ** -24
                        assert bool((pool[page, :, slot, hd + hd // 16:] == 0).all())
                    else:                              # a rounding of the cache's type, f32's rounding of norm and rotation (of a pair's length) before it
                        tol = HALF_STEP[pool.dtype] * want.abs() + 2.0 ** -20 * want.abs().amax() + 2.0 ** -25
                    assert bool(((have - want).abs() <= tol).all())
            r += 1
    keep = ~touched[:, None, :, None].expand(*c.k.shape)
    assert torch.equal(c.k[keep], k0[keep]) and torch.equal(c.v[keep], v0[keep])      # no other position
    if with_q:
        want = rotated(qin[:n], qn, pos, dims, theta, 1e-6)
        there = pos >= 0
        tol = HALF_STEP[c.io] * want.abs() + 2.0 ** -20 * want.abs().amax()
        assert bool(((got[:n].double() - want).abs() <= tol)[there].all())
        if got is not q:
            assert bool((got[:n][~there] == 55.0).all()) and bool((got[n:] == 55.0).all())


@pytest.mark.parametrize("cache", ["f16", "bf16", "q8"])
@pytest.mark.parametrize("io", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("hd,dims,norm", [(64, 32, True), (128, 128, False), (256, 64, True), (64, 0, True), (128, 2, False), (256, 256, True)])
def test_append(io, cache, hd, dims, norm):
    check_append(Case([1, 40, 17], [1, 3, 17], nh=4, nkv=2, hd=hd, io=io, cache=cache, seed=hd + dims), dims, norm)


@pytest.mark.parametrize("page,layout", [(8, "nhd"), (128, "hnd"), (1024, "nhd")])
def test_append_pages_and_layouts(page, layout):
    check_append(Case([300, 17, page + 1], [2, 1, 4], page=page, layout=layout, io="bf16", cache="q8", hd=128, seed=page, pad=3), 128, False)


@pytest.mark.parametrize("io,cache", [("bf16", "bf16"), ("f32", "q8")])
def test_append_many_rows(io, cache):
    """Blocks of several rows, rows of several sequences in one, none among them, and rows that are left out."""
    check_append(Case([1500, 3, 40, 0, 5, 90], [1401, 1, 17, 0, 9, 2], nh=4, nkv=2, hd=128, io=io, cache=cache, seed=9, pad=5), 64, True)
    check_append(Case([1 + i for i in range(1210)], [1] * 1210, nh=2, nkv=1, hd=64, io=io, cache=cache, seed=10, page=8), 32, True)


def test_append_behind_a_shared_prefix_and_without_queries():
    check_append(Case([70, 101], [2, 37], shared=64, page=16, seed=21), 32, True)
    check_append(Case([70, 101], [2, 37], page=16, seed=22), 32, True, with_q=False)


def test_append_in_place_and_from_alternating_heads():
    c = Case([9, 33], [2, 5], nh=4, hd=128, io="bf16", cache="bf16", seed=23)
    check_append(c, 64, True, q=c.q, q_out=c.q)
    both = c.rnd(c.rows, c.nh, 2 * c.hd).to(c.io)
    check_append(c, 64, True, q=both[:, :, :c.hd])


def test_append_leaves_out_rows_before_position_zero():
    check_append(Case([3, 20], [5, 2], seed=24), 32, False)


@pytest.mark.parametrize("far", [24576, 1048575, 16777217])
def test_append_at_far_positions(far):
    """The table's early pages may be anything; the angle of a far position keeps its digits."""
    c = Case([20], [2], nh=4, nkv=1, hd=64, io="f32", cache="f16", page=1024, seed=25)
    width = far // 1024 + 1
    c.pages = torch.zeros(1, width, dtype=torch.int32, device="cuda")
    c.lens = [far + 1]
    c.len_t.fill_(far + 1)
    c.make_step()
    check_append(c, 64, False, theta=1e4)


def test_append_reports_what_it_leaves_out():
    c = Case([40, 20], [1, 1], seed=26)
    kin = c.rnd(2, 2, 64)
    k0 = c.k.clone()
    c.pages[0, 2] = 10 ** 6
    c.step.append(kin, kin)
    assert c.step.status() == 1
    o = 19
    page = int(c.pages[1, 1])
    k0[page, :, o % 16] = kin[1].half()
    assert torch.equal(c.k, k0)
    c = Case([70, 30], [1, 1], shared=64, seed=27)
    k0 = c.k.clone()
    c.step.append(c.rnd(2, 2, 64), c.rnd(2, 2, 64))
    assert c.step.status() == 4
    k0[int(c.pages[0, 0]), :, 5] = c.k[int(c.pages[0, 0]), :, 5]
    assert torch.equal(c.k, k0)
    c = Case([40, 20], [1, 1], seed=28)
    c.len_t[0] = 16 * c.pages.shape[1] + 1
    c.step.append(c.rnd(2, 2, 64), c.rnd(2, 2, 64))
    assert c.step.status() == 2


def test_steps_as_a_server_makes_them():
    """A prompt behind a shared system prompt, then tokens one after the other and drafts: what is appended is what is attended to."""
    nh, nkv, hd, ps, shared = 8, 2, 128, 16, 50
    g = torch.Generator(device="cuda").manual_seed(31)
    rnd = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    n, width = 3, 8
    total = n * width + 4
    k, v = torch.full((total, nkv, ps, hd), math.nan, device="cuda").half(), torch.full((total, nkv, ps, hd), math.nan, device="cuda").half()
    cache = paged.Cache(k, v, hd)
    order = torch.randperm(total, device="cuda", generator=g).to(torch.int32)
    pages, shared_pages = order[:n * width].view(n, width).contiguous(), order[n * width:].contiguous()
    lens, rs = torch.zeros(n, dtype=torch.int32, device="cuda"), torch.zeros(n + 1, dtype=torch.int32, device="cuda")
    sys_k, sys_v = rnd(shared, nkv, hd), rnd(shared, nkv, hd)
    # the system prompt goes in as a sequence of its own, whose pages are then the shared list
    one = paged.Step(cache, shared_pages.view(1, -1), torch.tensor([0, shared], dtype=torch.int32, device="cuda"), torch.tensor([shared], dtype=torch.int32, device="cuda"), shared, nh)
    one.append(sys_k, sys_v, rope_dims=hd)
    assert one.status() == 0
    hist_k = [rotated(sys_k, None, torch.arange(shared, device="cuda"), hd, 1e4, 0) for _ in range(n)]
    hist_v = [sys_v.double() for _ in range(n)]
    for ms in ([20, 7, 33], [1, 1, 1], [4, 1, 3], [1, 4, 1]):
        R = sum(ms)
        rs.copy_(torch.tensor([0] + list(np.cumsum(ms)), dtype=torch.int32))
        lens += torch.tensor(ms, dtype=torch.int32, device="cuda") + (shared if ms[0] == 20 else 0)
        step = paged.Step(cache, pages, rs, lens, R, nh, shared_pages=shared_pages, shared_len=shared)
        kin, vin, q = rnd(R, nkv, hd), rnd(R, nkv, hd), rnd(R, nh, hd)
        qr = step.append(kin, vin, q=q, rope_dims=hd)
        out = step.attend(qr)
        assert step.status() == 0
        r = 0
        for b, m in enumerate(ms):
            pos = torch.arange(hist_k[b].shape[0], hist_k[b].shape[0] + m, device="cuda")
            hist_k[b] = torch.cat([hist_k[b], rotated(kin[r:r + m], None, pos, hd, 1e4, 0)])
            hist_v[b] = torch.cat([hist_v[b], vin[r:r + m].double()])
            qw = rotated(q[r:r + m], None, pos, hd, 1e4, 0)
            for j in range(m):
                for h in range(nh):
                    K, V = hist_k[b][:pos[j] + 1, h // 4].half().double(), hist_v[b][:pos[j] + 1, h // 4].half().double()
                    w = torch.softmax(K @ qw[j, h] / math.sqrt(hd), 0)
                    # keys that round to the other f16 neighbour: 2^-11 of a key here and there; scores move by 2^-11 |q| at most
                    assert float((out[r + j, h].double() - w @ V).abs().max()) < 2.0 ** -11 * float(qw[j, h].norm()) * float(w @ V.abs().amax(-1)) + 1e-4
            r += m


def test_rows_that_overlap_are_refused():
    """Expanded rows or heads have strides that the kernels do not take; one row or one head has any."""
    c = Case([9, 33], [2, 5], nh=4, nkv=2, hd=64, io="bf16", cache="bf16", seed=90)
    kv, q = c.rnd(c.rows, 2, 64).to(c.io), c.q
    for bad in (kv[:1].expand(7, 2, 64), kv[:, :1].expand(7, 2, 64)):
        with pytest.raises(ValueError):
            c.step.append(bad, kv)
        with pytest.raises(ValueError):
            c.step.append(kv, bad)
    for bad in (q[:1].expand(7, 4, 64), q[:, :1].expand(7, 4, 64)):
        for call in (lambda: c.step.append(kv, kv, q=bad), lambda: c.step.attend(bad), lambda: c.step.attend(q, gate=bad), lambda: c.step.attend(q, out=bad)):
            with pytest.raises(ValueError):
                call()
    with pytest.raises(ValueError):
        c.step.append(kv, kv, q_out=q)
    c = Case([33], [1], nh=2, nkv=1, hd=64, io="bf16", cache="bf16", seed=91)
    want = c.step.attend(c.q)
    assert torch.equal(c.step.attend(c.q.expand(1, 2, 64).as_strided((1, 2, 64), (0, 64, 1))), want)


@pytest.mark.parametrize("n,m,shared", [(3, 5, 0), (3, 5, 32), (300, 2, 0), (300, 2, 32)])
def test_a_descending_row_start_is_reported(n, m, shared):
    """Its sequences would have more tiles than the tables have room for: no row is attended, nothing but zeros comes out, the status tells."""
    c = Case([shared + 40] * n, [m] * n, nh=4, nkv=2, hd=64, io="bf16", cache="bf16", shared=shared, seed=92)
    want = c.step.attend(c.q).clone()
    good = c.row_start.clone()
    c.row_start[1::2] = c.rows
    c.row_start[0] = 0
    c.row_start[2::2] = 0
    out = torch.full_like(c.q, 7.0)
    c.step.attend(c.q, out=out)
    assert c.step.status() & 8
    if not shared:
        assert bool(((out == 0) | (out == 7.0)).all())
    c.row_start.copy_(good)
    assert torch.equal(c.step.attend(c.q), want)


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("seqs,m,nh,nkv,io,cache,shared", [(75, 1, 16, 2, "f32", "q8", 0), (250, 2, 3, 3, "f32", "f16", 0), (40, 1, 30, 6, "bf16", "bf16", 700), (20, 3, 35, 7, "f16", "f16", 0)])
def test_parts_joined_by_two_warps(hd, seqs, m, nh, nkv, io, cache, shared):
    """Rows times heads between those that eight warps and those that one joins; heads that are no multiple of a block's."""
    Case([shared + 100 + 37 * i % 900 for i in range(seqs)], [m] * seqs, nh=nh, nkv=nkv, hd=hd, io=io, cache=cache, shared=shared, seed=hd + seqs, pad=1).check()


@pytest.mark.parametrize("n,m,shared,io,cache", [(300, 2, 32, "bf16", "bf16"), (300, 2, 640, "f16", "f16"), (300, 1, 100, "f32", "q8"), (3, 50, 0, "bf16", "bf16"), (3, 50, 130, "f32", "bf16"), (1, 3, 0, "f32", "f16")])
def test_what_the_scratch_held_does_not_matter(n, m, shared, io, cache):
    c = Case([shared + 400 // (1 + n // 100)] * n, [m] * n, nh=4, nkv=2, hd=64, io=io, cache=cache, shared=shared, seed=93)
    first = c.check().clone()
    at = c.step.scratch - c.step._mem.data_ptr()
    for byte in (0, 255, 63):
        c.step._mem[at + 256:].fill_(byte)           # (the first 256 bytes hold the status)
        assert torch.equal(c.check(), first)


@pytest.mark.parametrize("cache", ["f16", "bf16", "q8"])
@pytest.mark.parametrize("lens,ms,shared", [([130, 77], [3, 1], 0), ([300, 260, 290], [2, 1, 30], 250)])
def test_f32_rows_keep_their_accuracy(cache, lens, ms, shared):
    """Heads of 64, scores of six and less with magnitudes |q_i k_i| scale below 16 in sum.  A score's f32 sums cut 2^-23 of it in each of four steps, a query's pieces
    leave 2^-23 of every product: 4 6 2^-23 + 16 2^-23 = 2^-17.7 at most, a weight as much, and the quotient of two sums of weights twice
    that: below 2^-16 of the weighted magnitudes, with weights of 22 bits and more.  (One piece of 11 bits would be four to ten times over it.)"""
    c = Case(lens, ms, nh=8, nkv=2, hd=64, io="f32", cache=cache, shared=shared, seed=40)
    out = c.step.attend(c.q)
    want, mag, _ = c.want()
    off = (out.double() - want).abs() / (2.0 ** -24 * want.abs() + 2.0 ** -16 * mag)
    assert float(off.max()) < 1.0, float(off.max())


def spoil(pool, hd, page, slots, scale, groups=slice(None)):
    """Packed heads at `slots` of a page: codes of 127 under scales of `scale`."""
    at = pool[page, :, slots]
    at[..., :hd] = 127
    sc = at[..., hd:hd + hd // 16].contiguous().view(torch.float16)
    sc[..., groups] = scale
    at[..., hd:hd + hd // 16] = sc.view(torch.uint8)
    pool[page, :, slots] = at


@pytest.mark.parametrize("bad", [65504.0, math.inf, math.nan])
@pytest.mark.parametrize("io,hd,m,size", [("f32", 64, 4, 1.0), ("f32", 256, 4, 1e-3), ("bf16", 128, 4, 1e-3), ("f32", 128, 20, 0.01), ("f16", 256, 20, 0.01), ("bf16", 64, 9, 1.0)])
def test_what_hidden_packed_positions_hold_does_not_matter(io, hd, m, size, bad):
    """As above for packed heads: a scale that no row may see, or only a later one, chooses nothing for the others - not a bit."""
    c = Case([70, 33], [m, 2], cache="q8", io=io, nh=8, nkv=2, hd=hd, seed=41, scale_kv=size)
    before = c.check().clone()
    last = c.pages[0, (70 - 1) // 16]
    spoil(c.k, hd, last, slice(70 % 16, None), bad)
    spoil(c.v, hd, last, slice(70 % 16, None), bad)
    assert torch.equal(c.step.attend(c.q), before)
    spoil(c.v, hd, last, slice(69 % 16, 70 % 16), bad, slice(0, 1))                    # the last row's own: its output, and no other row's
    out = c.step.attend(c.q)
    assert torch.equal(out[:m - 1], before[:m - 1]) and torch.equal(out[m:], before[m:])
    if not math.isfinite(bad):
        assert not bool(torch.isfinite(out[m - 1, :, :32]).any()) and bool(torch.isfinite(out[m - 1, :, 32:]).all())


def test_scales_far_apart_on_one_head():
    """A unit's largest value scale is 2^29 times its smallest: the small ones' positions keep their bits in rows that do not see the large one."""
    for m in (3, 20):
        c = Case([64 + m], [m], cache="q8", io="f32", nh=4, nkv=1, hd=64, seed=42, scale_kv=1e-3)
        c.v[c.pages[0, (64 + m - 1) // 16], :, (64 + m - 1) % 16] = q8_pack(1e6 * c.rnd(1, 64))
        out = c.step.attend(c.q)
        want, mag, _ = c.want()
        assert float(((out.double() - want).abs() / (2.0 ** -16 * mag + 2.0 ** -24 * want.abs()))[:m - 1].max()) < 1.0


@pytest.mark.parametrize("nats", [10, 13, 17])
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_a_tail_far_below_the_first_position(kind, hd, nats):
    """A position of value 0 in front that takes nearly all the weight, and thousands far below it whose values are the answer: a weight e^-17 of the largest
    keeps its type's bits (f16 11, bf16 8), so that each is off by half a step of its own size, and the sum by no more; the scores are equal, so nothing averages out.
    f32's part of it: a score of `nats` and less is off by hd / 16 steps of 2^-23 of it, 2^-16 at most."""
    n, nkv = 1024, 8                                                                 # (tiles and heads enough that a block takes nearly all of an item's positions)
    c = Case([n + 1] * 640, [1] * 640, nh=64, nkv=nkv, hd=hd, io=kind, cache=kind, shared=n, page=64, seed=43)
    c.q.zero_()
    c.q[:, :, 0] = 4.0
    c.k.zero_()
    c.k[c.shared_pages[0], :, 0, 0] = 8.0 * nats                                     # its score: 4 * 8 nats / 32; all others': 0
    c.v.abs_()
    c.v[c.shared_pages[0], :, 0] = 0
    out = c.step.attend(c.q, scale=1 / 32)
    assert c.step.status() == 0
    w = torch.full((n + 1,), math.exp(-nats), dtype=torch.float64, device="cuda")
    w[0] = 1
    for b in (0, 17, 333, 639):
        want = torch.einsum("t,thd->hd", w, c.positions(c.v, b)).repeat_interleave(64 // nkv, 0) / w.sum()
        off = (out[b].double() - want).abs() / (2 * HALF_STEP[c.io] * want + 2.0 ** -16 * want + (2.0 ** -25 if kind == "f16" else 0))      # (f16's subnormals: half of 2^-24)
        assert float(off.max()) < 1.0, float(off.max())


@pytest.mark.parametrize("kind,hd,nh,m", [("bf16", 256, 8, 13), ("f16", 128, 8, 13), ("bf16", 64, 3, 33), ("bf16", 256, 16, 45)])
def test_a_tile_that_ends_inside_a_warp(kind, hd, nh, m):
    """Vectors that fill a part of a warp's 32, written straight to the output, gated; and once more with a value that is not finite where only later rows see it."""
    c = Case([500, 200], [m, m], nh=nh, nkv=1, hd=hd, io=kind, cache=kind, page=16, seed=44, pad=2)
    gate = c.rnd(c.rows, nh, hd).to(c.io)
    before = c.check(gate=gate).clone()
    c.v[c.pages[0, (500 - 2) // 16], :, (500 - 2) % 16, 3] = math.inf                # the last two rows see it
    out = c.step.attend(c.q, gate=gate)
    assert torch.equal(out[m:2 * m], before[m:2 * m]) and torch.equal(out[:m - 2], before[:m - 2])
    assert bool(torch.isinf(out[m - 2:m, :, 3]).all()) and bool(torch.isfinite(out[m - 2:m, :, 4:]).all()) and bool(torch.isfinite(out[m - 2:m, :, :3]).all())


@pytest.mark.parametrize("m,kept,io,cache,shared", [(5, 2, "f32", "f16", 0), (5, 2, "bf16", "q8", 32), (40, 33, "bf16", "bf16", 0), (40, 33, "bf16", "bf16", 64), (1500, 1300, "bf16", "bf16", 0)])
def test_rows_that_are_not_there_are_left_out(m, kept, io, cache, shared):
    """row_start goes on behind the rows that the call has: those that it has keep their places and their results, the others' places are left alone."""
    whole = Case([shared + 60, shared + m + 20], [2, m], nh=8, nkv=2, hd=64, io=io, cache=cache, shared=shared, seed=45)
    kin, vin = whole.rnd(2 + m, 2, 64).to(whole.io), whole.rnd(2 + m, 2, 64).to(whole.io)
    k0, v0 = whole.k.clone(), whole.v.clone()
    qw = whole.step.append(kin, vin, q=whole.q, rope_dims=32)
    assert whole.step.status() == 0
    k1, v1 = whole.k.clone(), whole.v.clone()
    n = 2 + kept
    part = paged.Step(whole.cache, whole.pages, whole.row_start, whole.len_t, n, 8, shared_pages=whole.shared_pages, shared_len=shared)
    whole.k.copy_(k0)
    whole.v.copy_(v0)
    assert torch.equal(part.append(kin[:n].contiguous(), vin[:n].contiguous(), q=whole.q[:n].contiguous(), rope_dims=32), qw[:n])
    assert part.status() == 8
    for have, first, then in ((whole.k, k0, k1), (whole.v, v0, v1)):
        expect = then.clone()
        for t in range(shared + 20 + kept, shared + 20 + m):                            # the left out rows' places: as they were
            page, slot = int(whole.pages[1, (t - shared) // 16]), (t - shared) % 16
            expect[page, :, slot] = first[page, :, slot]
        assert torch.equal(have, expect)
    whole.k.copy_(k1)
    whole.v.copy_(v1)
    out = part.attend(whole.q[:n].contiguous())
    want, mag, _ = whole.want()
    assert float(((out.double() - want[:n]).abs() / whole.tolerance(want, mag)[:n]).max()) < 1.0


@pytest.mark.parametrize("m,shared", [(2, 0), (130, 0), (130, 1024)])
@pytest.mark.parametrize("bad", [-2, -1, -2147483648])
def test_any_page_id_out_of_range_is_reported(m, shared, bad):
    c = Case([shared + 700], [m], nh=4, nkv=1, hd=128, io="bf16", cache="bf16", page=16, shared=shared, seed=46)
    (c.shared_pages if shared else c.pages[0])[5] = bad
    c.step.attend(c.q)
    assert c.step.status() == 1


@pytest.mark.parametrize("io,cache", [("f32", "f16"), ("f32", "bf16"), ("f32", "q8"), ("bf16", "bf16"), ("f16", "f16"), ("bf16", "q8")])
def test_a_sequence_alone_and_in_a_batch(io, cache):
    """What else the batch holds moves the cuts between blocks and, for 16-bit rows over their own type, chooses the kernel: both results lie within the tolerance of
    the same values, so within twice that of each other (f32: of what test_f32_rows_keep_their_accuracy allows)."""
    big = Case([333, 1200, 64, 901, 77], [2, 60, 1, 3, 40], nh=16, nkv=2, hd=64, io=io, cache=cache, seed=49)
    out = big.step.attend(big.q)
    want, mag, _ = big.want()
    r = 0
    for b, m in enumerate(big.ms):
        alone = paged.Step(big.cache, big.pages[b:b + 1].contiguous(), torch.tensor([0, m], dtype=torch.int32, device="cuda"), big.len_t[b:b + 1].clone(), m, 16)
        one = alone.attend(big.q[r:r + m].contiguous())
        w, g = want[r:r + m], mag[r:r + m]
        tol = 2.0 ** -24 * w.abs() + 2.0 ** -16 * g if io == "f32" else HALF_STEP[big.io] * (w.abs() + g) + 2.0 ** -10 * g
        assert float(((one.double() - out[r:r + m].double()).abs() / (2 * tol)).max()) < 1.0
        r += m


@pytest.mark.parametrize("io,cache", [("f32", "f16"), ("bf16", "bf16"), ("f16", "bf16")])
@pytest.mark.parametrize("hd,dims", [(256, 64), (64, 32), (128, 2), (128, 64), (256, 256)])
@pytest.mark.parametrize("rows", [3, 1190])
def test_append_of_heads_that_are_not_finite(io, cache, hd, dims, rows):
    """An infinity or NaN reaches its own dimension and the one it is turned with; every other dimension of the head is what it would be without."""
    c = Case([rows + 4], [rows], nh=4, nkv=2, hd=hd, io=io, cache=cache, page=64, seed=47)
    kin, vin = c.rnd(rows, 2, hd).to(c.io), c.rnd(rows, 2, hd).to(c.io)
    clean = c.step.append(kin, vin, q=c.q, rope_dims=dims).clone()
    k0 = c.k.clone()
    for bad in (math.inf, -math.inf, math.nan):
        for d in sorted({0, dims // 2 - 1, dims // 2, dims - 1, min(dims, hd - 1), hd - 1}):
            q, k = c.q.clone(), kin.clone()
            q[:, :, d] = bad
            k[:, :, d] = bad
            got = c.step.append(k, vin, q=q, rope_dims=dims)
            hit = {d, (d + dims // 2) % dims} if d < dims else {d}
            keep = [x for x in range(hd) if x not in hit]
            assert torch.equal(got[:, :, keep], clean[:, :, keep]) and torch.equal(c.k[..., keep], k0[..., keep])
            assert not bool(torch.isfinite(got[:, :, d]).any())


@pytest.mark.parametrize("rows", [6, 1200])
def test_append_reports_a_descending_row_start(rows):
    """A row would be two sequences': nothing is stored, nothing given back, the status tells."""
    c = Case([rows + 9, rows + 70, 40], [rows // 2, rows // 2 - 1, 1], nh=4, nkv=2, hd=64, io="bf16", cache="bf16", page=64, seed=48)
    kin = c.rnd(rows, 2, 64).bfloat16()
    k0, v0 = c.k.clone(), c.v.clone()
    c.row_start.copy_(torch.tensor([0, rows - 1, rows // 2, rows], dtype=torch.int32))
    q_out = torch.full_like(c.q, 3.0)
    c.step.append(kin, kin, q=c.q, q_out=q_out, rope_dims=32)
    assert c.step.status() == 8
    assert torch.equal(c.k, k0) and torch.equal(c.v, v0) and bool((q_out == 3.0).all())


def test_one_row_has_any_stride():
    """Rows 130 elements apart are no multiple of 16 bytes; of a single one only its address counts."""
    c = Case([33], [1], nh=2, nkv=1, hd=64, io="bf16", cache="bf16", seed=94)
    want, kv = c.step.attend(c.q, gate=c.q).clone(), c.rnd(1, 1, 64).bfloat16()
    wide = lambda x: torch.zeros(130, dtype=x.dtype, device="cuda").as_strided(x.shape, (130, 64, 1)).copy_(x)  # noqa: E731
    assert torch.equal(c.step.attend(wide(c.q), gate=wide(c.q)), want)
    first = c.step.append(kv, kv, q=c.q, rope_dims=32)
    k1 = c.k.clone()
    assert torch.equal(c.step.append(wide(kv), wide(kv), q=wide(c.q), rope_dims=32), first) and torch.equal(c.k, k1)


# ---- calls at the ends of what is allowed --------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("io,cache,m", [("f32", "f16", 2), ("f32", "q8", 2), ("bf16", "bf16", 130)])
def test_pools_of_more_than_four_gigabytes(io, cache, m):
    """Pages whose bytes lie behind 2^32: the last of a pool of 5 GB, beside its first."""
    nkv, hd, ps = 2, 256, 16
    head = paged.head_bytes(hd) if cache == "q8" else hd
    kind = torch.uint8 if cache == "q8" else IO[cache]
    size = nkv * ps * head * torch.empty(0, dtype=kind).element_size()
    n = 5 * 2 ** 30 // size
    c = Case([200, 77], [m, 1], nh=8, nkv=nkv, hd=hd, io=io, cache=cache, page=ps, seed=50)
    want = c.check().clone()
    k, v = torch.empty(n, nkv, ps, head, dtype=kind, device="cuda"), torch.empty(n, nkv, ps, head, dtype=kind, device="cuda")
    old = c.pages.clamp(min=0).long()
    new = torch.where(c.pages >= 0, torch.where(c.pages % 2 == 0, n - 1 - c.pages, c.pages), c.pages)
    k[new.clamp(min=0).long().reshape(-1)] = c.k[old.reshape(-1)]
    v[new.clamp(min=0).long().reshape(-1)] = c.v[old.reshape(-1)]
    c.k, c.v, c.pages = k, v, new.to(torch.int32).contiguous()
    c.make_step()
    assert torch.equal(c.check(), want)
    kin = c.rnd(c.rows, nkv, hd).to(c.io)
    c.step.append(kin, kin)
    assert c.step.status() == 0
    for b, (x, mm) in enumerate(zip(c.lens, c.ms)):
        page = int(c.pages[b, (x - 1) // ps])
        row = kin[sum(c.ms[:b + 1]) - 1].double()
        have = values(c.k[page, :, (x - 1) % ps], hd)
        assert float((have - row).abs().max()) < 2.0 ** -8 * float(row.abs().max())


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("nh", [128, 4096])
def test_one_row_of_many_heads_on_one(kind, nh):
    Case([700, 65], [1, 1], nh=nh, nkv=1, hd=64, io=kind, cache=kind, seed=51).check()


@pytest.mark.parametrize("io,cache,m", [("f32", "q8", 3), ("bf16", "bf16", 3), ("bf16", "bf16", 60), ("f16", "f16", 60)])
@pytest.mark.parametrize("scale", [0.0, -0.2, 1.0])
def test_any_finite_scale(io, cache, m, scale):
    """0: the mean of the values; below 0: the smallest product weighs most.  (1: scores of 60, whose f32 sums cut 2^-23 of them in each of four steps, and weights
    2^-15 by that - f32's part stays below a quarter of the tolerance's.)"""
    Case([300, 90], [m, 2], nh=8, nkv=2, hd=64, io=io, cache=cache, seed=52).check(scale=scale)


@pytest.mark.parametrize("hd", [64, 256])
@pytest.mark.parametrize("page", [8, 1024])
def test_many_rows_smallest_and_largest_pages(hd, page):
    Case([1500, 300], [60, 111], nh=8, nkv=2, hd=hd, io="bf16", cache="bf16", page=page, seed=page + hd, shared=0).check()
    Case([1500 + i for i in range(16)], [2] * 16, nh=16, nkv=2, hd=hd, io="f16", cache="f16", page=page, seed=page + hd, shared=1391).check()


@pytest.mark.parametrize("hd", [64, 128, 256])
def test_many_rows_before_the_first_position(hd):
    """A padded prompt: more rows than positions, and a sequence of none."""
    c = Case([60, 300, 0], [130, 100, 40], nh=4, nkv=1, hd=hd, io="bf16", cache="bf16", seed=53, pad=7)
    out = c.check()
    assert bool((out[:70] == 0).all()) and bool((out[230:270] == 0).all())


@pytest.mark.parametrize("bad", [math.nan, math.inf, 65504.0])
@pytest.mark.parametrize("io,cache,seqs", [("f32", "f16", 3), ("f32", "q8", 3), ("bf16", "q8", 30), ("bf16", "bf16", 3), ("bf16", "bf16", 30), ("f16", "f16", 30)])
def test_what_lies_behind_the_shared_positions_does_not_matter(io, cache, seqs, bad):
    """The shared list's last page goes on behind shared_len, with anything."""
    c = Case([141 + 3 * i for i in range(seqs)], [1 + i % 2 for i in range(seqs)], nh=8, nkv=2, hd=128, io=io, cache=cache, shared=133, page=32, seed=54)
    before = c.check().clone()
    last = c.shared_pages[-1]
    for pool in (c.k, c.v):
        if cache == "q8":
            spoil(pool, 128, last, slice(133 % 32, None), bad)
        else:
            pool[last, :, 133 % 32:] = bad
    assert torch.equal(c.step.attend(c.q), before)


def test_as_many_sequences_as_a_call_takes():
    c = Case([1 + i % 9 for i in range(4096)], [1] * 4096, nh=2, nkv=2, hd=64, page=16, io="bf16", cache="bf16", seed=55, pad=1)
    out = torch.full_like(c.q, 7.0)
    c.step.attend(c.q, out=out)
    assert c.step.status() == 0 and bool((out[4096:] == 7.0).all())
    k, v = values(c.k[c.pages[:, 0].long()], 64), values(c.v[c.pages[:, 0].long()], 64)          # [sequence, head, position, dimension]
    s = torch.einsum("bhd,bhtd->bht", c.q[:4096].double(), k) / 8
    s = s.masked_fill(torch.arange(16, device="cuda") >= c.len_t[:, None, None], -math.inf)
    w = torch.softmax(s, -1)
    want, mag = torch.einsum("bht,bhtd->bhd", w, v), torch.einsum("bht,bhtd->bhd", w, v.abs())
    assert float(((out[:4096].double() - want).abs() / (HALF_STEP[c.io] * want.abs() + 2.0 ** -10 * mag + 1e-30)).max()) < 1.0


@pytest.mark.parametrize("io,cache,ms", [("bf16", "bf16", [100, 3]), ("f32", "q8", [2, 3]), ("f16", "f16", [1, 1])])
def test_two_steps_at_once(io, cache, ms):
    """Two batches over one cache, a Step and a stream each, and their captured graphs side by side: neither sees the other's scratch."""
    a = Case([900, 70], ms, nh=8, nkv=2, hd=128, io=io, cache=cache, seed=56)
    pages, rs, lens = a.pages.flip(0).contiguous(), torch.tensor([0, 2, 3], dtype=torch.int32, device="cuda"), a.len_t.flip(0).contiguous()
    b = paged.Step(a.cache, pages, rs, lens, 3, 8)
    qb = a.rnd(3, 8, 128).to(a.io)
    wa, wb = a.step.attend(a.q).clone(), b.attend(qb).clone()
    outs, graphs, streams = [torch.empty_like(wa), torch.empty_like(wb)], [], [torch.cuda.Stream(), torch.cuda.Stream()]
    for step, q, out, st in ((a.step, a.q, outs[0], streams[0]), (b, qb, outs[1], streams[1])):
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            for _ in range(20):
                step.attend(q, out=out)
    torch.cuda.synchronize()
    assert torch.equal(outs[0], wa) and torch.equal(outs[1], wb)
    for step, q, out in ((a.step, a.q, outs[0]), (b, qb, outs[1])):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            step.attend(q, out=out)
            step.attend(q, out=out)
        graphs.append(g)
    for out in outs:
        out.zero_()
    torch.cuda.synchronize()
    for _ in range(20):
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], wa) and torch.equal(outs[1], wb)
