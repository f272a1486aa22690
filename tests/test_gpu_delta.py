"""The DeltaNet layer of a served step on the GPU: the convolution and the gated delta rule against plain 64-bit arithmetic, at the sizes, types, tables and
row counts where they can go wrong."""
import math

import pytest
import torch

from tests.util import pkg

delta, sampling, szlib = pkg.delta, pkg.sampling, pkg.lib
pytestmark = pytest.mark.gpu

IO = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


class Case:
    """A batch over a pool.  counts: rows of the sequences; past: their positions before them (0: new); `pad` rows follow the last sequence."""

    def __init__(self, counts, past, kh=2, vh=4, d=64, io="f32", grouped=False, fork=False, take=None, gate=True, pad=0, seed=0, conv_k=4, conv_type=None, v_scale=1.0, slow=True, max_rows=None,
                 slots=None, to=None, n_slots=None):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.rnd = lambda *s: torch.randn(*s, device="cuda", generator=g)
        n = len(counts)
        self.counts, self.past, self.kh, self.vh, self.d, self.io, self.grouped, self.take, self.conv_k = counts, past, kh, vh, d, IO[io], grouped, take, conv_k
        self.rows, self.ch = sum(counts) + pad, (2 * kh + vh) * d
        self.n_slots = n_slots or (2 if fork else 1) * n + 2
        order = torch.randperm(self.n_slots, generator=torch.Generator().manual_seed(seed)).tolist()
        self.slots = order[:n] if slots is None else slots
        self.to = (order[n:2 * n] if fork else self.slots) if to is None else to
        ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
        starts = [0]
        for m in counts:
            starts.append(starts[-1] + m)
        self.row_start, self.lens, self.slot_t = ints(starts), ints([m + p for m, p in zip(counts, past)]), ints(self.slots)
        self.to_t, self.take_t = (ints(self.to) if self.to != self.slots else None), (None if take is None else ints(take))
        self.state = self.rnd(self.n_slots, vh, d, d) * v_scale / 4
        self.carried = self.rnd(self.n_slots, conv_k - 1, self.ch).to(IO[conv_type or io])
        self.x, self.w, self.bias = self.rnd(self.rows, self.ch).to(self.io), 0.3 * self.rnd(self.ch, conv_k), 0.1 * self.rnd(self.ch)
        y = torch.nn.functional.silu(self.rnd(self.rows, self.ch))
        y[:, 2 * kh * d:] *= v_scale
        y = y.to(self.io)
        self.q, self.k, self.v = (t.unflatten(1, (-1, d)) for t in y.split([kh * d, kh * d, vh * d], 1))      # (views: rows are far apart)
        ab = self.rnd(self.rows, 2 * vh).to(self.io)
        self.alpha, self.beta = ab[:, :vh], ab[:, vh:]
        self.a = -torch.logspace(math.log10(0.002), math.log10(3.0), vh, device="cuda") if slow else -0.5 - torch.rand(vh, device="cuda", generator=g)
        self.dt = 0.1 * self.rnd(vh)
        self.z, self.norm = (self.rnd(self.rows, vh, d).to(self.io), 1 + 0.1 * self.rnd(d)) if gate else (None, None)
        self.pool = delta.States(kh, vh, d, self.state, self.carried, grouped)
        self.step = delta.Step(self.pool, self.row_start, self.lens, self.slot_t, self.rows, to=self.to_t, take=self.take_t, max_rows=max_rows)

    def taken(self, b):
        return self.counts[b] if self.take is None else max(0, min(self.counts[b], self.take[b]))

    def want_conv(self, bias=True):
        """(y, its tolerance, the carried rows), 64-bit; rows that are nobody's are NaN.  K products and sums in f32, silu's exponential and quotient: 2^-20 of the taps' magnitudes."""
        y = torch.full((self.rows, self.ch), math.nan, dtype=torch.float64, device="cuda")
        mag = torch.zeros_like(y)
        pool, r = self.carried.double(), 0
        old = pool.clone()
        for b, m in enumerate(self.counts):
            n = self.taken(b)
            if m:
                seq = torch.cat([old[self.slots[b]] * (self.past[b] > 0), self.x[r:r + n].double()])
                if n:
                    taps = seq.unfold(0, self.conv_k, 1) * self.w.double()
                    s = taps.sum(-1) + (self.bias.double() if bias else 0)
                    y[r:r + n], mag[r:r + n] = s * torch.sigmoid(s), taps.abs().sum(-1) + 0.5
                pool[self.to[b]] = seq[n:]
            r += m
        return y, HALF_STEP[self.io] * y.abs() + 2.0 ** -20 * mag, pool

    def check_conv(self, bias=True):
        y = torch.full((self.rows, self.ch), 77.0, dtype=self.io, device="cuda")
        want, tol, pool = self.want_conv(bias)
        self.step.conv(self.x, self.w, bias=self.bias if bias else None, out=y)
        assert self.step.status() == 0
        none = want.isnan()
        assert bool((y[none] == 77).all())
        assert bool(((y.double() - want).abs() <= tol)[~none].all())
        assert bool(((self.carried.double() - pool).abs() <= HALF_STEP[self.carried.dtype] * pool.abs()).all())
        return y

    def want_rule(self):
        """(out, tolerance, states, tolerance), 64-bit.  A step changes the state by sums of d products in f32 (some 20 roundings of a number that is at most the
        column's length, as |k| = 1), the row's norm, decay and beta (a few half steps each): below 40 half steps of N, the column's largest length so far plus
        its largest value.  A step turns and shrinks what was wrong before (its map is a contraction), so 40 n 2^-24 N holds a state after n rows; in chunks factors
        are held to 22 bits, and a chunk of 64 rows has 64 times 40 half steps of room for the sums of those.  An output is the state times a q of length
        1 / sqrt(d).  16-bit outputs: factors of 11 bits in the last products, 2^-10 of their magnitudes.  The norm takes the sum over a head's errors; half a
        step of the result's type comes last."""
        d, half = self.d, HALF_STEP[self.io]
        out = torch.full((self.rows, self.vh, d), math.nan, dtype=torch.float64, device="cuda")
        tol = torch.zeros_like(out)
        pool, r0 = self.state.double(), 0
        old, stol = pool.clone(), torch.zeros_like(pool)
        of = [h // (self.vh // self.kh) if self.grouped else h % self.kh for h in range(self.vh)]
        unit = lambda t: t.double() / torch.sqrt(t.double().square().sum(-1, keepdim=True) + 1e-6)  # noqa: E731
        q, k, v = unit(self.q)[:, of] / math.sqrt(d), unit(self.k)[:, of], self.v.double()
        beta = torch.sigmoid(self.beta.double())
        dec = torch.exp(self.a.double() * torch.nn.functional.softplus(self.alpha.double() + self.dt.double()))
        for b, m in enumerate(self.counts):
            n = self.taken(b)
            if m:
                S = old[self.slots[b]] * (self.past[b] > 0)
                E = S.abs()
                N = S.square().sum(1).sqrt()                                        # [heads, value dimensions]
                most = torch.zeros_like(N)
                for j in range(n):
                    r = r0 + j
                    S = S * dec[r][:, None, None]
                    dl = (v[r] - torch.einsum("hij,hi->hj", S, k[r])) * beta[r][:, None]
                    S = S + k[r][:, :, None] * dl[:, None, :]
                    E = E * dec[r][:, None, None] + k[r].abs()[:, :, None] * dl.abs()[:, None, :]
                    N, most = torch.maximum(N, S.square().sum(1).sqrt()), torch.maximum(most, v[r].abs())
                    out[r] = torch.einsum("hij,hi->hj", S, q[r])
                    tol[r] = 40 * (j + 2) * 2.0 ** -24 * (N + most) / math.sqrt(d)
                    if self.io != torch.float32:
                        tol[r] += 2.0 ** -10 * torch.einsum("hij,hi->hj", E, q[r].abs())
                pool[self.to[b]], stol[self.to[b]] = S, (40 * (n + 1) * 2.0 ** -24 * (N + most))[:, None, :]
            r0 += m
        if self.z is not None:
            rr = torch.rsqrt(out.square().mean(-1, keepdim=True) + 1e-6)
            gate = self.norm.double() * torch.sigmoid(self.z.double())
            spread = tol.square().sum(-1, keepdim=True).sqrt() / (out.square().sum(-1, keepdim=True) + d * 1e-6).sqrt()
            tol = (rr * gate).abs() * (tol + out.abs() * (spread + 2.0 ** -20)) * (1 + spread)
            out = out * rr * gate
        return out, tol + half * out.abs(), pool, stol

    def run(self, out=None):
        return self.step.rule(self.q, self.k, self.v, self.alpha, self.beta, self.a, self.dt, z=self.z, norm=self.norm, out=out)

    def check_rule(self):
        out = torch.full((self.rows, self.vh, self.d), 77.0, dtype=self.io, device="cuda")
        want, tol, pool, stol = self.want_rule()
        self.run(out)
        assert self.step.status() == 0
        none = want.isnan()
        assert bool((out[none] == 77).all())
        worst = ((out.double() - want).abs() / tol)[~none]
        assert worst.numel() == 0 or float(worst.max()) <= 1, float(worst.max())
        off = (self.state.double() - pool).abs()
        assert bool((off <= stol).all()), float((off / stol.clamp_min(1e-30)).max())
        return out


# ---- the convolution --------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("conv_k", [2, 3, 4, 5, 6, 7, 8])
@pytest.mark.parametrize("io", ["f32", "bf16", "f16"])
def test_conv_over_so_many_rows(conv_k, io):
    Case([1, 2, 0, 3, 9, 1, 40], [5, 0, 7, 11, 0, 0, 1], io=io, conv_k=conv_k, pad=3, fork=True).check_conv()


@pytest.mark.parametrize("rows", [1, 31, 32, 33, 700, 4093])
@pytest.mark.parametrize("io", ["f32", "bf16"])
def test_conv_of_one_sequence(rows, io):
    for past in (0, 9):
        Case([rows], [past], kh=2, vh=2, io=io).check_conv(bias=False)


@pytest.mark.parametrize("n", [2, 33, 64, 1100, 4096])
@pytest.mark.parametrize("max_rows", [None, 3])
def test_conv_of_many_sequences(n, max_rows):
    Case([(i * 7) % 4 for i in range(n)], [(i % 3) * 5 for i in range(n)], kh=1, vh=1, io="bf16", fork=True, max_rows=max_rows, pad=2).check_conv()


def test_conv_of_more_rows_than_were_said():
    Case([0, 100, 1, 40], [3, 0, 4, 9], io="bf16", max_rows=2, pad=3).check_conv()


@pytest.mark.parametrize("io, carried", [("bf16", "f32"), ("f32", "f16"), ("f16", "bf16")])
def test_conv_with_carried_rows_of_another_type(io, carried):
    Case([1, 5, 2], [3, 0, 8], io=io, conv_type=carried).check_conv()


def test_conv_with_rows_that_do_not_count():
    Case([4, 4, 4, 4, 8], [3, 0, 8, 1, 9], io="bf16", take=[1, 0, 9, -3, 5], fork=True).check_conv()


def test_conv_continues_itself():
    """A prompt in pieces is the prompt: bit for bit, wherever it is cut."""
    whole = Case([300], [0], io="bf16", seed=3)
    y = whole.check_conv()
    for cuts in ((1, 2, 297), (100, 199, 1), (64, 64, 172)):
        pieces = Case([300], [0], io="bf16", seed=3)
        r, slot = 0, pieces.slot_t
        for m in cuts:
            ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
            step = delta.Step(pieces.pool, ints([0, m]), ints([r + m]), slot, m)
            assert torch.equal(step.conv(pieces.x[r:r + m], pieces.w, bias=pieces.bias), y[r:r + m])
            r += m
        assert torch.equal(pieces.carried[whole.slots[0]], whole.carried[whole.slots[0]])


# ---- the rule ---------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("io", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("kh, vh, grouped", [(1, 1, False), (2, 4, False), (2, 4, True), (3, 3, True)])
def test_rule_of_few_rows(d, io, kh, vh, grouped):
    Case([1, 2, 0, 7, 8, 1, 9], [5, 0, 7, 11, 0, 0, 1], kh=kh, vh=vh, d=d, io=io, grouped=grouped, pad=3).check_rule()


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("io", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows", [15, 16, 17, 35, 36, 43, 44, 63, 64, 65, 127, 128, 129, 200, 449])
def test_rule_of_one_sequence(d, io, rows):
    for past in (0, 9):
        Case([rows], [past], d=d, io=io, gate=past == 0, seed=rows).check_rule()


@pytest.mark.parametrize("d, io", [(128, "bf16"), (64, "f16"), (128, "f32")])
def test_rule_of_prompts_and_tokens_together(d, io):
    Case([1, 130, 0, 64, 3, 1, 260, 31, 1], [700, 0, 9, 64, 8, 0, 100, 0, 77], d=d, io=io, fork=True, pad=5).check_rule()


@pytest.mark.parametrize("n", [64, 300])
def test_rule_of_many_sequences(n):
    Case([(i * 7) % 4 for i in range(n)], [(i % 3) * 5 for i in range(n)], kh=1, vh=2, io="bf16", fork=True).check_rule()


@pytest.mark.parametrize("scale", [1e-12, 1e-4, 3e4])
@pytest.mark.parametrize("rows", [5, 150])
def test_rule_at_other_magnitudes(scale, rows):
    """What is held in fewer bits is scaled by what there is."""
    for io in ("f32", "bf16") if scale > 1e-6 else ("f32",):
        Case([rows], [3], io=io, v_scale=scale, gate=False, slow=False).check_rule()


def test_rule_whose_values_grow_and_shrink():
    c = Case([400], [3], d=64, io="f32", gate=False)
    c.v.mul_(torch.logspace(-3, 3, 400, device="cuda")[:, None, None])
    c.check_rule()


def test_heads_that_forget_at_once_and_never():
    c = Case([200], [3], d=64, vh=8, io="bf16", gate=False)
    c.a.copy_(torch.tensor([0.0, -1e-6, -1e-3, -0.1, -1.0, -10.0, -100.0, -1e4], device="cuda"))
    c.check_rule()


def test_rows_of_nothing():
    """k, q or v of zeros, and betas that are 0 or 1 in f32."""
    c = Case([150, 4], [3, 3], d=64, io="f32", gate=False)
    c.k[3:9] = 0
    c.k[100:150] = 0
    c.q[5] = 0
    c.v[20:30] = 0
    c.beta[40:60] = -200.0
    c.beta[60:62] = 200.0
    c.check_rule()


@pytest.mark.parametrize("rows", [4, 90])
def test_a_replay_leaves_what_the_rule_leaves(rows):
    """The states alone, after as many rows as are kept: bit for bit those of a rule over them."""
    n = 5
    take = [(3 * i) % (rows + 1) for i in range(n)]
    a, b = (Case([rows] * n, [3, 0, 8, 1, 9], d=128, io="bf16", take=take, fork=True) for _ in range(2))
    a.check_rule()
    b.step.replay(b.k, b.v, b.alpha, b.beta, b.a, b.dt)
    assert b.step.status() == 0 and torch.equal(a.state, b.state)


def test_a_verified_step_and_its_replay():
    """Drafts from one slot to another, some refused: the kept rows again from the old slot give the state that stepping them alone gives."""
    n = 6
    counts, kept = [4] * n, [1, 4, 2, 3, 1, 4]
    v = Case(counts, [9] * n, d=128, io="f32", fork=True)
    base = v.state.clone()
    v.run()
    full = v.state.clone()
    for b in range(n):
        assert torch.equal(full[v.slots[b]], base[v.slots[b]])                       # the old slots are as they were
    again = delta.Step(v.pool, v.row_start, v.lens, v.slot_t, v.rows, take=torch.tensor(kept, dtype=torch.int32, device="cuda"))
    again.replay(v.k, v.v, v.alpha, v.beta, v.a, v.dt)
    for b in range(n):
        if kept[b] == 4:
            assert torch.equal(v.state[v.slots[b]], full[v.to[b]])
        else:
            assert not torch.equal(v.state[v.slots[b]], full[v.to[b]])
    one = Case(counts, [9] * n, d=128, io="f32", fork=True, take=kept)
    want = one.want_rule()
    for b in range(n):
        assert bool(((v.state[v.slots[b]].double() - want[2][one.to[b]]).abs() <= want[3][one.to[b]]).all())


def test_a_sequence_alone_and_in_a_batch():
    """The same bits, whoever else is in the call."""
    c = Case([3, 100, 1, 64], [5, 0, 9, 3], d=64, io="bf16")
    out = c.check_rule()
    alone = Case([3, 100, 1, 64], [5, 0, 9, 3], d=64, io="bf16")
    r = 0
    for b, m in enumerate(c.counts):
        ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
        cut = lambda t: t[r:r + m]  # noqa: E731
        step = delta.Step(alone.pool, ints([0, m]), ints([m + c.past[b]]), ints([c.slots[b]]), m, max_rows=100)
        got = step.rule(*(cut(t) for t in (c.q, c.k, c.v, c.alpha, c.beta)), c.a, c.dt, z=cut(c.z), norm=c.norm)
        assert torch.equal(got, out[r:r + m]) and torch.equal(alone.state[c.slots[b]], c.state[c.slots[b]])
        r += m


def test_a_prompt_in_pieces():
    """Cut wherever, the state goes on; results to the tolerance of the whole."""
    c = Case([333], [0], d=128, io="bf16", gate=False)
    want, tol, pool, stol = c.want_rule()
    for cuts in ((64, 64, 205), (1, 300, 32), (333,)):
        p = Case([333], [0], d=128, io="bf16", gate=False)
        r = 0
        for m in cuts:
            ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
            cut = lambda t: t[r:r + m]  # noqa: E731
            step = delta.Step(p.pool, ints([0, m]), ints([r + m]), p.slot_t, m)
            got = step.rule(*(cut(t) for t in (p.q, p.k, p.v, p.alpha, p.beta)), p.a, p.dt)
            assert bool(((got.double() - want[r:r + m]).abs() <= tol[r:r + m]).all())
            r += m
        assert bool(((p.state.double() - pool).abs() <= stol).all())


def test_forks_read_one_slot():
    """Two sequences from one state (two answers to a prompt): each goes on in a slot of its own."""
    c = Case([3, 3, 70], [9, 9, 9], d=64, io="f32", slots=[1, 1, 1], to=[0, 2, 3], n_slots=5)
    c.check_rule()
    c = Case([3, 3, 70], [9, 9, 9], d=64, io="f32", slots=[1, 1, 1], to=[0, 2, 3], n_slots=5)
    c.check_conv()


def test_more_chunks_than_a_pass_takes():
    """6,300 rows of the benchmark's heads: more than 96 MB of what the chunks leave, so the chain goes on in a second pass; a short sequence in each."""
    c = Case([6150, 97, 53], [0, 4, 0], kh=16, vh=32, d=128, io="bf16", gate=False, seed=2)
    need = delta.C.c_int64()
    szlib.check(c.step.lib.sz_delta_scratch_bytes(c.step._c, c.step._b, szlib.TYPE_BF16, delta.C.byref(need)))
    assert need.value < 100 << 20
    c.check_rule()


@pytest.mark.parametrize("rows", [3, 70])
def test_pools_past_four_gigabytes(rows):
    """Slots 3 GB apart: a slot's place passes 32 bits."""
    c = Case([rows, rows], [5, 0], d=64, io="bf16", slots=[2, 1], to=[1, 2], n_slots=3)
    apart = 3 << 30
    mem = torch.zeros(2 * apart + (1 << 20), dtype=torch.uint8, device="cuda")
    state = mem.view(torch.float32).as_strided((3, c.vh, c.d, c.d), (apart // 4, c.d * c.d, c.d, 1))
    ref = Case([rows, rows], [5, 0], d=64, io="bf16", slots=[2, 0], to=[1, 2], n_slots=3)
    state.copy_(c.state)
    step = delta.Step(delta.States(c.kh, c.vh, c.d, state=state), c.row_start, c.lens, torch.tensor([2, 0], dtype=torch.int32, device="cuda"), c.rows,
                      to=torch.tensor([1, 2], dtype=torch.int32, device="cuda"))
    # (the second is new, and writes where the first reads: left out)
    out = torch.full((c.rows, c.vh, c.d), 77.0, dtype=c.io, device="cuda")
    step.rule(c.q, c.k, c.v, c.alpha, c.beta, c.a, c.dt, z=c.z, norm=c.norm, out=out)
    assert step.status() == 4
    got = ref.run()
    assert ref.step.status() == 4
    assert torch.equal(out[:rows], got[:rows]) and bool((out[rows:] == 77).all()) and torch.equal(state, ref.state)
    carried = mem.view(torch.bfloat16).as_strided((3, c.conv_k - 1, c.ch), (apart // 2, c.ch, 1))
    carried.copy_(c.carried)
    slots = torch.tensor([2, 1], dtype=torch.int32, device="cuda")
    conv = delta.Step(delta.States(c.kh, c.vh, c.d, conv=carried), c.row_start, c.lens, slots, c.rows)
    y = conv.conv(c.x, c.w)
    same = Case([rows, rows], [5, 0], d=64, io="bf16", slots=[2, 1], to=[2, 1], n_slots=3)
    assert torch.equal(y, same.step.conv(same.x, same.w)) and torch.equal(carried, same.carried) and conv.status() == 0


def test_decays_of_nothing():
    """Rows whose decay is 0, by an infinite or a huge exponent, among others: what was before them is gone, what comes after is as ever."""
    c = Case([150, 7], [3, 3], d=64, io="f32", gate=False)
    for r, x in ((4, math.inf), (70, 1e30), (71, math.inf), (100, 3e4), (140, math.inf), (152, math.inf)):
        c.alpha[r] = x
    c.a[0] = -1e-3
    c.check_rule()


@pytest.mark.parametrize("rows", [6, 150])
def test_what_is_not_finite_stays_in_its_sequence_and_head(rows):
    c, ref = (Case([rows] * 3, [4, 0, 2], kh=2, vh=4, d=64, io="bf16", fork=True) for _ in range(2))
    want = ref.run()
    c.v[rows + 2, 1] = math.nan
    c.v[rows + 3, 1, 5] = math.inf
    got = c.run()
    assert c.step.status() == 0
    bad = torch.zeros_like(got, dtype=torch.bool)
    bad[rows:2 * rows, 1] = True
    assert torch.equal(got[~bad], want[~bad]) and bool(got[rows + 2, 1].isnan().any())
    assert torch.equal(got[rows:rows + 2], want[rows:rows + 2]) or rows > 31
    for b in (0, 2):
        assert torch.equal(c.state[c.to[b]], ref.state[ref.to[b]])
    assert torch.equal(c.state[c.to[1]][[0, 2, 3]], ref.state[ref.to[1]][[0, 2, 3]])


def test_a_batch_whose_prompts_are_worth_chunks_later():
    """Many blocks: sequences of up to 111 rows go row by row, longer ones in chunks."""
    n = 20
    Case([1 + (i * 37) % 130 for i in range(n)], [5 * (i % 3) for i in range(n)], kh=16, vh=32, d=128, io="bf16", gate=False).check_rule()


def test_more_rows_than_were_said():
    """max_rows chooses kernels, not results: a sequence of more rows is right, row by row."""
    Case([100, 1, 40], [0, 4, 9], d=128, io="bf16", max_rows=4).check_rule()


# ---- tables that do not fit ---------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("rows", [3, 80])
@pytest.mark.parametrize("call", ["conv", "rule"])
def test_tables_that_do_not_fit_are_reported(rows, call):
    """The sequence is left out, the others are not; nothing outside the pool or the rows is touched (the kernels check every entry before they use it)."""
    def go(code, slots=(1, 2, 3), to=None, starts=None, untouched=(), past=(5, 5, 5)):
        c = Case([rows] * 3, list(past), d=64, io="f32", slots=list(slots), to=None if to is None else list(to), n_slots=6, max_rows=None if rows > 3 else 3)
        if starts is not None:
            c.row_start.copy_(torch.tensor(starts, dtype=torch.int32))
        state, carried = c.state.clone(), c.carried.clone()
        y = torch.full((c.rows, c.ch), 77.0, device="cuda")
        out = torch.full((c.rows, c.vh, c.d), 77.0, device="cuda")
        if call == "conv":
            c.step.conv(c.x, c.w, out=y)
            got = y
        else:
            c.run(out)
            got = out
        assert c.step.status() == code
        for b in untouched:
            assert bool((got[b * rows:(b + 1) * rows] == 77).all())
        if starts is None:
            for b in set(range(3)) - set(untouched):
                assert bool((got[b * rows:(b + 1) * rows] != 77).any())
        return c, state, carried
    for bad in (-1, 6, 2 ** 31 - 1, -2 ** 31):
        c, state, carried = go(1, slots=(1, bad, 3), untouched=(1,))
        assert torch.equal(c.state[2], state[2]) and torch.equal(c.carried[2], carried[2])
        go(1, to=(1, bad, 3), untouched=(1,))
    go(0, slots=(1, -1, 3), to=(1, 2, 3), past=(5, 0, 5))            # (a new one comes from nowhere)
    go(4, slots=(1, 1, 3), untouched=(1,))                            # one slot twice
    go(4, to=(4, 4, 5), untouched=(1,))
    go(4, to=(2, 4, 5), untouched=(1,))                               # .. written by the first, read by the second
    go(4, to=(4, 1, 5), untouched=(1,))                               # .. read by the first, written by the second
    go(2, starts=[0, rows, 2 * rows, 3 * rows + 1], untouched=(2,))
    go(2, starts=[0, rows, 2 * rows, 2 ** 31 - 1], untouched=(2,))
    go(2, starts=[-5, rows, 2 * rows, 3 * rows], untouched=(0,))
    go(2, starts=[0, 2 * rows, rows, rows])
    go(2, starts=[3 * rows + 5, 3 * rows + 6, 3 * rows + 7, 3 * rows + 8], untouched=(0, 1, 2))


# ---- streams, graphs, the layer as it is used ------------------------------------------------------------------------------------------------
def test_a_captured_step_reads_the_tables_as_they_are():
    c = Case([2, 100, 3], [5, 0, 9], d=128, io="bf16", gate=True)
    ref = Case([2, 100, 3], [5, 0, 9], d=128, io="bf16", gate=True)
    y, out = torch.empty_like(c.x), torch.empty(c.rows, c.vh, c.d, dtype=c.io, device="cuda")
    kd = c.kh * c.d

    def layer(s):
        s.step.conv(s.x, s.w, out=y)
        q, k, v = (t.unflatten(1, (-1, s.d)) for t in y.split([kd, kd, s.vh * s.d], 1))
        s.step.rule(q, k, v, s.alpha, s.beta, s.a, s.dt, z=s.z, norm=s.norm, out=out)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        state, carried = c.state.clone(), c.carried.clone()
        layer(c)
        c.state.copy_(state)
        c.carried.copy_(carried)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            layer(c)
        for starts, lens in (([0, 2, 102, 105], [7, 100, 12]), ([0, 70, 71, 105], [70, 9, 50]), ([0, 0, 1, 2], [0, 4, 5])):
            for s in (c, ref):
                s.row_start.copy_(torch.tensor(starts, dtype=torch.int32))
                s.lens.copy_(torch.tensor(lens, dtype=torch.int32))
            graph.replay()
            got = out[:starts[-1]].clone()
            layer(ref)
            assert torch.equal(got, out[:starts[-1]]) and torch.equal(c.state, ref.state) and torch.equal(c.carried, ref.carried)
    side.synchronize()
    assert c.step.status() == 0 and ref.step.status() == 0


def test_two_steps_at_once():
    """A scratch each, two streams: nothing is shared but the pool."""
    base = [Case([90, 3, 150], [4, 0, 9], d=64, io="bf16", seed=s) for s in (1, 2)]
    want = [b.check_rule() for b in base]
    two = [Case([90, 3, 150], [4, 0, 9], d=64, io="bf16", seed=s) for s in (1, 2)]
    streams = [torch.cuda.Stream() for _ in two]
    torch.cuda.synchronize()
    got = []
    for c, st in zip(two, streams):
        with torch.cuda.stream(st):
            got.append(c.run())
    torch.cuda.synchronize()
    for g, w, c, b in zip(got, want, two, base):
        assert torch.equal(g, w) and torch.equal(c.state, b.state)


def test_a_layer_behind_its_convolution_and_a_step_to_its_tokens():
    """Convolution, rule, a head's logits, a draw and its score, twice in a row with the states carried: as a host's step runs them, against 64 bits."""
    n, vocab = 3, 1000
    c = Case([70, 5, 1], [0, 0, 0], d=64, io="f32", seed=5)
    head = c.rnd(c.vh * c.d, vocab) / math.sqrt(c.vh * c.d)
    kd = c.kh * c.d
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    states = [torch.zeros(c.vh, c.d, c.d, dtype=torch.float64, device="cuda") for _ in range(n)]
    past = [torch.zeros(c.conv_k - 1, c.ch, dtype=torch.float64, device="cuda") for _ in range(n)]
    counts, lens = [70, 5, 1], [70, 5, 1]
    for _ in range(2):
        R = sum(counts)
        starts = [0]
        for m in counts:
            starts.append(starts[-1] + m)
        step = delta.Step(c.pool, ints(starts), ints(lens), c.slot_t, R)
        x, alpha, beta, z = c.rnd(R, c.ch), c.rnd(R, c.vh), c.rnd(R, c.vh), c.rnd(R, c.vh, c.d)
        y = step.conv(x, c.w)
        q, k, v = (t.unflatten(1, (-1, c.d)) for t in y.split([kd, kd, c.vh * c.d], 1))
        out = step.rule(q, k, v, alpha, beta, c.a, c.dt, z=z, norm=c.norm)
        last = [s - 1 for s in starts[1:]]
        logits = out[last].flatten(1) @ head
        u = torch.rand(n, dtype=torch.float64, device="cuda")
        tokens = sampling.sample_rows(logits, u)
        score = sampling.logprob_rows(logits, tokens, top=4)
        assert step.status() == 0
        dec = torch.exp(c.a.double() * torch.nn.functional.softplus(alpha.double() + c.dt.double()))
        rows = []
        for b, m in enumerate(counts):
            seq = torch.cat([past[b], x[starts[b]:starts[b + 1]].double()])
            s = (seq.unfold(0, c.conv_k, 1) * c.w.double()).sum(-1)
            s = s * torch.sigmoid(s)
            past[b] = seq[-(c.conv_k - 1):]
            for j in range(m):
                r = starts[b] + j
                unit = lambda t: t / torch.sqrt(t.square().sum(-1, keepdim=True) + 1e-6)  # noqa: E731
                of = [h % c.kh for h in range(c.vh)]
                qh, kk = unit(s[j, :kd].view(c.kh, c.d))[of] / math.sqrt(c.d), unit(s[j, kd:2 * kd].view(c.kh, c.d))[of]
                S = states[b] * dec[r][:, None, None]
                dl = (s[j, 2 * kd:].view(c.vh, c.d) - torch.einsum("hij,hi->hj", S, kk)) * torch.sigmoid(beta[r].double())[:, None]
                states[b] = S + kk[:, :, None] * dl[:, None, :]
                o = torch.einsum("hij,hi->hj", states[b], qh)
            o = o * torch.rsqrt(o.square().mean(-1, keepdim=True) + 1e-6) * c.norm.double() * torch.sigmoid(z[starts[b + 1] - 1].double())
            rows.append(o.flatten())
        lp = torch.log_softmax(torch.stack(rows) @ head.double(), 1)
        # (an output is off by 2^-14 of its head's values at 70 rows by the rule's tolerance, a logit by 16 of those with signs that differ: 2^-10 is wide)
        assert float((score.logprob.double() - lp.gather(1, tokens.long()[:, None])[:, 0]).abs().max()) < 2.0 ** -10
        assert float((score.entropy.double() + (lp.exp() * lp).sum(1)).abs().max()) < 2.0 ** -9
        counts, lens = [1, 2, 1], [lens[0] + 1, lens[1] + 2, lens[2] + 1]
