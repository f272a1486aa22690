"""The DeltaNet layer of a served step (`sz_delta_*`): sequences whose states and carried rows lie in slots of a pool; the causal convolution and the
gated delta rule over their rows, single tokens, drafts and prompts."""
import ctypes as C

import torch

from . import lib as szlib
from .paged import _HERE, TYPES
from .sampling import _raw_stream


class DeltaPoolC(C.Structure):
    """struct sz_delta_pool"""
    _fields_ = [(n, C.c_int32) for n in ("n_slots", "k_heads", "v_heads", "head_dim", "grouped", "conv_k", "conv_type", "reserved")] + \
               [("state", C.c_uint64), ("conv", C.c_uint64), ("state_stride", C.c_int64), ("conv_stride", C.c_int64)]


class DeltaBatchC(C.Structure):
    """struct sz_delta_batch"""
    _fields_ = [(n, C.c_int32) for n in ("n_seq", "rows", "max_rows", "reserved")] + [(n, C.c_uint64) for n in ("row_start", "lens", "from_", "to", "take")]


class DeltaGatesC(C.Structure):
    """struct sz_delta_gates"""
    _fields_ = [("a", C.c_uint64), ("dt", C.c_uint64), ("norm", C.c_uint64), ("eps", C.c_float), ("reserved", C.c_float)]


class States:
    """The pool of one layer.  state float32 [slots, v_heads, head_dim, head_dim] (key dimension, then value dimension), conv [slots, rows of the convolution - 1,
    (2 k_heads + v_heads) head_dim] of float32, float16 or bfloat16, the oldest row first; a slot contiguous, slots any distance apart.  Either may be None where
    only the other's call is made.  grouped: the value heads of a key head lie side by side (else they are tiled over the key heads)."""

    def __init__(self, k_heads, v_heads, head_dim, state=None, conv=None, grouped=False):
        if state is None and conv is None:
            raise ValueError("neither states nor carried rows")
        ch = (2 * k_heads + v_heads) * head_dim
        one = state if state is not None else conv
        self.state, self.conv, self.device = state, conv, one.device
        self.kh, self.vh, self.hd, self.channels, self.conv_k = k_heads, v_heads, head_dim, ch, 0
        self.c = DeltaPoolC(n_slots=one.shape[0], k_heads=k_heads, v_heads=v_heads, head_dim=head_dim, grouped=int(bool(grouped)))
        for name, t, shape in (("state", state, (v_heads, head_dim, head_dim)), ("conv", conv, None)):
            if t is None:
                continue
            if shape is None:
                shape = (t.shape[1] if t.dim() == 3 else 1, ch)
            if one.shape[0] < 1 or t.shape != (one.shape[0],) + shape or t.device != self.device or not t[0].is_contiguous() or (t.shape[0] > 1 and t.stride(0) < t[0].numel()):
                raise ValueError("%s: [%d, %s], a slot contiguous" % (name, one.shape[0], ", ".join(map(str, shape))))
            if t.dtype not in TYPES or (name == "state" and t.dtype != torch.float32):
                raise ValueError("%s: %s" % (name, "float32" if name == "state" else "float32, float16 or bfloat16"))
            setattr(self.c, name, t.data_ptr())
            setattr(self.c, name + "_stride", (t.stride(0) if t.shape[0] > 1 else t[0].numel()) * t.element_size())
        if conv is not None:
            self.conv_k = self.c.conv_k = conv.shape[1] + 1
            self.c.conv_type = TYPES[conv.dtype]


class Step:
    """The tables of a batch over a pool, and the scratch of its calls.  row_start int32 [sequences + 1], lens int32 [sequences] (all positions, the step's rows included:
    a paged step's tables), slots int32 [sequences]: where a sequence's state is; to: where it goes (None: the same); take: how many of its rows count (None: all).  They
    are the caller's tensors: change their values from step to step, behind the calls that read them.  max_rows: the most rows that a sequence has (it chooses
    kernels).  Calls on one Step follow one another on a stream - the one it was made on, or another that waits for that -, and it is kept until they are done; what
    may overlap needs a Step each.  Each has a scratch of its own: up to 96 MB where a sequence may have many rows, else 256 bytes."""

    def __init__(self, states, row_start, lens, slots, rows, to=None, take=None, max_rows=None):
        self.lib = szlib.load()
        n = lens.shape[0]
        for name, t, size in (("row_start", row_start, n + 1), ("lens", lens, n), ("slots", slots, n), ("to", to, n), ("take", take, n)):
            if t is None and name in ("to", "take"):
                continue
            if t is None or t.dtype != torch.int32 or t.shape != (size,) or not t.is_contiguous() or t.device != states.device:
                raise ValueError("%s: a contiguous int32 tensor of %d on the pool's device" % (name, size))
        if states.device.type != "cuda":
            raise ValueError("the pool and tables lie on a GPU, not on %s" % states.device)
        self.pool, self.rows, self.device, self._index = states, rows, states.device, states.device.index
        self._keep = (row_start, lens, slots, to, take)
        p = states
        self._wide, self._narrow, self._heads, self._chan = (rows, p.vh, p.hd), (rows, p.kh, p.hd), (rows, p.vh), (rows, p.channels)
        self._in = (p.hd, 1)
        ptr = lambda t: 0 if t is None else t.data_ptr()  # noqa: E731
        self.b = DeltaBatchC(n_seq=n, rows=rows, max_rows=max_rows or 0, row_start=ptr(row_start), lens=ptr(lens), from_=ptr(slots), to=ptr(to), take=ptr(take))
        self._c, self._b = C.byref(states.c), C.byref(self.b)
        need = C.c_int64()
        szlib.check(self.lib.sz_delta_scratch_bytes(self._c, self._b, szlib.TYPE_F32, C.byref(need)))      # (no type of rows needs more)
        with self._here():
            self._mem = torch.empty(need.value + 256, dtype=torch.uint8, device=self.device)
            self.scratch, self.scratch_bytes = self._mem.data_ptr() + (-self._mem.data_ptr()) % 256, need.value
            szlib.check(self.lib.sz_delta_status(self.scratch, 1, None, self._stream()))

    def _here(self):
        """Makes the pool's device the current one, where another is."""
        return _HERE if torch.cuda.current_device() == self._index else torch.cuda.device(self._index)

    def _stream(self):
        return _raw_stream(self._index)

    def _rows(self, name, t, shape, inner, dtype):
        """Checks [rows, *shape] of dtype, what belongs to a row side by side (strides `inner`); returns its address and the stride of rows."""
        st = t.stride()
        if t.dtype is dtype and dtype in TYPES and t.shape == shape and st[1:] == inner and t.get_device() == self._index and st[0] >= shape[1] * inner[0]:
            return t.data_ptr(), st[0]
        if t.shape != shape or t.device != self.device:
            raise ValueError("%s: %s on the pool's device" % (name, list(shape)))
        if t.dtype is not dtype or dtype not in TYPES:
            raise ValueError("%s: float32, float16 or bfloat16, the same for all rows of a call" % name)
        if any(n > 1 and a != b for n, a, b in zip(shape[1:], st[1:], inner)):
            raise ValueError("%s: heads side by side, the last dimension contiguous" % name)
        width = shape[1] * inner[0]
        if self.rows > 1 and st[0] < width:
            raise ValueError("%s: rows that overlap" % name)
        return t.data_ptr(), st[0] if self.rows > 1 else width

    def _f32(self, name, t, *shape):
        if t.dtype is not torch.float32 or t.shape != shape or not t.is_contiguous() or t.get_device() != self._index:
            raise ValueError("%s: contiguous float32 %s on the pool's device" % (name, list(shape)))
        return t.data_ptr()

    def conv(self, x, w, bias=None, out=None):
        """silu of the causal convolution of x [rows, channels] with w float32 [channels, rows of the convolution] (and bias float32 [channels]), a sequence's earlier rows
        from its slot; the last ones are carried on.  Returns [rows, channels]: queries, keys and values side by side."""
        p = self.pool
        if p.conv is None:
            raise ValueError("the pool has no carried rows")
        xp, xs = self._rows("x", x, self._chan, (1,), x.dtype)
        if out is None:
            out = torch.empty((self.rows, p.channels), dtype=x.dtype, device=x.device)
        op, os = self._rows("out", out, self._chan, (1,), x.dtype)
        wp, bp = self._f32("w", w, p.channels, p.conv_k), 0 if bias is None else self._f32("bias", bias, p.channels)
        with self._here():
            rc = self.lib.sz_delta_conv(self._c, self._b, TYPES[x.dtype], xp, xs, wp, bp, op, os, self.scratch, self.scratch_bytes, self._stream())
        if rc:
            szlib.check(rc)
        return out

    def rule(self, q, k, v, alpha, beta, a, dt, z=None, norm=None, eps=1e-6, out=None):
        """The gated delta rule over the rows.  q, k [rows, k_heads, head_dim] (normed here), v [rows, v_heads, head_dim], alpha, beta [rows, v_heads] as their projections give them;
        a, dt float32 [v_heads]: a row's decay is exp(a softplus(alpha + dt)).  z (as v) and norm (float32 [head_dim]): the outputs are normed per head and
        times sigmoid(z).  Returns [rows, v_heads, head_dim]; the states move on."""
        p, dtype = self.pool, k.dtype
        if out is None:
            out = torch.empty((self.rows, p.vh, p.hd), dtype=dtype, device=k.device)
        return self._rule(self._rows("q", q, self._narrow, self._in, dtype), k, v, alpha, beta, a, dt, z, norm, eps, out)

    def replay(self, k, v, alpha, beta, a, dt):
        """The states alone, without outputs (after a refusal of drafts: `take` says how many rows are kept)."""
        self._rule((0, 0), k, v, alpha, beta, a, dt, None, None, 0.0, None)

    def _rule(self, q, k, v, alpha, beta, a, dt, z, norm, eps, out):
        p, dtype = self.pool, k.dtype
        if p.state is None:
            raise ValueError("the pool has no states")
        if (z is None) != (norm is None):
            raise ValueError("z and norm come together")
        rows, wide, inner = self._rows, self._wide, self._in
        args = q + rows("k", k, self._narrow, inner, dtype) + rows("v", v, wide, inner, dtype) + rows("alpha", alpha, self._heads, (1,), dtype) + rows("beta", beta, self._heads, (1,), dtype)
        args += (0, 0) if z is None else rows("z", z, wide, inner, dtype)
        args += (0, 0) if out is None else rows("out", out, wide, inner, dtype)
        gates = DeltaGatesC(self._f32("a", a, p.vh), self._f32("dt", dt, p.vh), 0 if norm is None else self._f32("norm", norm, p.hd), eps, 0.0)
        io = TYPES[dtype]
        with self._here():
            rc = self.lib.sz_delta_rows(self._c, self._b, C.byref(gates), io, *args, self.scratch, self.scratch_bytes, self._stream())
        if rc:
            szlib.check(rc)
        return out

    def status(self):
        """What the calls so far have met (synchronises): 0, or the bits of sz_delta_status."""
        code = C.c_int()
        with self._here():
            rc = self.lib.sz_delta_status(self.scratch, 0, C.byref(code), self._stream())
        if rc not in (szlib.OK, szlib.E_DEVICE):
            szlib.check(rc)
        return code.value
