"""A cache in pages (`sz_paged_*`): rows are appended to it and attend to it, over a prefix that the whole batch shares, too."""
import contextlib
import ctypes as C
import math

import torch

from . import lib as szlib

_HERE = contextlib.nullcontext()
TYPES = {torch.float32: szlib.TYPE_F32, torch.float16: szlib.TYPE_F16, torch.bfloat16: szlib.TYPE_BF16}


class PagedCacheC(C.Structure):
    """struct sz_paged_cache"""
    _fields_ = [("type", C.c_int32), ("n_kv_head", C.c_int32), ("head_dim", C.c_int32), ("page_size", C.c_int32), ("n_pages", C.c_int32),
                ("reserved", C.c_int32), ("k", C.c_uint64), ("v", C.c_uint64), ("page_stride", C.c_int64), ("head_stride", C.c_int64), ("pos_stride", C.c_int64)]


class PagedBatchC(C.Structure):
    """struct sz_paged_batch"""
    _fields_ = [("n_seq", C.c_int32), ("rows", C.c_int32), ("max_pages", C.c_int32), ("shared_len", C.c_int32), ("pages", C.c_uint64),
                ("row_start", C.c_uint64), ("lens", C.c_uint64), ("shared_pages", C.c_uint64)]


class PagedRopeC(C.Structure):
    """struct sz_paged_rope"""
    _fields_ = [("dims", C.c_int32), ("eps", C.c_float), ("theta", C.c_double), ("q_norm", C.c_uint64), ("k_norm", C.c_uint64)]


def head_bytes(head_dim):
    """Bytes of a packed head (SZ_TYPE_Q8_KV): head_dim codes, then head_dim / 32 f16 scales, padded to 16 bytes."""
    return head_dim + ((head_dim // 32 * 2 + 15) & ~15)


class Cache:
    """The pools of one layer: k and v [pages, kv heads, positions a page, head_dim] of f16 or bf16, or of uint8 packed heads
    [.., head_bytes(head_dim)].  Any order of the first three dimensions (a transposed view is one), the last contiguous."""

    def __init__(self, k, v, head_dim):
        if k.dim() != 4 or v.shape != k.shape or v.stride() != k.stride() or v.dtype != k.dtype or v.device != k.device:
            raise ValueError("k and v: two pools of one shape, type and layout, [pages, kv heads, positions, head]")
        packed = k.dtype == torch.uint8
        if not packed and k.dtype not in (torch.float16, torch.bfloat16):
            raise ValueError("pools of float16, bfloat16 or uint8 (packed heads)")
        if k.stride(3) != 1 or k.shape[3] != (head_bytes(head_dim) if packed else head_dim):
            raise ValueError("a head is %d contiguous elements" % (head_bytes(head_dim) if packed else head_dim))
        self.k, self.v, self.device, self.head_dim = k, v, k.device, head_dim
        if any(n > 1 and st < k.shape[3] for n, st in zip(k.shape, k.stride()[:3])):
            raise ValueError("pools whose heads overlap")
        e = k.element_size()
        head = k.shape[3] * e
        # (of a dimension of one the stride says nothing)
        page_stride, head_stride = (st * e if n > 1 else head for n, st in zip(k.shape[:2], k.stride()[:2]))
        self.c = PagedCacheC(type=szlib.TYPE_Q8_KV if packed else TYPES[k.dtype], n_kv_head=k.shape[1], head_dim=head_dim, page_size=k.shape[2], n_pages=k.shape[0],
                             k=k.data_ptr(), v=v.data_ptr(), page_stride=page_stride, head_stride=head_stride, pos_stride=k.stride(2) * e)


class Step:
    """The tables of a batch over a cache, and the scratch of its calls.  pages int32 [sequences, pages of one], row_start int32 [sequences + 1],
    lens int32 [sequences] (all positions, the step's rows included) are the caller's tensors: change their values from step to step, behind the
    calls that read them.
    shared_pages int32: the pages of the first shared_len positions, the same for all sequences.  Calls on one Step follow one another on
    a stream - the one it was made on, or another that waits for that -, and it is kept until they are done; what may overlap needs a Step each."""

    def __init__(self, cache, pages, row_start, lens, rows, n_head, shared_pages=None, shared_len=0):
        self.lib = szlib.load()
        for name, t, dims in (("pages", pages, 2), ("row_start", row_start, 1), ("lens", lens, 1)) + ((("shared_pages", shared_pages, 1),) if shared_len else ()):
            if t is None or t.dtype != torch.int32 or t.dim() != dims or not t.is_contiguous() or t.device != cache.device:
                raise ValueError("%s: a contiguous int32 tensor of %d dimension(s) on the cache's device" % (name, dims))
        n = lens.shape[0]
        if pages.shape[0] != n or row_start.shape[0] != n + 1:
            raise ValueError("pages and row_start: one row a sequence, one entry more than sequences")
        if shared_len and shared_pages.shape[0] * cache.c.page_size < shared_len:
            raise ValueError("shared_pages hold %d positions, shared_len is %d" % (shared_pages.shape[0] * cache.c.page_size, shared_len))
        if cache.device.type != "cuda":
            raise ValueError("the pools and tables lie on a GPU, not on %s" % cache.device)
        self.cache, self.n_head, self.rows, self.device = cache, n_head, rows, cache.device
        self.hd, self._index = cache.head_dim, cache.device.index
        self.nkv, self._scale = cache.c.n_kv_head, 1 / math.sqrt(cache.head_dim)
        self._keep = (pages, row_start, lens, shared_pages)
        self.b = PagedBatchC(n_seq=n, rows=rows, max_pages=pages.shape[1], shared_len=shared_len, pages=pages.data_ptr(), row_start=row_start.data_ptr(),
                             lens=lens.data_ptr(), shared_pages=shared_pages.data_ptr() if shared_len else 0)
        need = C.c_int64()
        self._c, self._b = C.byref(cache.c), C.byref(self.b)
        szlib.check(self.lib.sz_paged_scratch_bytes(self._c, self._b, n_head, C.byref(need)))
        with torch.cuda.device(self.device):
            self._mem = torch.empty(need.value + 256, dtype=torch.uint8, device=self.device)
            self.scratch, self.scratch_bytes = self._mem.data_ptr() + (-self._mem.data_ptr()) % 256, need.value
            szlib.check(self.lib.sz_paged_status(self.scratch, 1, None, self._stream()))

    def _here(self):
        """Makes the cache's device the current one, where another is."""
        return _HERE if torch.cuda.current_device() == self._index else torch.cuda.device(self._index)

    def _stream(self):
        return torch.cuda.current_stream(self._index).cuda_stream

    def _rows(self, name, t, heads, dtype, apart=False):
        """Checks [rows, heads, head_dim] of dtype; returns its address and its strides of rows and (apart: any) heads."""
        hd = self.hd
        if t.shape != (self.rows, heads, hd) or t.device != self.device:
            raise ValueError("%s: [%d, %d, %d] on the cache's device" % (name, self.rows, heads, hd))
        if t.dtype is not dtype or dtype not in TYPES:
            raise ValueError("%s: float32, float16 or bfloat16, the same for all rows of a call" % name)
        row, head, one = t.stride()
        if one != 1:
            raise ValueError("%s: the last dimension contiguous" % name)
        if head != hd:
            if heads == 1:
                head = hd
            elif not apart or head < hd:
                raise ValueError("%s: heads %s" % (name, "that overlap" if apart else "side by side"))
        if self.rows == 1:
            row = (heads - 1) * head + hd
        elif row < (heads - 1) * head + hd:
            raise ValueError("%s: rows that overlap" % name)
        return t.data_ptr(), row, head

    def append(self, k, v, q=None, q_out=None, rope_dims=0, theta=1e4, q_norm=None, k_norm=None, eps=1e-6):
        """Stores the rows' keys (normed, turned) and values at their positions; returns the rows' queries, normed and turned (None without q).
        k, v [rows, kv heads, head_dim]; q [rows, heads, head_dim] (any stride of heads); q_norm, k_norm float32 [head_dim]."""
        hd, nkv, dt = self.hd, self.nkv, k.dtype
        kp, ks, _ = self._rows("k", k, nkv, dt)
        vp, vs, _ = self._rows("v", v, nkv, dt)
        qp = qs = qh = op = os = qn = kn = 0
        if q is not None:
            qp, qs, qh = self._rows("q", q, self.n_head, dt, True)
            if q_out is None:
                q_out = torch.empty(q.shape, dtype=dt, device=q.device)
            op, os, _ = self._rows("q_out", q_out, self.n_head, dt)
        elif q_out is not None:
            raise ValueError("q_out without q")
        if q_norm is not None:
            qn = self._norm(q_norm, hd)
        if k_norm is not None:
            kn = self._norm(k_norm, hd)
        rope = PagedRopeC(rope_dims, eps, theta, qn, kn)
        with self._here():
            rc = self.lib.sz_paged_append(self._c, self._b, C.byref(rope), TYPES[dt], self.n_head, kp, ks, vp, vs, qp, qs, qh, op, os, self.scratch, self.scratch_bytes,
                                          self._stream())
        if rc:
            szlib.check(rc)
        return q_out

    def _norm(self, w, hd):
        if w.dtype != torch.float32 or w.shape != (hd,) or w.stride(0) != 1 or w.device != self.device:
            raise ValueError("norm weights: float32 [%d] on the cache's device" % hd)
        return w.data_ptr()

    def attend(self, q, out=None, scale=None, gate=None, lse=None):
        """Attention of the rows over their sequences' positions up to their own, shared ones first.  q [rows, heads, head_dim]; gate: the
        same (any stride of heads), out *= sigmoid(gate); lse float32 [rows, heads] receives the logarithm of the softmax's denominator; scale 1 / sqrt(head_dim)."""
        dt = q.dtype
        qp, qs, _ = self._rows("q", q, self.n_head, dt)
        if out is None:
            out = torch.empty(q.shape, dtype=dt, device=q.device)
        op, os, _ = self._rows("out", out, self.n_head, dt)
        gp = gs = gh = lp = 0
        if gate is not None:
            gp, gs, gh = self._rows("gate", gate, self.n_head, dt, True)
        if lse is not None:
            if lse.dtype != torch.float32 or lse.shape != (self.rows, self.n_head) or not lse.is_contiguous() or lse.device != self.device:
                raise ValueError("lse: float32 [%d, %d] on the cache's device" % (self.rows, self.n_head))
            lp = lse.data_ptr()
        with self._here():
            rc = self.lib.sz_paged_attend(self._c, self._b, TYPES[dt], self.n_head, self._scale if scale is None else scale, qp, qs, gp, gs, gh, op, os, lp, self.scratch,
                                          self.scratch_bytes, self._stream())
        if rc:
            szlib.check(rc)
        return out

    def status(self):
        """What the calls so far have met (synchronises): 0, or the bits of sz_paged_status."""
        code = C.c_int()
        with self._here():
            rc = self.lib.sz_paged_status(self.scratch, 0, C.byref(code), self._stream())
        if rc not in (szlib.OK, szlib.E_DEVICE):
            szlib.check(rc)
        return code.value
