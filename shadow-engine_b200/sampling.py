"""Draws over whole rows of logits on the device (`sz_sample_rows`): the sampler of the reference (crates/shadowzero-serve/src/sampler.rs:112-210)
for many rows at once, every row with settings of its own, from uniform numbers the caller gives."""
import torch

from . import lib as szlib
from .paged import TYPES


def sample_rows(logits, uniform, temperature=None, top_k=None, top_p=None, min_p=None, out=None, prob=None):
    """logits [rows, vocab] (float32, float16 or bfloat16, vocab <= 262144), uniform float64 [rows] in [0, 1); temperature, top_p, min_p float32
    [rows], top_k int32 [rows], None: 1, 1, 0 and no limit.  Returns the tokens, int32 [rows]; prob (float32 [rows]) receives each
    token's probability among those that were left."""
    L = szlib.load()
    if logits.dim() != 2 or logits.dtype not in TYPES or (logits.shape[1] > 1 and logits.stride(1) != 1):
        raise ValueError("logits: [rows, vocab] of float32, float16 or bfloat16, rows contiguous")
    rows, dev = logits.shape[0], logits.device
    if out is None:
        out = torch.empty(rows, dtype=torch.int32, device=dev)
    for name, t, dt in (("uniform", uniform, torch.float64), ("temperature", temperature, torch.float32), ("top_k", top_k, torch.int32), ("top_p", top_p, torch.float32),
                        ("min_p", min_p, torch.float32), ("out", out, torch.int32), ("prob", prob, torch.float32)):
        if t is not None and (t.dtype != dt or t.shape != (rows,) or not t.is_contiguous() or t.device != dev):
            raise ValueError("%s: %s [%d] on the logits' device" % (name, dt, rows))
    p = lambda t: 0 if t is None else t.data_ptr()  # noqa: E731
    with torch.cuda.device(dev):
        szlib.check(L.sz_sample_rows(TYPES[logits.dtype], logits.data_ptr(), max(logits.stride(0), logits.shape[1]), rows, logits.shape[1], p(temperature), p(top_k),
                                     p(top_p), p(min_p), uniform.data_ptr(), out.data_ptr(), p(prob), torch.cuda.current_stream(dev).cuda_stream))
    return out
