"""Draws over whole rows of logits on the device (`sz_sample_rows`): the sampler of the reference (crates/shadowzero-serve/src/sampler.rs:112-210)
for many rows at once, every row with settings of its own, from uniform numbers the caller gives."""
import torch

from . import lib as szlib
from .paged import _HERE, TYPES


def sample_rows(logits, uniform, temperature=None, top_k=None, top_p=None, min_p=None, out=None, prob=None):
    """logits [rows, vocab] (float32, float16 or bfloat16, vocab <= 262144), uniform float64 [rows] in [0, 1); temperature, top_p, min_p float32
    [rows], top_k int32 [rows], None: 1, 1, 0 and no limit.  Returns the tokens, int32 [rows]; prob (float32 [rows]) receives each
    token's probability among those that were left."""
    L = szlib.load()
    if logits.dim() != 2 or logits.dtype not in TYPES or (logits.shape[1] > 1 and logits.stride(1) != 1):
        raise ValueError("logits: [rows, vocab] of float32, float16 or bfloat16, rows contiguous")
    (rows, vocab), stride, dev = logits.shape, logits.stride(0), logits.device
    if stride < vocab:
        if rows > 1:
            raise ValueError("logits: rows that overlap")
        stride = vocab
    if out is None:
        out = torch.empty(rows, dtype=torch.int32, device=dev)
    of = (rows,)

    def at(name, t, dt):
        if t is None:
            return 0
        if t.dtype != dt or t.shape != of or t.device != dev or not t.is_contiguous():
            raise ValueError("%s: %s [%d] on the logits' device" % (name, dt, rows))
        return t.data_ptr()

    if uniform is None:
        raise ValueError("uniform: a number in [0, 1) a row")
    f32 = torch.float32
    ptrs = (at("temperature", temperature, f32), at("top_k", top_k, torch.int32), at("top_p", top_p, f32), at("min_p", min_p, f32), at("uniform", uniform, torch.float64),
            at("out", out, torch.int32), at("prob", prob, f32))
    if dev.type != "cuda":
        raise ValueError("logits, settings and results lie on a GPU, not on %s" % dev)
    with _HERE if torch.cuda.current_device() == dev.index else torch.cuda.device(dev):
        rc = L.sz_sample_rows(TYPES[logits.dtype], logits.data_ptr(), stride, rows, vocab, *ptrs, torch.cuda.current_stream(dev.index).cuda_stream)
    if rc:
        szlib.check(rc)
    return out
