"""Draws over whole rows of logits on the device (`sz_sample_rows`): the sampler of the reference (crates/shadowzero-serve/src/sampler.rs:112-210)
for many rows at once, every row with settings of its own, from uniform numbers the caller gives; and what given tokens weigh in whole rows (`sz_logprob_rows`)."""
import collections

import torch

from . import lib as szlib
from .paged import _HERE, TYPES

try:                                                     # (the stream's handle alone: an object for it takes 3 us)
    from torch._C import _cuda_getCurrentRawStream as _raw_stream
except ImportError:
    def _raw_stream(index):
        return torch.cuda.current_stream(index).cuda_stream


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


LogProbs = collections.namedtuple("LogProbs", "logprob rank entropy top_ids top_logprobs")


def logprob_rows(logits, tokens=None, top=0, temperature=None, out=None):
    """Log probabilities of given tokens.  logits [rows, vocab] (float32, float16 or bfloat16, vocab <= 262144), tokens int32 [rows] (None: none are given; an id outside the
    vocabulary, a padded row's: -inf and rank -1), temperature float32 [rows] (None: 1).  Returns LogProbs: logprob float32 [rows], rank int32 [rows] (0: the row's best),
    entropy float32 [rows], top_ids int32 and top_logprobs float32 [rows, top], the row's largest logits, top <= 64.  out: LogProbs of an earlier call with as many
    rows, to be written again."""
    L = szlib.load()
    if logits.dim() != 2 or logits.dtype not in TYPES or (logits.shape[1] > 1 and logits.stride(1) != 1):
        raise ValueError("logits: [rows, vocab] of float32, float16 or bfloat16, rows contiguous")
    (rows, vocab), stride, dev, index = logits.shape, logits.stride(0), logits.device, logits.get_device()
    if stride < vocab:
        if rows > 1:
            raise ValueError("logits: rows that overlap")
        stride = vocab
    f32, i32 = torch.float32, torch.int32
    if out is None:
        new = lambda dt, *of: torch.empty(of, dtype=dt, device=dev)  # noqa: E731
        out = LogProbs(None if tokens is None else new(f32, rows), None if tokens is None else new(i32, rows), new(f32, rows), new(i32, rows, top), new(f32, rows, top))

    def at(name, t, dt, *of):
        if t is None:
            return 0
        if t.dtype is not dt or t.shape != of or t.get_device() != index or not t.is_contiguous():
            raise ValueError("%s: %s %s on the logits' device" % (name, dt, list(of)))
        return t.data_ptr()

    if tokens is None and (out.logprob is not None or out.rank is not None):
        raise ValueError("log probabilities and ranks of no tokens")
    if top and (out.top_ids is None or out.top_logprobs is None):
        raise ValueError("places for the best ids and their log probabilities")
    ptrs = (at("logprob", out.logprob, f32, rows), at("rank", out.rank, i32, rows), at("entropy", out.entropy, f32, rows), at("top_ids", out.top_ids, i32, rows, top),
            at("top_logprobs", out.top_logprobs, f32, rows, top))
    tp, hp = at("tokens", tokens, i32, rows), at("temperature", temperature, f32, rows)
    if dev.type != "cuda":
        raise ValueError("logits, tokens and results lie on a GPU, not on %s" % dev)
    with _HERE if torch.cuda.current_device() == dev.index else torch.cuda.device(dev):
        rc = L.sz_logprob_rows(TYPES[logits.dtype], logits.data_ptr(), stride, rows, vocab, tp, hp, top, *ptrs, _raw_stream(index))
    if rc:
        szlib.check(rc)
    return out
