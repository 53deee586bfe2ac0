"""Sampling of tokens from logits over the C ABI (gb_sample), on torch CUDA
tensors.  The uniform numbers are the caller's, so a draw can be repeated."""
from __future__ import annotations

import ctypes

from . import paged
from ._lib import SampleArgs
from .paged import _bad, _call, _dtype, _vector

_SIZE = ctypes.sizeof(SampleArgs)


def sample(logits, u, *, temperature=None, top_k=None, top_p=None, min_p=None, tokens=None, logprobs=None):
    """One token per row of logits (rows, vocab) f32, bf16 or f16 by the
    uniform numbers u (rows,) f32 in [0, 1).  temperature, top_p, min_p (rows,)
    f32 and top_k (rows,) int32 are each row's settings (None: 1, all, all,
    all); a temperature of 0 takes the largest logit, the lowest id among
    equals.  Returns (tokens (rows,) int32, logprobs (rows,) f32): each token
    and the log of its probability among those kept; -1 and -inf for a row with
    nothing above -inf."""
    lib = paged._start()
    torch = paged.torch
    shape = logits.shape
    if len(shape) != 2 or not logits.is_cuda or (shape[1] > 1 and logits.stride(1) != 1):
        _bad("logits must be a CUDA tensor (rows, vocab) with contiguous rows")
    rows, dev = shape[0], logits.device
    a = SampleArgs()
    a.u_dev = _vector("u", u, rows, dev)
    if tokens is None:
        tokens = torch.empty_like(u, dtype=torch.int32)
        a.token_dev = tokens.data_ptr()
    else:
        a.token_dev = _vector("tokens", tokens, rows, dev, torch.int32)
    if logprobs is None:
        logprobs = torch.empty_like(u)
        a.logprob_dev = logprobs.data_ptr()
    else:
        a.logprob_dev = _vector("logprobs", logprobs, rows, dev)
    if temperature is not None:
        a.temperature_dev = _vector("temperature", temperature, rows, dev)
    if top_k is not None:
        a.top_k_dev = _vector("top_k", top_k, rows, dev, torch.int32)
    if top_p is not None:
        a.top_p_dev = _vector("top_p", top_p, rows, dev)
    if min_p is not None:
        a.min_p_dev = _vector("min_p", min_p, rows, dev)
    a.struct_size = _SIZE
    a.dtype, a.rows, a.vocab = _dtype(logits.dtype), rows, shape[1]
    a.row_stride = logits.stride(0) if rows > 1 else shape[1]
    a.logits_dev = logits.data_ptr()
    _call(lib.gb_sample, dev, ctypes.byref(a))
    return tokens, logprobs
