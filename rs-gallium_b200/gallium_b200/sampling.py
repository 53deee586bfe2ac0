"""Sampling of tokens from logits over the C ABI (gb_sample), on torch CUDA
tensors.  The uniform numbers are the caller's, so a draw can be repeated."""
from __future__ import annotations

import ctypes

from . import _lib
from ._lib import SampleArgs, load_library
from .paged import _bad, _Call, _check, _dtype, _on


def sample(logits, u, *, temperature=None, top_k=None, top_p=None, min_p=None, tokens=None, logprobs=None):
    """One token per row of logits (rows, vocab) f32, bf16 or f16 by the
    uniform numbers u (rows,) f32 in [0, 1).  temperature, top_p, min_p (rows,)
    f32 and top_k (rows,) int32 are each row's settings (None: 1, all, all,
    all); a temperature of 0 takes the largest logit, the lowest id among
    equals.  Returns (tokens (rows,) int32, logprobs (rows,) f32): each token
    and the log of its probability among those kept; -1 and -inf for a row with
    nothing above -inf."""
    import torch

    if logits.dim() != 2 or not logits.is_cuda or (logits.shape[1] > 1 and logits.stride(1) != 1):
        _bad("logits must be a CUDA tensor (rows, vocab) with contiguous rows")
    rows, dev = logits.shape[0], logits.device
    f32, i32 = torch.float32, torch.int32
    if tokens is None:
        tokens = torch.empty(rows, dtype=i32, device=dev)
    if logprobs is None:
        logprobs = torch.empty(rows, dtype=f32, device=dev)
    a = SampleArgs()
    for name, t, want, field in (("u", u, f32, "u_dev"), ("temperature", temperature, f32, "temperature_dev"),
                                 ("top_k", top_k, i32, "top_k_dev"), ("top_p", top_p, f32, "top_p_dev"),
                                 ("min_p", min_p, f32, "min_p_dev"), ("tokens", tokens, i32, "token_dev"),
                                 ("logprobs", logprobs, f32, "logprob_dev")):
        if t is not None:
            if t.dtype != want or t.shape != (rows,) or not t.is_contiguous():
                _bad(f"{name} must be a contiguous {want} ({rows},)")
            _on(dev, name, t)
            setattr(a, field, t.data_ptr())
    a.struct_size = ctypes.sizeof(SampleArgs)
    a.dtype, a.rows, a.vocab = _dtype(logits.dtype), rows, logits.shape[1]
    a.row_stride = logits.stride(0) if rows > 1 else logits.shape[1]
    a.logits_dev = logits.data_ptr()
    with _Call(dev) as stream:
        _check(load_library().gb_sample(ctypes.byref(a), stream))
    return tokens, logprobs
