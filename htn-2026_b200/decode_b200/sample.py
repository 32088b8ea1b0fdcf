"""Drawing a token per row of logits (no counterpart in the reference, which decodes greedily)."""

from __future__ import annotations

import torch

from . import lib as L
from .ops import _ptr, _stream

TYPES = {torch.bfloat16: L.QD_BF16, torch.float16: L.QD_FP16, torch.float32: L.QD_FP32}


def sample(logits, u, tok, temperature=None, top_k=None, top_p=None, min_p=None, logprob=None, vocab: int | None = None,
           pdl: bool = True):
    """tok[i] = a token of row i, drawn with the uniform number u[i] in [0, 1) (qd_sample, which defines the
    order of the filters and what ties, NaN and masked logits do). logits [rows, >= vocab] BF16, FP16 or
    fp32 with unit column stride; u fp32 [rows]; tok int64 [rows]; logprob (optional) fp32 [rows].
    temperature / top_p / min_p fp32 [rows] and top_k int32 [rows] are per row; None leaves that step out.
    Graph-capturable; launches on the current torch CUDA stream."""
    rows = logits.shape[0]
    assert logits.is_cuda and logits.dtype in TYPES and logits.dim() == 2 and logits.stride(1) == 1
    n = logits.shape[1] if vocab is None else vocab
    assert n <= logits.shape[1]
    assert u.dtype == torch.float32 and u.numel() == rows and u.is_contiguous() and u.is_cuda
    assert tok.dtype == torch.int64 and tok.numel() == rows and tok.is_contiguous() and tok.is_cuda
    for x, t in ((temperature, torch.float32), (top_k, torch.int32), (top_p, torch.float32), (min_p, torch.float32),
                 (logprob, torch.float32)):
        assert x is None or (x.dtype == t and x.numel() == rows and x.is_contiguous() and x.is_cuda)
    L.call("qd_sample", logits.data_ptr(), TYPES[logits.dtype], logits.stride(0), rows, n, _ptr(temperature),
           _ptr(top_k), _ptr(top_p), _ptr(min_p), u.data_ptr(), tok.data_ptr(), _ptr(logprob), int(pdl), _stream())
    return tok
