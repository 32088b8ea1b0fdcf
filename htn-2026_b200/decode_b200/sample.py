"""Drawing a token per row of logits (no counterpart in the reference, which decodes greedily)."""

from __future__ import annotations

import torch

from . import lib as L
from .paged import _current_device, _raw_stream

F32 = torch.float32
TYPES = {torch.bfloat16: L.QD_BF16, torch.float16: L.QD_FP16, torch.float32: L.QD_FP32}


def _row_values(t, dtype, shape, dev):
    if t is None:
        return None
    assert t.dtype is dtype and t.shape == shape and t.get_device() == dev and t.is_contiguous()
    return t.data_ptr()


def sample(logits, u, tok, temperature=None, top_k=None, top_p=None, min_p=None, logprob=None, vocab: int | None = None,
           pdl: bool = True):
    """tok[i] = a token of row i, drawn with the uniform number u[i] in [0, 1) (qd_sample, which defines the
    order of the filters and what ties, NaN and masked logits do). logits [rows, >= vocab] BF16, FP16 or
    fp32 with unit column stride; u fp32 [rows]; tok int64 [rows]; logprob (optional) fp32 [rows].
    temperature / top_p / min_p fp32 [rows] and top_k int32 [rows] are per row; None leaves that step out.
    Graph-capturable; launches on the current torch CUDA stream of the current device, on which every tensor
    has to be."""
    shape, dtype = logits.shape, logits.dtype
    ld, step = logits.stride()
    rows, n = shape[0], shape[1] if vocab is None else vocab
    dev = logits.get_device()
    assert dev >= 0 and dev == _current_device(), f"logits on device {dev} (-1: the host), which is not the current one"
    assert dtype in TYPES and (step == 1 or shape[1] == 1) and n <= shape[1]
    one = shape[:1]
    assert u is not None and tok is not None
    L.call("qd_sample", logits.data_ptr(), TYPES[dtype], max(ld, n) if rows <= 1 else ld, rows, n,
           _row_values(temperature, F32, one, dev), _row_values(top_k, torch.int32, one, dev),
           _row_values(top_p, F32, one, dev), _row_values(min_p, F32, one, dev), _row_values(u, F32, one, dev),
           _row_values(tok, torch.int64, one, dev), _row_values(logprob, F32, one, dev), pdl, _raw_stream(dev))
    return tok
