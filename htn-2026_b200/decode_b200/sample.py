"""Drawing a token per row of logits (no counterpart in the reference, which decodes greedily)."""

from __future__ import annotations

import torch

from . import lib as L

# the current stream's handle of a device, without the Stream object that torch.cuda.current_stream() makes
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)
F32 = torch.float32
TYPES = {torch.bfloat16: L.QD_BF16, torch.float16: L.QD_FP16, torch.float32: L.QD_FP32}


def _row_values(t, dtype, shape):
    if t is None:
        return None
    assert t.dtype is dtype and t.shape == shape and t.is_cuda and t.is_contiguous()
    return t.data_ptr()


def sample(logits, u, tok, temperature=None, top_k=None, top_p=None, min_p=None, logprob=None, vocab: int | None = None,
           pdl: bool = True):
    """tok[i] = a token of row i, drawn with the uniform number u[i] in [0, 1) (qd_sample, which defines the
    order of the filters and what ties, NaN and masked logits do). logits [rows, >= vocab] BF16, FP16 or
    fp32 with unit column stride; u fp32 [rows]; tok int64 [rows]; logprob (optional) fp32 [rows].
    temperature / top_p / min_p fp32 [rows] and top_k int32 [rows] are per row; None leaves that step out.
    Graph-capturable; launches on the current torch CUDA stream."""
    shape, dtype = logits.shape, logits.dtype
    ld, step = logits.stride()
    rows, n = shape[0], shape[1] if vocab is None else vocab
    assert logits.is_cuda and dtype in TYPES and (step == 1 or shape[1] == 1) and n <= shape[1]
    one = shape[:1]
    assert u.dtype is F32 and u.shape == one and u.is_cuda and u.is_contiguous()
    assert tok.dtype is torch.int64 and tok.shape == one and tok.is_cuda and tok.is_contiguous()
    L.call("qd_sample", logits.data_ptr(), TYPES[dtype], max(ld, n) if rows <= 1 else ld, rows, n,
           _row_values(temperature, F32, one), _row_values(top_k, torch.int32, one), _row_values(top_p, F32, one),
           _row_values(min_p, F32, one), u.data_ptr(), tok.data_ptr(), _row_values(logprob, F32, one), pdl, _raw_stream(logits.get_device()))
    return tok
