"""The paged K/V cache: appending new tokens to it and attending over it (no counterpart in the reference).

A cache of pages serves requests of any lengths side by side: a request owns the pages that its row of the
page table names, in any order, and takes another when its last one is full. Both calls take the same
ragged batch (all int32 on the device, so a captured graph follows what a later step writes into them):

  cu_tokens   [batch + 1]          request i has the token rows cu_tokens[i] .. cu_tokens[i + 1] - 1
  kv_len      [batch]              its cached positions, the new tokens' included
  page_table  [batch, max_pages]   position p is row p % page_size of page page_table[i, p // page_size]

and pools [pages, KV heads, page_size, head_dim] of BF16 or FP16 (`new_pools`). One call serves single
tokens, chunks of prompts and whole prompts together. Calls launch on the current torch CUDA stream of the
current device, on which every tensor has to be, and allocate nothing, so they are graph-capturable; device-side
faults (a page outside the pool, a position past the tables) are flagged in the optional `err` word, int32
(lib.describe_device_error).
"""

from __future__ import annotations

import ctypes
import math

import torch

from . import lib as L

# the current stream's handle of a device, without the Stream object that torch.cuda.current_stream() makes
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)
_current_device = getattr(torch._C, "_cuda_getDevice", None)
I32, F32 = torch.int32, torch.float32
TYPES = {torch.bfloat16: L.QD_BF16, torch.float16: L.QD_FP16}


def new_pools(pages: int, nkv: int, page_size: int, head_dim: int, device, dtype=torch.bfloat16):
    """Zeroed (k_pages, v_pages) of `pages` pages."""
    shape = (pages, nkv, page_size, head_dim)
    return torch.zeros(shape, dtype=dtype, device=device), torch.zeros(shape, dtype=dtype, device=device)


def rope_table(positions: int, head_dim: int, theta: float, device):
    """cos, sin [positions, head_dim / 2] fp32 of the angles p * theta^(-2r / head_dim), computed in 64 bits."""
    inv = theta ** (-torch.arange(0, head_dim, 2, dtype=torch.float64) / head_dim)
    angle = torch.arange(positions, dtype=torch.float64)[:, None] * inv[None, :]
    return angle.cos().float().to(device), angle.sin().float().to(device)


def _check_batch(dev, dtype, k_pages, v_pages, cu_tokens, kv_len, page_table, err):
    """(pool shape, pool strides, batch, table row stride, table columns), everything on the current device `dev`;
    each property is read once, since a call for a few tokens takes the GPU less time than reading it twice takes
    the host."""
    shape, strides, table = k_pages.shape, k_pages.stride(), page_table.shape
    assert dev >= 0 and dev == _current_device(), f"tensors on device {dev} (-1: the host), which is not the current one"
    assert k_pages.dtype is dtype and v_pages.dtype is dtype
    assert k_pages.get_device() == dev and v_pages.get_device() == dev
    assert v_pages.shape == shape and v_pages.stride() == strides and len(shape) == 4
    assert strides[3] == 1 and strides[2] == shape[3], "rows of a page must be contiguous"
    assert cu_tokens.dtype is I32 and kv_len.dtype is I32 and page_table.dtype is I32
    assert cu_tokens.get_device() == dev and kv_len.get_device() == dev and page_table.get_device() == dev
    if err is not None:
        assert err.dtype is I32 and err.get_device() == dev and err.numel() > 0
    ld_table, step = page_table.stride()
    assert cu_tokens.is_contiguous() and kv_len.is_contiguous() and (step == 1 or table[1] == 1)
    assert kv_len.shape == table[:1] and cu_tokens.shape == (table[0] + 1,)
    return shape, strides, table[0], max(ld_table, table[1]) if table[0] == 1 else ld_table, table[1]


def _rows(t, tokens: int, heads: int, D: int) -> int:
    """Row stride of a [tokens, heads, D] or [tokens, heads * D] tensor with contiguous rows."""
    strides = t.stride()
    if len(strides) == 3:
        assert t.shape == (tokens, heads, D) and strides[2] == 1 and (strides[1] == D or heads == 1)
    else:
        assert t.shape == (tokens, heads * D) and strides[1] == 1
    return heads * D if tokens <= 1 else strides[0]


def rope_append(qkv, cu_tokens, kv_len, page_table, nq: int, nkv: int, cos, sin, q_out, k_pages, v_pages, q_norm=None,
                k_norm=None, eps: float = 1e-6, err=None, pdl: bool = True):
    """q_out[t] = rope(norm(q)) and K = rope(norm(k)), V into the pages, for every new token t
    (qd_paged_rope_append). qkv [tokens, (nq + 2 nkv) * head_dim]; q_out [tokens, nq, head_dim] or
    [tokens, nq * head_dim]; cos / sin fp32 [positions, pairs turned] (`rope_table`)."""
    dtype = qkv.dtype
    assert dtype in TYPES, f"expected BF16 or FP16 tensors, got {dtype}"
    dev = qkv.get_device()
    pool, ps, batch, ld_table, max_pages = _check_batch(dev, dtype, k_pages, v_pages, cu_tokens, kv_len, page_table, err)
    D, tokens = pool[3], qkv.shape[0]
    assert q_out.get_device() == dev and q_out.dtype is dtype and pool[1] == nkv
    ldqkv, ldq = _rows(qkv, tokens, nq + 2 * nkv, D), _rows(q_out, tokens, nq, D)
    angles, ld = cos.shape, cos.stride()
    assert cos.dtype is F32 and sin.dtype is F32 and sin.shape == angles and sin.stride() == ld and ld[1] == 1
    assert cos.get_device() == dev and sin.get_device() == dev
    qn = kn = None
    if q_norm is not None or k_norm is not None:
        assert q_norm is not None and k_norm is not None and q_norm.shape == k_norm.shape == (D,)
        assert q_norm.dtype is dtype and q_norm.get_device() == dev and q_norm.is_contiguous()
        assert k_norm.dtype is dtype and k_norm.get_device() == dev and k_norm.is_contiguous()
        qn, kn = q_norm.data_ptr(), k_norm.data_ptr()
    L.call("qd_paged_rope_append", qkv.data_ptr(), ldqkv, TYPES[dtype], tokens, nq, nkv, D, qn, kn, eps,
           cos.data_ptr(), sin.data_ptr(), ld[0], angles[0], angles[1], cu_tokens.data_ptr(), kv_len.data_ptr(), batch,
           page_table.data_ptr(), ld_table, max_pages, q_out.data_ptr(), ldq, k_pages.data_ptr(), v_pages.data_ptr(),
           pool[0], pool[2], ps[0], ps[1], None if err is None else err.data_ptr(), pdl, _raw_stream(dev))
    return q_out


class PagedAttention:
    """Causal attention of every new token over its request's pages (qd_paged_attn), for one head layout.

    Holds the scratch, whose size depends on neither the batch nor the lengths; two calls that share an
    object must not overlap on the GPU. After a device error other than a page outside the pool (`err`),
    `reset` makes it ready again."""

    def __init__(self, nq: int, nkv: int, head_dim: int, device, dtype=torch.bfloat16, grid: int = 0):
        assert dtype in TYPES, f"expected BF16 or FP16, got {dtype}"
        self.nq, self.nkv, self.head_dim, self.dtype = nq, nkv, head_dim, dtype
        g, nbytes = ctypes.c_int(0), ctypes.c_int64(0)
        L.call("qd_paged_attn_plan", nq, nkv, head_dim, grid, ctypes.byref(g), ctypes.byref(nbytes))
        self.grid = g.value
        self.scratch = torch.zeros((nbytes.value,), dtype=torch.uint8, device=device)
        self.scratch_bytes = nbytes.value
        self.scale = 1.0 / math.sqrt(head_dim)

    def reset(self) -> None:
        """Zeroes the counts of finished pieces, which a call that ended early leaves behind: later calls would
        join pieces too early, or never."""
        self.scratch[:8 * self.grid].zero_()

    def __call__(self, q, k_pages, v_pages, cu_tokens, kv_len, page_table, out, lse=None, scale: float | None = None,
                 err=None, pdl: bool = True):
        """q, out [tokens, nq, head_dim] or [tokens, nq * head_dim]; lse (optional) fp32 [tokens, nq]."""
        nq, D, dtype, dev = self.nq, self.head_dim, self.dtype, q.get_device()
        pool, ps, batch, ld_table, max_pages = _check_batch(dev, dtype, k_pages, v_pages, cu_tokens, kv_len, page_table, err)
        tokens = q.shape[0]
        assert q.dtype is dtype and out.dtype is dtype and out.get_device() == dev and self.scratch.get_device() == dev
        assert pool[1] == self.nkv and pool[3] == D
        ldq, ldo = _rows(q, tokens, nq, D), _rows(out, tokens, nq, D)
        lse_ptr, ld_lse = None, 0
        if lse is not None:
            assert lse.dtype is F32 and lse.get_device() == dev and lse.shape == (tokens, nq)
            ld_lse, step = lse.stride()
            assert step == 1 or nq == 1
            lse_ptr, ld_lse = lse.data_ptr(), max(ld_lse, nq) if tokens <= 1 else ld_lse
        L.call("qd_paged_attn", q.data_ptr(), ldq, TYPES[dtype], tokens, nq, self.nkv, D, k_pages.data_ptr(),
               v_pages.data_ptr(), pool[0], pool[2], ps[0], ps[1], cu_tokens.data_ptr(), kv_len.data_ptr(), batch,
               page_table.data_ptr(), ld_table, max_pages, self.scale if scale is None else scale, out.data_ptr(), ldo,
               lse_ptr, ld_lse, self.grid, self.scratch.data_ptr(), self.scratch_bytes,
               None if err is None else err.data_ptr(), pdl, _raw_stream(dev))
        return out
