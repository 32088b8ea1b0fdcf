"""The paged K/V cache: appending new tokens to it and attending over it (no counterpart in the reference).

A cache of pages serves requests of any lengths side by side: a request owns the pages that its row of the
page table names, in any order, and takes another when its last one is full. Both calls take the same
ragged batch (all int32 on the device, so a captured graph follows what a later step writes into them):

  cu_tokens   [batch + 1]          request i has the token rows cu_tokens[i] .. cu_tokens[i + 1] - 1
  kv_len      [batch]              its cached positions, the new tokens' included
  page_table  [batch, max_pages]   position p is row p % page_size of page page_table[i, p // page_size]

and pools [pages, KV heads, page_size, head_dim] of BF16 or FP16 (`new_pools`). One call serves single
tokens, chunks of prompts and whole prompts together. Calls launch on the current torch CUDA stream and
allocate nothing, so they are graph-capturable; device-side faults (a page outside the pool, a position
past the tables) are flagged in the optional `err` word (lib.describe_device_error).
"""

from __future__ import annotations

import ctypes
import math

import torch

from . import lib as L
from .ops import _ptr, _stream

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


def _check_batch(dtype, k_pages, v_pages, cu_tokens, kv_len, page_table):
    assert dtype in TYPES, f"expected BF16 or FP16 tensors, got {dtype}"
    assert k_pages.dtype == dtype and v_pages.dtype == dtype and k_pages.is_cuda and v_pages.is_cuda
    assert k_pages.dim() == 4 and k_pages.shape == v_pages.shape and k_pages.stride() == v_pages.stride()
    assert k_pages.stride(3) == 1 and k_pages.stride(2) == k_pages.shape[3], "rows of a page must be contiguous"
    assert cu_tokens.dtype == kv_len.dtype == page_table.dtype == torch.int32
    assert cu_tokens.is_cuda and kv_len.is_cuda and page_table.is_cuda
    assert cu_tokens.is_contiguous() and kv_len.is_contiguous() and page_table.stride(-1) == 1
    assert kv_len.numel() == page_table.shape[0] and cu_tokens.numel() == kv_len.numel() + 1


def rope_append(qkv, cu_tokens, kv_len, page_table, nq: int, nkv: int, cos, sin, q_out, k_pages, v_pages, q_norm=None,
                k_norm=None, eps: float = 1e-6, err=None, pdl: bool = True):
    """q_out[t] = rope(norm(q)) and K = rope(norm(k)), V into the pages, for every new token t
    (qd_paged_rope_append). qkv [tokens, (nq + 2 nkv) * head_dim]; q_out [tokens, nq, head_dim] or
    [tokens, nq * head_dim]; cos / sin fp32 [positions, pairs turned] (`rope_table`)."""
    D = k_pages.shape[3]
    _check_batch(qkv.dtype, k_pages, v_pages, cu_tokens, kv_len, page_table)
    assert qkv.is_cuda and qkv.dim() == 2 and qkv.shape[1] == (nq + 2 * nkv) * D and qkv.stride(1) == 1
    assert q_out.dtype == qkv.dtype and q_out.shape[0] == qkv.shape[0] and q_out.numel() == qkv.shape[0] * nq * D
    assert q_out.stride(-1) == 1 and (q_out.dim() == 2 or q_out.stride(1) == D)
    assert k_pages.shape[1] == nkv
    assert cos.dtype == sin.dtype == torch.float32 and cos.shape == sin.shape and cos.stride() == sin.stride()
    assert cos.stride(1) == 1
    for w in (q_norm, k_norm):
        assert w is None or (w.dtype == qkv.dtype and w.numel() == D and w.is_contiguous())
    L.call("qd_paged_rope_append", qkv.data_ptr(), qkv.stride(0), TYPES[qkv.dtype], qkv.shape[0], nq, nkv, D,
           _ptr(q_norm), _ptr(k_norm), eps, cos.data_ptr(), sin.data_ptr(), cos.stride(0), cos.shape[0], cos.shape[1],
           cu_tokens.data_ptr(), kv_len.data_ptr(), kv_len.numel(), page_table.data_ptr(), page_table.stride(0),
           page_table.shape[1], q_out.data_ptr(), q_out.stride(0), k_pages.data_ptr(), v_pages.data_ptr(),
           k_pages.shape[0], k_pages.shape[2], k_pages.stride(0), k_pages.stride(1), _ptr(err), int(pdl), _stream())
    return q_out


class PagedAttention:
    """Causal attention of every new token over its request's pages (qd_paged_attn), for one head layout.

    Holds the scratch, whose size depends on neither the batch nor the lengths; two calls that share an
    object must not overlap on the GPU."""

    def __init__(self, nq: int, nkv: int, head_dim: int, device, dtype=torch.bfloat16, grid: int = 0):
        assert dtype in TYPES, f"expected BF16 or FP16, got {dtype}"
        self.nq, self.nkv, self.head_dim, self.dtype = nq, nkv, head_dim, dtype
        g, nbytes = ctypes.c_int(0), ctypes.c_int64(0)
        L.call("qd_paged_attn_plan", nq, nkv, head_dim, grid, ctypes.byref(g), ctypes.byref(nbytes))
        self.grid = g.value
        self.scratch = torch.zeros((max(1, nbytes.value),), dtype=torch.uint8, device=device)
        self.scale = 1.0 / math.sqrt(head_dim)

    def __call__(self, q, k_pages, v_pages, cu_tokens, kv_len, page_table, out, lse=None, scale: float | None = None,
                 err=None, pdl: bool = True):
        """q, out [tokens, nq, head_dim] or [tokens, nq * head_dim]; lse (optional) fp32 [tokens, nq]."""
        nq, D = self.nq, self.head_dim
        _check_batch(q.dtype, k_pages, v_pages, cu_tokens, kv_len, page_table)
        assert q.dtype == out.dtype == self.dtype and q.is_cuda and out.is_cuda
        assert q.numel() == out.numel() == q.shape[0] * nq * D and out.shape[0] == q.shape[0]
        assert q.stride(-1) == 1 and out.stride(-1) == 1
        assert (q.dim() == 2 or q.stride(1) == D) and (out.dim() == 2 or out.stride(1) == D)
        assert k_pages.shape[1] == self.nkv and k_pages.shape[3] == D
        if lse is not None:
            assert lse.dtype == torch.float32 and lse.shape == (q.shape[0], nq) and lse.stride(1) == 1
        L.call("qd_paged_attn", q.data_ptr(), q.stride(0), TYPES[self.dtype], q.shape[0], nq, self.nkv, D,
               k_pages.data_ptr(), v_pages.data_ptr(), k_pages.shape[0], k_pages.shape[2], k_pages.stride(0),
               k_pages.stride(1), cu_tokens.data_ptr(), kv_len.data_ptr(), kv_len.numel(), page_table.data_ptr(),
               page_table.stride(0), page_table.shape[1], self.scale if scale is None else scale, out.data_ptr(),
               out.stride(0), _ptr(lse), lse.stride(0) if lse is not None else 0, self.grid, self.scratch.data_ptr(),
               self.scratch.numel(), _ptr(err), int(pdl), _stream())
        return out
