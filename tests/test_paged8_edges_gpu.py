"""Calls of the 8-bit operators at the ends of what they take: more requests than their kernels have threads, none with
new tokens, pools of more bytes than 32 bits count, and a promise that the call does not keep."""

import pytest
import torch

import paged8_ref as R8
import paged_ref as R
from test_paged8_gpu import _append8, _attend8
from test_paged_gpu import _check, _err

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16, FP16 = torch.bfloat16, torch.float16
U8 = torch.uint8


def test_attention8_of_more_requests_than_threads():
    """Chunks among single tokens, before and behind the first round of both kernels' walks."""
    spec = [(20 + i % 30, 60 + i % 70) if i % 37 == 5 else (i % 3, 3 + i % 40) for i in range(1100)]
    b = R8.Batch8(spec, 4, 1, 128, 16, seed=3, device=DEV, pad_tokens=2)
    err = _err()
    out, lse = _attend8(b, err=err)
    _check(b, out, lse)
    assert int(err.item()) == 0


def test_calls_without_any_new_token():
    P = R8.Batch8([(0, 5), (0, 0), (0, 300)], 4, 2, 128, 16, seed=1, device=DEV, pad_tokens=3)
    err = _err()
    for max_new in (None, 1):
        out, lse = _attend8(P, err=err, max_new=max_new)
        assert bool((out == 7).all()) and bool((lse == 7).all())
    _, q, *pools = _append8(P, 64, True, err)
    assert bool((q == 7).all()) and int(err.item()) == 0
    for x, y in zip(pools, (P.k_pages, P.v_pages, P.k_scale, P.v_scale)):
        assert torch.equal(x.view(U8), y.view(U8))


@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_attention8_of_more_tokens_than_the_call_said(dtype):
    """The longer request's rows are left as they were and flagged; the others' are right."""
    b = R8.Batch8([(1, 1000), (20, 90), (1, 60), (4, 30), (5, 300)], 8, 2, 128, 16, dtype, seed=2, device=DEV)
    ref, ref_lse, tol, lse_tol = R.attention(b)
    for max_new in (1, 4):  # (both are few rows)
        err = _err()
        out, lse = (x.cpu() for x in _attend8(b, max_new=max_new, err=err))
        assert int(err.item()) == 16
        long = torch.zeros(b.tokens, dtype=torch.bool)
        long[1:21], long[26:] = True, True
        assert bool((out[long] == 7).all()) and bool((lse[long] == 7).all())
        assert bool(((out.double() - ref).abs() <= tol)[~long].all())
        assert bool(((lse.double() - ref_lse).abs() <= lse_tol)[~long].all())
    err = _err()
    out, lse = _attend8(b, max_new=5, err=err)  # (more than few rows: tiles too)
    _check(b, out, lse)
    assert int(err.item()) == 0


@pytest.mark.parametrize("dim,page", [(128, 64), (64, 128)])
def test_pools8_past_32_bits(dim, page):
    """Pages at the end of pools of 5 GB."""
    from decode_b200 import paged as P

    b = R8.Batch8([(1, 300), (40, 170), (2, 2)], 8, 2, dim, page, seed=8, device=DEV)
    pages = 5_000_000_000 // (2 * page * dim)
    at = pages - b.pages
    assert at * 2 * page * dim > 2 ** 32
    table = torch.where((b.table >= 0) & (b.table < b.pages), b.table + at, b.table)
    small = [getattr(b, n) for n in ("k_pages", "v_pages", "k_scale", "v_scale")]
    large = [torch.empty((pages, *s.shape[1:]), dtype=U8, device=DEV) for s in small]
    for s, x in zip(small, large):
        x[at:] = s.view(U8).to(DEV)
    pools = [x.view(s.dtype) for s, x in zip(small, large)]
    cos, sin = P.rope_table(400, dim, 5e6, DEV)
    rest = b.on("qkv"), b.on("cu"), b.on("kv_len")
    q_far, q_near = (torch.empty((b.tokens, 8, dim), dtype=BF16, device=DEV) for _ in range(2))
    near = [s.to(DEV) for s in small]
    P.rope_append8(*rest, b.on("table"), 8, 2, cos, sin, q_near, *near)
    P.rope_append8(*rest, table.to(DEV), 8, 2, cos, sin, q_far, *pools)
    assert torch.equal(q_far, q_near)
    assert all(torch.equal(x[at:], n.view(U8)) for x, n in zip(large, near))
    handle, outs = P.PagedAttention8(8, 2, dim, DEV), []
    for t, p in ((b.on("table"), near), (table.to(DEV), pools)):
        outs.append(handle(q_near, *p, *rest[1:], t, torch.empty_like(q_near)))
    torch.cuda.synchronize()
    assert torch.equal(*outs) and bool(outs[0].isfinite().all())
