"""Infinities and NaN in the 8-bit append (qd_paged_rope_append8): queries come out as the 16-bit append's, bit for bit,
whatever heads share a warp; held rows have NaN where they were not finite."""

import math

import pytest
import torch

import paged8_ref as R8

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16, FP16 = torch.bfloat16, torch.float16
U8 = torch.uint8


@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("nq,nkv,dim,half", [(14, 2, 64, 32), (5, 1, 128, 32), (6, 2, 128, 64), (32, 8, 128, 64), (3, 3, 64, 8)])
def test_append8_queries_with_infinities(nq, nkv, dim, half, dtype, norm):
    from decode_b200 import paged as P

    # (more tokens: two groups of heads a warp)
    for tokens in (12, 700):
        b = R8.Batch8([(tokens, tokens)], nq, nkv, dim, 16, dtype, seed=nq, device=DEV)
        x = b.qkv.view(tokens, nq + 2 * nkv, dim)
        for t in range(12):  # one element of a head, the last query heads and the K heads beside them among them
            x[t, (nq - 1 - t) % (nq + nkv), t * 5 % dim] = (math.inf, -math.inf, math.nan)[t % 3]
        x[7, nq:, 3] = math.inf
        x[8, nq + nkv:, 4] = -math.inf
        cos, sin = P.rope_table(tokens + 1, 2 * half, 5e6, DEV)
        w = torch.linspace(0.5, 1.5, dim).to(dtype).to(DEV) if norm else None
        call = dict(cos=cos, sin=sin, q_norm=w, k_norm=w)
        qkv, cu, kv_len, table = b.on("qkv"), b.on("cu"), b.on("kv_len"), b.on("table")
        q16, q8 = (torch.full((tokens, nq, dim), 7.0, dtype=dtype, device=DEV) for _ in range(2))
        k16, v16 = P.new_pools(b.pages, nkv, 16, dim, DEV, dtype)
        P.rope_append(qkv, cu, kv_len, table, nq, nkv, q_out=q16, k_pages=k16, v_pages=v16, **call)
        k8, v8, ks, vs = P.new_pools8(b.pages, nkv, 16, dim, DEV)
        P.rope_append8(qkv, cu, kv_len, table, nq, nkv, q_out=q8, k_pages=k8, v_pages=v8, k_scale=ks, v_scale=vs, **call)
        torch.cuda.synchronize()
        assert bool(q16.isinf().any()) or norm, "a case with infinities"
        assert torch.equal(q8.view(torch.int16), q16.view(torch.int16)), tokens
        for p16, p8, scale in ((k16, k8, ks), (v16, v8, vs)):
            held = P.held_values(p8, scale)
            assert torch.equal(held.isnan(), ~p16.float().isfinite())
