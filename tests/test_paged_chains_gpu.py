"""The paged operators' calls one after the other with nothing between them, as the layers and steps of a model make
them: the same buffers again and again, each call reading what the one before wrote, whatever starts early."""

import pytest
import torch

import paged8_ref as R8
from test_paged_gpu import _err

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16, FP16 = torch.bfloat16, torch.float16
PASSES = 6


def _paged():
    from decode_b200 import paged

    return paged


def _passes(b, step):
    """(out, lse) of every pass: step(pass, qkv, q, out, lse, pdl) over one q buffer, once with a wait for the GPU after each
    call's launches and no early start, then all in a row, then from a graph."""
    g = torch.Generator().manual_seed(5)
    qkv = [(torch.randn(b.qkv.shape, generator=g) * (1 + i)).to(b.dtype).to(DEV) for i in range(PASSES)]
    q = torch.zeros((b.tokens, b.nq, b.dim), dtype=b.dtype, device=DEV)
    out = torch.zeros((PASSES, b.tokens, b.nq, b.dim), dtype=b.dtype, device=DEV)
    lse = torch.zeros((PASSES, b.tokens, b.nq), device=DEV)
    got = []
    for i in range(PASSES):
        step(qkv[i], q, out[i], lse[i], False)
        torch.cuda.synchronize()
    got.append((out.clone(), lse.clone()))
    for _ in range(3):
        out.fill_(7), lse.fill_(7)
        torch.cuda.synchronize()
        for i in range(PASSES):
            step(qkv[i], q, out[i], lse[i], True)
        torch.cuda.synchronize()
        got.append((out.clone(), lse.clone()))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
        for i in range(PASSES):
            step(qkv[i], q, out[i], lse[i], True)
    for _ in range(3):
        out.fill_(7), lse.fill_(7)
        graph.replay()
        torch.cuda.synchronize()
        got.append((out.clone(), lse.clone()))
    return got


def _all_alike(got):
    (want, want_lse), *rest = got
    assert bool(want.isfinite().all()) and not torch.equal(want[0], want[1]), "passes that differ"
    for k, (out, lse) in enumerate(rest):
        for i in range(PASSES):
            assert torch.equal(out[i], want[i]) and torch.equal(lse[i], want_lse[i]), (k, i)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("spec", [[(1, 3000), (60, 900), (1, 700), (2, 90), (1, 1)], [(1, 1500 - 17 * i) for i in range(40)] + [(33, 70)]])
def test_append8_and_attention8_over_one_query_buffer(spec, dtype):
    """Single tokens beside chunks: the kernel for few rows starts while the tiles' is at work."""
    P = _paged()
    b = R8.Batch8(spec, 8, 2, 128, 32, dtype, seed=7, device=DEV)
    cos, sin = P.rope_table(3001, 128, 5e6, DEV)
    handle, err = P.PagedAttention8(8, 2, 128, DEV, dtype=dtype), _err()
    pools = [b.on(n) for n in ("k_pages", "v_pages", "k_scale", "v_scale")]
    cu, kv_len, table = b.on("cu"), b.on("kv_len"), b.on("table")

    def step(qkv, q, out, lse, pdl):
        P.rope_append8(qkv, cu, kv_len, table, 8, 2, cos, sin, q, *pools, err=err, pdl=pdl)
        handle(q, *pools, cu, kv_len, table, out, lse=lse, err=err, pdl=pdl)

    _all_alike(_passes(b, step))
    assert int(err.item()) == 0
