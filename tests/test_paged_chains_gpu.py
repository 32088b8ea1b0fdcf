"""The paged operators' calls one after the other with nothing between them, as the layers and steps of a model make
them: the same buffers again and again, each call reading what the one before wrote, whatever starts early."""

import pytest
import torch

import paged8_ref as R8
from test_paged_gpu import _err
from test_prefix_gpu import Groups

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


@pytest.mark.parametrize("groups", [[(512, [(1, 90), (17, 40), (1, 1), (1, 7), (1, 300)]), (1024, [(1, 30)] * 9)],
                                    [(2048, [(1, 5 + i) for i in range(40)]), (0, [(60, 600), (1, 900)])]])
def test_append_and_attention_over_shared_beginnings_in_a_row(groups):
    """Three launches a call over one scratch, which the call before may still be reading."""
    P = _paged()
    b = Groups(groups, 8, 2, 128, 16, seed=3, device=DEV)
    cos, sin = P.rope_table(4096, 128, 5e6, DEV)
    handle, err = P.PrefixAttention(8, 2, 128, DEV, b.tokens, len(b.spec)), _err()
    k, v, cu, kv_len, table = b.on("k_pages"), b.on("v_pages"), b.on("cu"), b.on("kv_len"), b.on("table")
    cu_groups, prefix_len = b.on("cu_groups"), b.on("prefix_len")

    def step(qkv, q, out, lse, pdl):
        P.rope_append(qkv, cu, kv_len, table, 8, 2, cos, sin, q, k, v, err=err, pdl=pdl)
        handle(q, k, v, cu, kv_len, table, cu_groups, prefix_len, out, lse=lse, err=err, pdl=pdl)

    _all_alike(_passes(b, step))
    assert int(err.item()) == 0


def test_two_objects_on_two_streams_at_once():
    """Each with a scratch of its own, over the same pools."""
    P = _paged()
    b = R8.Batch8([(1, 3000), (60, 900), (1, 700), (2, 90)], 8, 2, 128, 32, seed=7, device=DEV)
    pools = [b.on(n) for n in ("k_pages", "v_pages", "k_scale", "v_scale")]
    cu, kv_len, table, q = b.on("cu"), b.on("kv_len"), b.on("table"), b.on("q")
    g = Groups([(1024, [(1, 90), (17, 40), (1, 300)] * 3)], 8, 2, 128, 32, seed=4, device=DEV)
    given = [g.on(n) for n in ("q", "k_pages", "v_pages", "cu", "kv_len", "table", "cu_groups", "prefix_len")]
    calls = []
    for _ in range(2):
        h8, hp = P.PagedAttention8(8, 2, 128, DEV), P.PrefixAttention(8, 2, 128, DEV, g.tokens, len(g.spec))
        calls.append((lambda out, h8=h8: h8(q, *pools, cu, kv_len, table, out), torch.empty_like(q)))
        calls.append((lambda out, hp=hp: hp(*given, out), torch.empty_like(given[0])))
    want = []
    for call, out in calls:
        call(out)
        torch.cuda.synchronize()
        want.append(out.clone())
        out.fill_(7)
    streams = [torch.cuda.Stream() for _ in calls]
    torch.cuda.synchronize()
    for _ in range(5):
        for (call, out), s in zip(calls, streams):
            with torch.cuda.stream(s):
                call(out)
    torch.cuda.synchronize()
    assert all(torch.equal(out, w) for (_, out), w in zip(calls, want))
