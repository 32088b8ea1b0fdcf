"""The paged-cache operators (qd_paged_rope_append, qd_paged_attn) on the GPU against their definitions in
64 bits (tests/paged_ref.py, where the tolerances are derived), at the lengths, pages and masks where the
kernels change path: around a page, around 128 keys, around a tile of query rows, and at none at all."""

import math

import pytest
import torch

import paged_ref as R

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16, FP16 = torch.bfloat16, torch.float16


def _paged():
    from decode_b200 import paged

    return paged


def _err():
    return torch.zeros((1,), dtype=torch.int32, device=DEV)


def _attend(b, handle=None, scale=None, lse=True, err=None):
    P = _paged()
    handle = handle or P.PagedAttention(b.nq, b.nkv, b.dim, DEV, dtype=b.dtype)
    out = torch.full((b.tokens, b.nq, b.dim), 7.0, dtype=b.dtype, device=DEV)
    z = torch.full((b.tokens, b.nq), 7.0, dtype=torch.float32, device=DEV) if lse else None
    handle(b.on("q"), b.on("k_pages"), b.on("v_pages"), b.on("cu"), b.on("kv_len"), b.on("table"), out, lse=z,
           scale=scale, err=err)
    torch.cuda.synchronize()
    return out, z


def _check(b, out, lse, scale=None):
    ref, ref_lse, tol, lse_tol = R.attention(b, scale)
    n = int(b.cu[-1])
    d = (out.double().cpu() - ref).abs()[:n]
    assert bool((d <= tol[:n]).all()), (float((d - tol[:n]).max()), float(d.max()), b.spec)
    assert bool((out[n:] == 7).all()), "rows that belong to no request were written"
    if lse is not None:
        got, want = lse.double().cpu()[:n], ref_lse[:n]
        empty = want == -math.inf
        assert torch.equal(got == -math.inf, empty)
        assert bool(((got - want).abs() <= lse_tol[:n])[~empty].all()), float((got - want).abs()[~empty].max())


LENGTHS = {
    "one-key": [(1, 1)],
    "around-a-page": [(1, 15), (1, 16), (1, 17), (1, 31), (1, 33)],
    "around-128-keys": [(1, 127), (1, 128), (1, 129), (1, 255), (1, 257)],
    "empty-requests": [(0, 0), (1, 5), (0, 40), (0, 0), (1, 200), (0, 3)],
    "chunk-at-start": [(33, 33)],
    "chunk-after-cache": [(7, 140), (5, 260)],
    "chunk-over-tiles": [(131, 300), (64, 64), (65, 193)],
    "mixed": [(1, 300), (40, 41), (1, 1), (130, 130), (0, 9), (3, 511)],
    "more-tokens-than-keys": [(5, 3), (1, 0), (2, 0), (4, 4), (40, 10)],
    "long": [(1, 3001), (2, 2047)],
}


@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("lengths", list(LENGTHS))
def test_attention_at_lengths(lengths, page):
    b = R.Batch(LENGTHS[lengths], 8, 2, 128, page, seed=len(lengths) + page, device=DEV)
    err = _err()
    out, lse = _attend(b, err=err)
    _check(b, out, lse)
    assert int(err.item()) == 0


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("nq,nkv,dim,page", [(4, 4, 64, 32), (14, 2, 64, 16), (6, 2, 128, 128), (5, 1, 128, 32), (32, 8, 128, 128),
                                             (24, 1, 64, 64), (33, 1, 128, 16), (128, 1, 64, 16), (96, 2, 128, 64)])
def test_attention_head_layouts_and_types(nq, nkv, dim, page, dtype):
    spec = [(1, 130), (19, 150), (3, 3), (1, 64)]
    b = R.Batch(spec, nq, nkv, dim, page, dtype, seed=nq + dim, device=DEV)
    out, lse = _attend(b)
    _check(b, out, lse)


def test_attention_many_requests():
    g = torch.Generator().manual_seed(5)
    spec = [(int(torch.randint(0, 4, (1,), generator=g)), int(torch.randint(3, 90, (1,), generator=g))) for _ in range(333)]
    b = R.Batch(spec, 4, 1, 128, 16, seed=9, device=DEV)
    out, lse = _attend(b)
    _check(b, out, lse)


def test_attention_one_request_split_over_every_sm():
    """A long cache and few rows: each SM takes a part of the keys and the parts are joined."""
    b = R.Batch([(3, 9000)], 4, 1, 128, 64, seed=4, device=DEV)
    out, lse = _attend(b)
    _check(b, out, lse)


@pytest.mark.parametrize("spec,nq,nkv,dim,page,dtype", [
    ([(1500, 4000)], 8, 2, 128, 64, BF16), ([(1, 900), (700, 701), (300, 2000), (1, 3000)], 16, 4, 128, 16, BF16),
    ([(301, 777), (277, 512), (290, 300)], 14, 2, 64, 32, FP16), ([(2000, 2000)], 4, 4, 128, 128, BF16),
    ([(40, 3000), (30, 2500), (25, 700)], 32, 8, 128, 32, BF16), ([(9, 5000)] * 5, 8, 2, 64, 16, FP16)])
def test_attention_large(spec, nq, nkv, dim, page, dtype):
    """Units of many blocks, cut and whole, with every SM busy; several runs, since what could go wrong here
    (memory given back too early) shows only sometimes."""
    b = R.Batch(spec, nq, nkv, dim, page, dtype, seed=17, device=DEV)
    ref, ref_lse, tol, lse_tol = R.attention_on_gpu(b, DEV)
    first, err = None, _err()
    for _ in range(8):
        out, lse = _attend(b, err=err)
        assert int(err.item()) == 0
        d = (out.double() - ref).abs()
        assert bool((d <= tol).all()), (int((~(d <= tol)).sum()), float(d.max()))
        assert bool(((lse.double() - ref_lse).abs() <= lse_tol).all())
        first = out if first is None else first
        assert torch.equal(out, first)


def test_attention_padding_rows_scale_and_no_lse():
    b = R.Batch([(2, 40), (1, 17)], 8, 2, 128, 16, pad_tokens=3, seed=2, device=DEV)
    out, lse = _attend(b, scale=0.3)
    _check(b, out, lse, scale=0.3)
    out2, none = _attend(b, scale=0.3, lse=False)
    assert none is None and torch.equal(out, out2)


def test_attention_repeats_bit_for_bit_and_the_scratch_stays_ready():
    P = _paged()
    handle = P.PagedAttention(8, 2, 128, DEV)
    big = R.Batch([(1, 2900), (70, 333), (1, 5)], 8, 2, 128, 32, seed=1, device=DEV)
    small = R.Batch([(1, 50)], 8, 2, 128, 32, seed=3, device=DEV)
    first, _ = _attend(big, handle)
    for _ in range(3):
        out, lse = _attend(small, handle)
        _check(small, out, lse)
        again, _ = _attend(big, handle)
        assert torch.equal(first, again)


def test_attention_large_scores_of_one_sign():
    """Scores whose running maximum grows at every tile, and scores far below zero."""
    b = R.Batch([(4, 700), (1, 700)], 4, 1, 128, 64, seed=8, device=DEV)
    ramp = torch.linspace(0.0, 6.0, 700)[:, None, None]
    for sign, i in ((1, 0), (-1, 1)):
        b.k[i] = (b.k[i].float() * 0.1 + sign * ramp).to(BF16)
        for p in range(700):
            b.k_pages[int(b.table[i, p // 64]), :, p % 64] = b.k[i][p]
    b.q = (b.q.float().abs() * 0.5).to(BF16)
    out, lse = _attend(b)
    _check(b, out, lse)


def test_attention_strided_pools_and_rows():
    """Keys and values interleaved in one pool, and q / out as views of wider rows."""
    b = R.Batch([(1, 70), (20, 90)], 8, 2, 128, 32, seed=6, device=DEV)
    pool = torch.full((b.pages, 2, b.nkv, 32, 128), math.nan, dtype=BF16, device=DEV)
    pool[:, 0], pool[:, 1] = b.on("k_pages"), b.on("v_pages")
    wide = torch.zeros((b.tokens, 8 * 128 + 64), dtype=BF16, device=DEV)
    wide[:, :1024] = b.on("q").view(b.tokens, -1)
    out = torch.full((b.tokens, 2048), 7.0, dtype=BF16, device=DEV)
    lse = torch.full((b.tokens, 11), 7.0, device=DEV)
    table = torch.full((2, 40), -1, dtype=torch.int32, device=DEV)
    table[:, :b.table.shape[1]] = b.on("table")
    P = _paged()
    P.PagedAttention(8, 2, 128, DEV)(wide[:, :1024], pool[:, 0], pool[:, 1], b.on("cu"), b.on("kv_len"),
                                     table[:, :b.table.shape[1]], out[:, 512:1536], lse=lse[:, 1:9])
    torch.cuda.synchronize()
    _check(b, out[:, 512:1536].reshape(-1, 8, 128), lse[:, 1:9])
    assert bool((out[:, :512] == 7).all()) and bool((out[:, 1536:] == 7).all())
    assert bool((lse[:, 0] == 7).all()) and bool((lse[:, 9:] == 7).all())


def test_attention_in_a_graph_follows_the_lengths():
    """A captured call serves later steps: the lengths and the table are read on the device."""
    P = _paged()
    b = R.Batch([(1, 400), (2, 300)], 4, 1, 128, 16, seed=12, device=DEV)
    handle = P.PagedAttention(4, 1, 128, DEV)
    q, k, v, table = b.on("q"), b.on("k_pages"), b.on("v_pages"), b.on("table")
    cu, kv_len = b.on("cu"), b.on("kv_len")
    out = torch.zeros((3, 4, 128), dtype=BF16, device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        handle(q, k, v, cu, kv_len, table, out)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            handle(q, k, v, cu, kv_len, table, out)
    for lens in ([400, 300], [129, 2], [1, 255]):
        kv_len.copy_(torch.tensor(lens, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        c = R.Batch([(1, lens[0]), (2, lens[1])], 4, 1, 128, 16, seed=12)
        c.q, c.k, c.v = b.q, [x[:n] for x, n in zip(b.k, lens)], [x[:n] for x, n in zip(b.v, lens)]
        ref, _, tol, _ = R.attention(c)
        assert bool(((out.double().cpu() - ref).abs() <= tol).all()), lens


def test_attention_flags_what_it_cannot_reach():
    from decode_b200 import lib as L

    b = R.Batch([(1, 100), (1, 60)], 4, 1, 128, 32, seed=3, device=DEV)
    b.table[0, 1] = b.pages  # one past the pool
    err = _err()
    out, _ = _attend(b, err=err)
    assert int(err.item()) == 128 and "page" in L.describe_device_error(128)
    ref, _, tol, _ = R.attention(b)
    assert bool(((out.double().cpu() - ref).abs() <= tol)[1].all()), "the other request is not affected"
    b = R.Batch([(1, 64), (1, 60)], 4, 1, 128, 32, seed=3, device=DEV)
    b.table, b.kv_len = b.table[:, :2].contiguous(), torch.tensor([65, 60], dtype=torch.int32)
    err = _err()
    out, _ = _attend(b, err=err)
    assert int(err.item()) == 128
    b.spec = [(1, 64), (1, 60)]
    ref, _, tol, _ = R.attention(b)
    assert bool(((out.double().cpu() - ref).abs() <= tol).all()), "a request cut to its table row uses the row's keys"


# ------------------------------------------------------------------------------------ append
def _append(b, half, norm, err=None, tables=None, pdl=True):
    P = _paged()
    g = torch.Generator().manual_seed(77)
    top = max(kv for _, kv in b.spec) + 1
    cos, sin = P.rope_table(top, 2 * half, 5e6, "cpu") if tables is None else tables
    w = [(1 + 0.3 * torch.randn(b.dim, generator=g)).to(b.dtype) for _ in range(2)] if norm else [None, None]
    q_out = torch.full((b.tokens, b.nq, b.dim), 7.0, dtype=b.dtype, device=DEV)
    k, v = b.on("k_pages"), b.on("v_pages")
    P.rope_append(b.on("qkv"), b.on("cu"), b.on("kv_len"), b.on("table"), b.nq, b.nkv, cos.to(DEV), sin.to(DEV), q_out, k, v,
                  q_norm=w[0].to(DEV) if norm else None, k_norm=w[1].to(DEV) if norm else None, eps=1e-6, err=err, pdl=pdl)
    torch.cuda.synchronize()
    return (cos, sin, *w), q_out.cpu(), k.cpu(), v.cpu()


def _check_append(b, given, q_out, k, v):
    cos, sin, qn, kn = given
    ref_q, tol_q, keys, values = R.append(b, cos, sin, qn, kn, 1e-6)
    want_k, want_v = b.k_pages.clone(), b.v_pages.clone()
    for t in range(b.tokens):
        if t in ref_q:
            assert bool(((q_out[t].double() - ref_q[t]).abs() <= tol_q[t]).all()), t
        else:
            assert bool((q_out[t] == 7).all())
    for (i, pos), (y, tol) in keys.items():
        at = int(b.table[i, pos // b.page]), slice(None), pos % b.page
        assert bool(((k[at].double() - y).abs() <= tol).all()), (i, pos)
        assert torch.equal(v[at], values[i, pos])
        want_k[at], want_v[at] = k[at], v[at]
    same = lambda x, y: torch.equal(x.view(torch.int16), y.view(torch.int16))  # noqa: E731  (bits: the rest is NaN)
    assert same(k, want_k) and same(v, want_v), "a row that is not a new token's was written"


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("nq,nkv,dim,half,page,norm", [(32, 8, 128, 64, 64, True), (14, 2, 64, 32, 32, False), (5, 1, 128, 32, 16, True),
                                                       (3, 3, 64, 8, 128, True), (9, 3, 128, 48, 16, False)])
def test_append_head_layouts_and_types(nq, nkv, dim, half, page, norm, dtype):
    b = R.Batch([(1, 1), (0, 5), (20, 150), (1, 64), (33, 33), (1, 17)], nq, nkv, dim, page, dtype, pad_tokens=2, seed=nq, device=DEV)
    err = _err()
    _check_append(b, *_append(b, half, norm, err))
    assert int(err.item()) == 0


def test_append_many_requests():
    b = R.Batch([(i % 3, 3 + i % 50) for i in range(1100)], 4, 2, 64, 16, seed=2, device=DEV)
    _check_append(b, *_append(b, 32, True))


def test_append_strided_rows_and_pools():
    P = _paged()
    b = R.Batch([(3, 20), (2, 2)], 4, 2, 128, 16, seed=1, device=DEV)
    wide = torch.zeros((b.tokens, 8 * 128 + 128), dtype=BF16, device=DEV)
    wide[:, 64:64 + 1024] = b.on("qkv")
    pool = torch.stack((b.on("k_pages"), b.on("v_pages")), 1).contiguous()
    q = torch.full((b.tokens, 640), 7.0, dtype=BF16, device=DEV)
    cos, sin = P.rope_table(32, 128, 1e4, DEV)
    both = torch.cat((cos, sin), 1)  # one table, cos beside sin
    P.rope_append(wide[:, 64:1088], b.on("cu"), b.on("kv_len"), b.on("table"), 4, 2, both[:, :64], both[:, 64:], q[:, 128:640],
                  pool[:, 0], pool[:, 1])
    torch.cuda.synchronize()
    assert bool((q[:, :128] == 7).all())
    _check_append(b, (cos.cpu(), sin.cpu(), None, None), q[:, 128:].reshape(-1, 4, 128).cpu(), pool[:, 0].cpu(), pool[:, 1].cpu())


def test_append_flags_positions_and_pages():
    from decode_b200 import lib as L

    P = _paged()
    # position past the tables: nothing of that token is written
    b = R.Batch([(1, 9), (1, 30)], 4, 2, 128, 16, seed=1, device=DEV)
    err = _err()
    given, q, k, v = _append(b, 64, True, err, tables=P.rope_table(20, 128, 1e4, "cpu"))
    assert int(err.item()) == 16 and "position" in L.describe_device_error(16)
    assert bool((q[1] == 7).all()) and not bool((q[0] == 7).any())
    # negative positions (more new tokens than positions)
    b = R.Batch([(3, 1), (1, 4)], 4, 2, 128, 16, seed=1, device=DEV)
    err = _err()
    _, q, k, v = _append(b, 64, True, err)
    assert int(err.item()) == 16 and bool((q[:2] == 7).all()) and not bool((q[2:] == 7).any())
    # a page outside the pool, and a position past the table row: q_out alone
    for change in ("page", "row"):
        b = R.Batch([(1, 40), (1, 8)], 4, 2, 128, 16, seed=1, device=DEV)
        if change == "page":
            b.table[0, 2] = b.pages
        else:
            b.table = b.table[:, :2].contiguous()
        err = _err()
        _, q, k, v = _append(b, 64, True, err)
        assert int(err.item()) == 128 and not bool((q == 7).any())
        same = k.view(torch.int16) == b.k_pages.view(torch.int16)
        assert int((~same.all(-1)).sum()) == b.nkv, "only the other request's key rows changed"


def test_append_then_attention_on_another_stream():
    """The two calls as a model layer makes them, on a stream of their own and without host waits."""
    P = _paged()
    b = R.Batch([(1, 90), (17, 40), (1, 1)], 8, 2, 128, 16, seed=21, device=DEV)
    cos, sin = P.rope_table(128, 128, 5e6, DEV)
    handle = P.PagedAttention(8, 2, 128, DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        q = torch.empty((b.tokens, 8, 128), dtype=BF16, device=DEV)
        out = torch.empty_like(q)
        k, v, cu, kv_len, table = b.on("k_pages"), b.on("v_pages"), b.on("cu"), b.on("kv_len"), b.on("table")
        P.rope_append(b.on("qkv"), cu, kv_len, table, 8, 2, cos, sin, q, k, v)
        handle(q, k, v, cu, kv_len, table, out)
    side.synchronize()
    kc, vc = k.cpu(), v.cpu()
    b.q = q.cpu()
    for i, (_, kv) in enumerate(b.spec):
        at = [(int(b.table[i, p // 16]), p % 16) for p in range(kv)]
        b.k[i], b.v[i] = torch.stack([kc[a, :, r] for a, r in at]), torch.stack([vc[a, :, r] for a, r in at])
    ref, _, tol, _ = R.attention(b)
    assert bool(((out.double().cpu() - ref).abs() <= tol).all())


def _with_nan_key(spec, at, dim, dtype, what):
    """Requests whose key (or value) at position `at` is not a number, in one KV head."""
    b = R.Batch(spec, 8, 2, dim, 32, dtype, seed=31, device=DEV)
    for i, (_, kv) in enumerate(spec):
        if at < kv:
            (b.k if what == "key" else b.v)[i][at, 1] = math.nan
            (b.k_pages if what == "key" else b.v_pages)[int(b.table[i, at // 32]), 1, at % 32] = math.nan
    return b


@pytest.mark.parametrize("dim,dtype", [(128, BF16), (64, FP16)])
@pytest.mark.parametrize("spec", [[(1, 9000)], [(3, 9000)], [(1, 700), (4, 300), (70, 4000)], [(200, 5000), (1, 60)], [(8, 70)]])
def test_attention_shows_a_key_that_is_not_a_number(spec, dim, dtype):
    """A row that sees a NaN score is NaN, its log-sum-exp too, wherever its request is cut into pieces; the rows of
    other heads, and those that do not see the key, are as they are without it."""
    at = 50
    b = _with_nan_key(spec, at, dim, dtype, "key")
    out, lse = _attend(b)
    out, lse = out.cpu(), lse.cpu()
    clean = R.Batch(spec, 8, 2, dim, 32, dtype, seed=31)
    ref, ref_lse, tol, lse_tol = R.attention(clean)
    for i, t, pos in b.rows():
        sees = at <= pos and at < b.spec[i][1]
        for h in range(8):
            if sees and h >= 4:
                assert bool(out[t, h].isnan().all()) and bool(lse[t, h].isnan()), (i, t, h, float(lse[t, h]))
            else:
                assert bool(((out[t, h].double() - ref[t, h]).abs() <= tol[t, h]).all()), (i, t, h)
                assert float((lse[t, h].double() - ref_lse[t, h]).abs()) <= float(lse_tol[t, h])


@pytest.mark.parametrize("spec", [[(1, 9000)], [(3, 9000)], [(60, 5000)]])
def test_attention_of_queries_that_are_not_numbers(spec):
    """A NaN query: all its scores are NaN, in every piece."""
    b = R.Batch(spec, 8, 2, 128, 64, seed=5, device=DEV)
    b.q[0, 3] = math.nan
    out, lse = _attend(b)
    assert bool(out[0, 3].isnan().all()) and bool(lse[0, 3].isnan())
    other = torch.ones((b.tokens, 8), dtype=torch.bool)
    other[0, 3] = False
    ref, ref_lse, tol, lse_tol = R.attention(b)
    assert bool(((out.cpu().double() - ref).abs() <= tol)[other].all())
    assert bool(((lse.cpu().double() - ref_lse).abs() <= lse_tol)[other].all())


def test_attention_scratch_is_made_ready_again():
    """A call that ends early (a bounded wait that runs out, flagged in `err`) leaves counts in the scratch, as
    they are set here; after reset() the object answers as a new one does."""
    P = _paged()
    b = R.Batch([(1, 2900), (70, 1333), (1, 5)], 8, 2, 128, 32, seed=1, device=DEV)
    handle = P.PagedAttention(8, 2, 128, DEV)
    first, _ = _attend(b, handle)
    handle.scratch[:8 * handle.grid] = 1
    handle.reset()
    out, lse = _attend(b, handle)
    _check(b, out, lse)
    assert torch.equal(out, first)


@pytest.mark.parametrize("n", [385, 1000])
def test_attention_more_requests_than_threads(n):
    """Each thread of the start sums the work of several requests, some of them empty."""
    g = torch.Generator().manual_seed(n)
    r = lambda lo, hi: int(torch.randint(lo, hi, (1,), generator=g))  # noqa: E731
    spec = [(r(0, 3) if i % 50 else r(30, 90), r(90, 200)) for i in range(n)]
    b = R.Batch(spec, 4, 2, 64, 16, FP16, seed=n, device=DEV)
    err = _err()
    out, lse = _attend(b, err=err)
    _check(b, out, lse)
    assert int(err.item()) == 0
