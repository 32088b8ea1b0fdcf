"""Pages of 8 bits (qd_paged_rope_append8, qd_paged_attn8) on the GPU against their definitions in 64 bits
(tests/paged8_ref.py, tests/paged_ref.py), at the lengths, pages and masks where the kernels change path.

The attention's tolerances are the 16-bit one's: what a row holds is exact, its scores are sums in fp32, and the
probabilities are off by no more than one rounding to the element type."""

import math

import pytest
import torch

import paged8_ref as R8
import paged_ref as R
from test_paged_gpu import LENGTHS, _check, _err

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16, FP16 = torch.bfloat16, torch.float16
U8 = torch.uint8


def _paged():
    from decode_b200 import paged

    return paged


# ------------------------------------------------------------------------------------ append
def _append8(b, half, norm, err=None, tables=None, pools=None):
    P = _paged()
    g = torch.Generator().manual_seed(77)
    top = max(kv for _, kv in b.spec) + 1
    cos, sin = P.rope_table(top, 2 * half, 5e6, "cpu") if tables is None else tables
    w = [(1 + 0.3 * torch.randn(b.dim, generator=g)).to(b.dtype) for _ in range(2)] if norm else [None, None]
    q_out = torch.full((b.tokens, b.nq, b.dim), 7.0, dtype=b.dtype, device=DEV)
    pools = [b.on(n) for n in ("k_pages", "v_pages", "k_scale", "v_scale")] if pools is None else pools
    P.rope_append8(b.on("qkv"), b.on("cu"), b.on("kv_len"), b.on("table"), b.nq, b.nkv, cos.to(DEV), sin.to(DEV), q_out, *pools,
                   q_norm=w[0].to(DEV) if norm else None, k_norm=w[1].to(DEV) if norm else None, eps=1e-6, err=err)
    torch.cuda.synchronize()
    return (cos, sin, *w), q_out.cpu(), *(p.cpu() for p in pools)


def _check_append8(b, given, q_out, k, v, ks, vs):
    cos, sin, qn, kn = given
    ref_q, tol_q, keys, values = R.append(b, cos, sin, qn, kn, 1e-6)
    want = [x.view(U8).clone() for x in (b.k_pages, b.v_pages, b.k_scale, b.v_scale)]
    got = [x.view(U8) for x in (k, v, ks, vs)]
    for t in range(b.tokens):
        if t in ref_q:
            assert bool(((q_out[t].double() - ref_q[t]).abs() <= tol_q[t]).all()), t
        else:
            assert bool((q_out[t] == 7).all())
    u = R.UNIT[b.dtype]
    for (i, pos), (y, tol16) in keys.items():
        at = int(b.table[i, pos // b.page]), slice(None), pos % b.page
        # what the fp32 arithmetic may be off by: the bound of the 16-bit append without its rounding
        off = tol16 - u * y.abs() - R.TINY[b.dtype]
        most, room = y.abs().amax(-1), off.amax(-1)
        e = got[2][at].long() - 127
        assert bool((R8.exponent((most - room).clamp(min=0)[:, None]) <= e).all())
        assert bool((e <= R8.exponent((most + room)[:, None])).all())
        held = k[at].double() * torch.exp2(e.double())[:, None]
        # one rounding to E4M3: half a step of 2^-3 of the value, or half the least step, 2^-9, of the row's power
        tol = torch.maximum(2.0 ** -4 * y.abs(), 2.0 ** -10 * torch.exp2(e.double())[:, None]) + 1.1 * off
        assert bool(((held - y).abs() <= tol).all()), (i, pos)
        codes, exps, _ = R8.hold(values[i, pos])
        assert torch.equal(got[1][at], codes.view(U8)) and torch.equal(got[3][at], exps), "V goes in as it was"
        for x, y2 in zip(want, got):
            x[at] = y2[at]
    assert all(torch.equal(x, y) for x, y in zip(want, got)), "a row that is not a new token's was written"


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("nq,nkv,dim,half,page,norm", [(32, 8, 128, 64, 64, True), (14, 2, 64, 32, 32, False), (5, 1, 128, 32, 16, True),
                                                       (3, 3, 64, 8, 128, True), (9, 3, 128, 48, 16, False)])
def test_append8_head_layouts_and_types(nq, nkv, dim, half, page, norm, dtype):
    b = R8.Batch8([(1, 1), (0, 5), (20, 150), (1, 64), (33, 33), (1, 17)], nq, nkv, dim, page, dtype, pad_tokens=2, seed=nq, device=DEV)
    err = _err()
    _check_append8(b, *_append8(b, half, norm, err))
    assert int(err.item()) == 0


def test_append8_many_requests_and_tokens():
    """More warps than take one group of heads each; more requests than one round of the search."""
    b = R8.Batch8([(i % 3, 3 + i % 50) for i in range(1100)], 4, 2, 64, 16, seed=2, device=DEV)
    _check_append8(b, *_append8(b, 32, True))
    b = R8.Batch8([(700, 700), (1, 3)], 8, 2, 128, 64, seed=3, device=DEV)
    _check_append8(b, *_append8(b, 64, False))


def test_append8_of_sizes_at_the_ends():
    """Rows of zeros, of a single value, at the border of a power, far below and above what the exponents reach, and with
    infinities and NaN: V goes in as it was, so every code is known."""
    b = R8.Batch8([(12, 12)], 4, 2, 128, 16, BF16, seed=1, device=DEV)
    v = b.qkv.view(12, 8, 128)[:, 6:]
    v[0] = 0
    v[1] = torch.where(torch.arange(128) == 5, 448.0, 0.0)
    v[2] = torch.where(torch.arange(128) == 5, 450.0, 1.0)  # the next BF16 above 448
    v[3] = v[3] * 2.0 ** -30
    v[4] = v[4] * 2.0 ** 14
    v[5, :, 3] = math.inf
    v[6, :, 4] = -math.inf
    v[7, :, 9] = math.nan
    v[8] = math.nan
    v[9] = 57344.0
    v[10] = 57600.0
    v[11] = -3.0e38
    given, q_out, k, vp, ks, vs = _append8(b, 64, False)
    _check_append8(b, given, q_out, k, vp, ks, vs)
    page = int(b.table[0, 0])
    assert vs.view(U8)[page, 0, :12].tolist()[:3] == [112, 127, 128] and vs.view(U8)[page, 0, 11] == 134
    held = vp[page, 0, :12].float() * vs[page, 0, :12].float()[:, None]
    assert bool(held[5, 3].isnan()) and int(held[5].isnan().sum()) == 1 and bool((held[11] == -57344).all())


def test_append8_strided_pools():
    """K and V (and their scales) side by side in one buffer."""
    b = R8.Batch8([(3, 20), (2, 2)], 4, 2, 128, 16, seed=1, device=DEV)
    pool = torch.stack((b.k_pages.view(U8), b.v_pages.view(U8)), 1).contiguous().to(DEV)
    scale = torch.stack((b.k_scale.view(U8), b.v_scale.view(U8)), 1).contiguous().to(DEV)
    views = [pool[:, 0].view(R8.E4M3), pool[:, 1].view(R8.E4M3), scale[:, 0].view(R8.E8M0), scale[:, 1].view(R8.E8M0)]
    _check_append8(b, *_append8(b, 64, True, pools=views))


def test_append8_flags_positions_and_pages():
    P = _paged()
    b = R8.Batch8([(1, 9), (1, 30)], 4, 2, 128, 16, seed=1, device=DEV)
    err = _err()
    _, q, *_ = _append8(b, 64, True, err, tables=P.rope_table(20, 128, 1e4, "cpu"))
    assert int(err.item()) == 16 and bool((q[1] == 7).all()) and not bool((q[0] == 7).any())
    b = R8.Batch8([(1, 40), (1, 8)], 4, 2, 128, 16, seed=1, device=DEV)
    b.table[0, 2] = b.pages
    err = _err()
    _, q, k, _, ks, _ = _append8(b, 64, True, err)
    assert int(err.item()) == 128 and not bool((q == 7).any())
    assert int((k.view(U8) != b.k_pages.view(U8)).any(-1).sum()) == b.nkv, "only the other request's key rows changed"
    assert int((ks.view(U8) != b.k_scale.view(U8)).sum()) <= b.nkv


# ------------------------------------------------------------------------------------ attention
def _attend8(b, handle=None, scale=None, lse=True, err=None, max_new=None):
    P = _paged()
    handle = handle or P.PagedAttention8(b.nq, b.nkv, b.dim, DEV, dtype=b.dtype)
    out = torch.full((b.tokens, b.nq, b.dim), 7.0, dtype=b.dtype, device=DEV)
    z = torch.full((b.tokens, b.nq), 7.0, dtype=torch.float32, device=DEV) if lse else None
    handle(b.on("q"), b.on("k_pages"), b.on("v_pages"), b.on("k_scale"), b.on("v_scale"), b.on("cu"), b.on("kv_len"), b.on("table"),
           out, lse=z, scale=scale, err=err, max_new=max_new)
    torch.cuda.synchronize()
    return out, z


@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("lengths", list(LENGTHS))
def test_attention8_at_lengths(lengths, page):
    b = R8.Batch8(LENGTHS[lengths], 8, 2, 128, page, seed=len(lengths) + page, device=DEV)
    err = _err()
    out, lse = _attend8(b, err=err)
    _check(b, out, lse)
    assert int(err.item()) == 0


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("nq,nkv,dim,page", [(4, 4, 64, 32), (14, 2, 64, 16), (6, 2, 128, 128), (5, 1, 128, 32), (32, 8, 128, 128),
                                             (24, 1, 64, 64), (33, 1, 128, 16), (128, 1, 64, 16), (96, 2, 128, 64)])
def test_attention8_head_layouts_and_types(nq, nkv, dim, page, dtype):
    spec = [(1, 130), (19, 150), (3, 3), (1, 64)]
    b = R8.Batch8(spec, nq, nkv, dim, page, dtype, seed=nq + dim, device=DEV)
    out, lse = _attend8(b)
    _check(b, out, lse)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("new", [1, 2, 4])
def test_attention8_few_rows(new, dim, dtype):
    """Single tokens and a few of them, short caches and ones that are cut between all SMs, with max_new given."""
    spec = [(1, kv) for kv in (1, 2, 127, 128, 129, 300, 1000)] + [(0, 77), (new, 2500), (new, new)]
    b = R8.Batch8(spec, 8, 2, dim, 32, dtype, seed=new, device=DEV)
    err = _err()
    out, lse = _attend8(b, max_new=new, err=err)
    _check(b, out, lse)
    again, _ = _attend8(b)
    assert torch.equal(out, again) and int(err.item()) == 0


def test_attention8_many_requests():
    g = torch.Generator().manual_seed(5)
    spec = [(int(torch.randint(0, 4, (1,), generator=g)), int(torch.randint(3, 90, (1,), generator=g))) for _ in range(433)]
    b = R8.Batch8(spec, 4, 1, 128, 16, seed=9, device=DEV)
    out, lse = _attend8(b)
    _check(b, out, lse)


def test_attention8_one_request_split_over_every_sm():
    b = R8.Batch8([(3, 9000)], 4, 1, 128, 64, seed=4, device=DEV)
    out, lse = _attend8(b)
    _check(b, out, lse)


@pytest.mark.parametrize("spec,nq,nkv,dim,page,dtype", [
    ([(1500, 4000)], 8, 2, 128, 64, BF16), ([(1, 900), (700, 701), (300, 2000), (1, 3000)], 16, 4, 128, 16, BF16),
    ([(301, 777), (277, 512), (290, 300)], 14, 2, 64, 32, FP16), ([(2000, 2000)], 4, 4, 128, 128, BF16),
    ([(40, 3000), (30, 2500), (25, 700)], 32, 8, 128, 32, FP16), ([(9, 5000)] * 5, 8, 2, 64, 16, BF16),
    ([(1, 1500 - 17 * i) for i in range(40)], 32, 8, 128, 16, BF16)])
def test_attention8_large(spec, nq, nkv, dim, page, dtype):
    """Units of many blocks, cut and whole, with every SM busy, several times with the same bits."""
    b = R8.Batch8(spec, nq, nkv, dim, page, dtype, seed=17, device=DEV)
    ref, ref_lse, tol, lse_tol = R.attention_on_gpu(b, DEV)
    handle, first, err = _paged().PagedAttention8(nq, nkv, dim, DEV, dtype=dtype), None, _err()
    for _ in range(8):
        out, lse = _attend8(b, handle, err=err)
        assert int(err.item()) == 0
        d = (out.double() - ref).abs()
        assert bool((d <= tol).all()), (int((~(d <= tol)).sum()), float(d.max()))
        assert bool(((lse.double() - ref_lse).abs() <= lse_tol).all())
        first = out if first is None else first
        assert torch.equal(out, first)


def test_attention8_padding_rows_scale_and_no_lse():
    b = R8.Batch8([(2, 40), (1, 17), (30, 50)], 8, 2, 128, 16, pad_tokens=3, seed=2, device=DEV)
    out, lse = _attend8(b, scale=0.3)
    _check(b, out, lse, scale=0.3)
    out2, none = _attend8(b, scale=0.3, lse=False)
    assert none is None and torch.equal(out, out2)


@pytest.mark.parametrize("new", [1, 40])
def test_attention8_of_sizes_far_apart(new):
    """Keys, values and queries whose rows differ by many powers of two, the least and the largest that a row can hold."""
    b = R8.Batch8([(new, 700)], 4, 1, 128, 32, seed=3, device=DEV, sizes=False)
    g = torch.Generator().manual_seed(1)
    for name, lo, hi in (("k", -12, 1), ("v", -14, 12)):
        x = getattr(b, name)[0] * torch.exp2(torch.randint(lo, hi, (700, 1, 1), generator=g).float())
        c, e, held = R8.hold(x)
        getattr(b, name)[0] = held
        for p in range(700):
            at = int(b.table[0, p // 32]), slice(None), p % 32
            getattr(b, name + "_pages").view(U8)[at] = c[p].view(U8)
            getattr(b, name + "_scale").view(U8)[at] = e[p]
    b.q = (b.q.float() * torch.exp2(torch.randint(-20, 3, (new, 4, 1), generator=g).float())).to(BF16)
    out, lse = _attend8(b)
    _check(b, out, lse)


def test_attention8_with_one_key_far_above_the_rest():
    """Thousands of keys that share a few hundredths of the weight, 2^-18 of the first key's each: what they add is not lost."""
    n = 12000
    b = R8.Batch8([(1, n), (30, n)], 4, 1, 128, 128, seed=3, device=DEV, sizes=False)
    for i in (0, 1):
        k = torch.zeros((n, 1, 128))
        k[0, :, 0] = 1.0
        v = torch.where(torch.arange(n) == 0, 0.0, 1.0)[:, None, None].expand(n, 1, 128).clone()
        for name, x in (("k", k), ("v", v)):
            c, e, held = R8.hold(x)
            getattr(b, name)[i] = held
            for p in range(n):
                at = int(b.table[i, p // 128]), slice(None), p % 128
                getattr(b, name + "_pages").view(U8)[at] = c[p].view(U8)
                getattr(b, name + "_scale").view(U8)[at] = e[p]
    b.q = torch.zeros_like(b.q)
    b.q[:, :, 0] = 144.0  # 144 / sqrt(128) = 12.73 = 18.36 log 2
    out, lse = _attend8(b)
    _check(b, out, lse)
    assert 0.02 < float(out[0, 0, 0]) < 0.06


def test_attention8_strided_pools_and_rows():
    b = R8.Batch8([(1, 70), (20, 90)], 8, 2, 128, 32, seed=6, device=DEV)
    pool = torch.stack((b.k_pages.view(U8), b.v_pages.view(U8)), 1).contiguous().to(DEV)
    scale = torch.stack((b.k_scale.view(U8), b.v_scale.view(U8)), 1).contiguous().to(DEV)
    wide = torch.zeros((b.tokens, 8 * 128 + 64), dtype=BF16, device=DEV)
    wide[:, :1024] = b.on("q").view(b.tokens, -1)
    out = torch.full((b.tokens, 2048), 7.0, dtype=BF16, device=DEV)
    lse = torch.full((b.tokens, 11), 7.0, device=DEV)
    table = torch.full((2, 40), -1, dtype=torch.int32, device=DEV)
    table[:, :b.table.shape[1]] = b.on("table")
    _paged().PagedAttention8(8, 2, 128, DEV)(
        wide[:, :1024], pool[:, 0].view(R8.E4M3), pool[:, 1].view(R8.E4M3), scale[:, 0].view(R8.E8M0), scale[:, 1].view(R8.E8M0),
        b.on("cu"), b.on("kv_len"), table[:, :b.table.shape[1]], out[:, 512:1536], lse=lse[:, 1:9])
    torch.cuda.synchronize()
    _check(b, out[:, 512:1536].reshape(-1, 8, 128), lse[:, 1:9])
    assert bool((out[:, :512] == 7).all()) and bool((out[:, 1536:] == 7).all())
    assert bool((lse[:, 0] == 7).all()) and bool((lse[:, 9:] == 7).all())


@pytest.mark.parametrize("what", ["key", "value"])
@pytest.mark.parametrize("spec", [[(1, 9000)], [(3, 700)], [(70, 4000)], [(8, 70), (1, 60)]])
def test_attention8_shows_a_code_of_nan(spec, what):
    """A row that sees a key of NaN is NaN, its log-sum-exp too; other heads' rows are as they are without it. A value of
    NaN reaches its own dim of the rows that see it."""
    at = 50
    b = R8.Batch8(spec, 8, 2, 128, 32, seed=31, device=DEV)
    clean = R8.Batch8(spec, 8, 2, 128, 32, seed=31)
    pool = b.k_pages if what == "key" else b.v_pages
    for i in range(len(spec)):
        pool.view(U8)[int(b.table[i, at // 32]), 1, at % 32, 7] = 0x7f
    out, lse = (x.cpu() for x in _attend8(b))
    ref, ref_lse, tol, lse_tol = R.attention(clean)
    for i, t, pos in b.rows():
        if at > pos:
            continue
        for h in range(8):
            if h >= 4 and what == "key":
                assert bool(out[t, h].isnan().all()) and bool(lse[t, h].isnan()), (i, t, h)
                continue
            dims = torch.arange(128) != 7 if h >= 4 else torch.ones(128, dtype=torch.bool)
            assert bool(((out[t, h].double() - ref[t, h]).abs() <= tol[t, h])[dims].all()), (i, t, h)
            assert bool(out[t, h, ~dims].isnan().all())
            assert float((lse[t, h].double() - ref_lse[t, h]).abs()) <= float(lse_tol[t, h])


@pytest.mark.parametrize("new", [1, 30])
@pytest.mark.parametrize("what", [math.nan, math.inf])
def test_attention8_of_queries_that_are_not_numbers(what, new):
    b = R8.Batch8([(new, 2000)], 8, 2, 128, 64, seed=5, device=DEV)
    b.q[0, 3, 11] = what
    out, lse = _attend8(b)
    assert bool(out[0, 3].isnan().all()) and bool(lse[0, 3].isnan())
    other = torch.ones((b.tokens, 8), dtype=torch.bool)
    other[0, 3] = False
    ref, ref_lse, tol, lse_tol = R.attention(b)
    assert bool(((out.cpu().double() - ref).abs() <= tol)[other].all())
    assert bool(((lse.cpu().double() - ref_lse).abs() <= lse_tol)[other].all())


def test_attention8_flags_what_it_cannot_reach():
    b = R8.Batch8([(1, 100), (1, 60), (20, 90)], 4, 1, 128, 32, seed=3, device=DEV)
    b.table[0, 1] = b.pages  # one past the pool
    b.table[2, 1] = -1
    err = _err()
    out, _ = _attend8(b, err=err)
    assert int(err.item()) == 128
    # a page that is not there reads as zeros
    for i in (0, 2):
        b.k[i][32:64], b.v[i][32:64] = 0, 0
    _check(b, out, None)
    b = R8.Batch8([(1, 64), (1, 60), (20, 64)], 4, 1, 128, 32, seed=3, device=DEV)
    b.table, b.kv_len = b.table[:, :2].contiguous(), torch.tensor([65, 60, 64], dtype=torch.int32)
    err = _err()
    out, _ = _attend8(b, err=err)
    assert int(err.item()) == 128
    ref, _, tol, _ = R.attention(b)
    assert bool(((out.double().cpu() - ref).abs() <= tol).all()), "a request cut to its table row uses the row's keys"


def test_attention8_scratch_is_made_ready_again():
    """A call that ends early leaves counts in the scratch, as they are set here; after reset() the object answers as a
    new one does."""
    b = R8.Batch8([(1, 2900), (70, 1333), (1, 5)], 8, 2, 128, 32, seed=1, device=DEV)
    handle = _paged().PagedAttention8(8, 2, 128, DEV)
    first, _ = _attend8(b, handle)
    handle.scratch[:16 * handle.grid] = 1
    handle.reset()
    out, lse = _attend8(b, handle)
    _check(b, out, lse)
    assert torch.equal(out, first)


@pytest.mark.parametrize("pdl", [True, False])
def test_attention8_calls_in_a_row_on_what_the_last_one_wrote(pdl):
    """Queries written by the kernel before, and results read by the kernel after, with both kernels at work: neither starts
    before what it reads is there, nor does a later call overtake an earlier one's kernels."""
    b = R8.Batch8([(1, 3000), (60, 900), (1, 700), (2, 90)], 8, 2, 128, 32, seed=7, device=DEV)
    handle = _paged().PagedAttention8(8, 2, 128, DEV)
    pools = [b.on(n) for n in ("k_pages", "v_pages", "k_scale", "v_scale")]
    cu, kv_len, table, q0 = b.on("cu"), b.on("kv_len"), b.on("table"), b.on("q")
    want, _ = _attend8(b, handle)
    q, out, sums = torch.zeros_like(q0), torch.empty_like(q0), []
    for k in range(6):
        q.zero_()
        handle(q, *pools, cu, kv_len, table, out, pdl=pdl)
        q.copy_(q0)
        handle(q, *pools, cu, kv_len, table, out, pdl=pdl)
        sums.append(out.clone())
        out.fill_(math.nan)
    torch.cuda.synchronize()
    assert all(torch.equal(s, want) for s in sums)


def test_attention8_in_a_graph_follows_the_lengths():
    P = _paged()
    b = R8.Batch8([(1, 400), (20, 300)], 4, 1, 128, 16, seed=12, device=DEV)
    handle = P.PagedAttention8(4, 1, 128, DEV)
    pools = [b.on(n) for n in ("k_pages", "v_pages", "k_scale", "v_scale")]
    q, table, cu, kv_len = b.on("q"), b.on("table"), b.on("cu"), b.on("kv_len")
    out = torch.zeros((21, 4, 128), dtype=BF16, device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        handle(q, *pools, cu, kv_len, table, out)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            handle(q, *pools, cu, kv_len, table, out)
    for lens in ([400, 300], [129, 20], [1, 255]):
        kv_len.copy_(torch.tensor(lens, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        c = R8.Batch8([(1, lens[0]), (20, lens[1])], 4, 1, 128, 16, seed=12)
        c.q, c.k, c.v = b.q, [x[:n] for x, n in zip(b.k, lens)], [x[:n] for x, n in zip(b.v, lens)]
        ref, _, tol, _ = R.attention(c)
        assert bool(((out.double().cpu() - ref).abs() <= tol).all()), lens


def test_append8_then_attention8_on_another_stream():
    """The two calls as a model layer makes them, on a stream of their own and without host waits."""
    P = _paged()
    b = R8.Batch8([(1, 90), (17, 40), (1, 1)], 8, 2, 128, 16, seed=21, device=DEV)
    cos, sin = P.rope_table(128, 128, 5e6, DEV)
    handle = P.PagedAttention8(8, 2, 128, DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        q = torch.empty((b.tokens, 8, 128), dtype=BF16, device=DEV)
        out = torch.empty_like(q)
        pools = [b.on(n) for n in ("k_pages", "v_pages", "k_scale", "v_scale")]
        cu, kv_len, table = b.on("cu"), b.on("kv_len"), b.on("table")
        P.rope_append8(b.on("qkv"), cu, kv_len, table, 8, 2, cos, sin, q, *pools)
        handle(q, *pools, cu, kv_len, table, out)
    side.synchronize()
    kc, vc = P.held_values(pools[0], pools[2]).cpu(), P.held_values(pools[1], pools[3]).cpu()
    b.q = q.cpu()
    for i, (_, kv) in enumerate(b.spec):
        at = [(int(b.table[i, p // 16]), p % 16) for p in range(kv)]
        b.k[i], b.v[i] = torch.stack([kc[a, :, r] for a, r in at]), torch.stack([vc[a, :, r] for a, r in at])
    ref, _, tol, _ = R.attention(b)
    assert bool(((out.double().cpu() - ref).abs() <= tol).all())
