"""Attention of requests that share their beginnings (qd_prefix_attn) on the GPU against the definition in 64 bits
(tests/paged_ref.py), with the tolerances of the attention that reads every request's keys: the two parts of a row are
joined in fp32."""

import math

import pytest
import torch

import paged_ref as R
from test_paged_gpu import _check, _err

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16, FP16 = torch.bfloat16, torch.float16


def _paged():
    from decode_b200 import paged

    return paged


class Groups(R.Batch):
    """Groups (common positions, [(new tokens, positions after the common ones)]): each group's table rows name its first
    request's pages for the common positions (whole pages), and hold junk where the page is not a common one's."""

    def __init__(self, groups, nq, nkv, dim, page, *args, told=None, alone=0, **kw):
        spec = [(n, p + own) for p, rs in groups for n, own in rs]
        super().__init__(spec, nq, nkv, dim, page, *args, **kw)
        at, bounds = 0, [0]
        for p, rs in groups:
            assert p % page == 0
            for i in range(at + 1, at + len(rs)):
                for e in range(p // page):  # the page that was its own is nobody's
                    self.k_pages[int(self.table[i, e])] = self.v_pages[int(self.table[i, e])] = math.nan
                self.table[i, :p // page] = self.table[at, :p // page]
                self.k[i][:p], self.v[i][:p] = self.k[at][:p], self.v[at][:p]
            at += len(rs)
            bounds.append(at)
        keep = len(groups) - alone  # the last `alone` groups are not told of: their requests stand alone
        self.cu_groups = torch.tensor(bounds[:keep + 1], dtype=torch.int32)
        self.prefix_len = torch.tensor([p for p, _ in groups] if told is None else told, dtype=torch.int32)[:keep]


def _attend(b, handle=None, scale=None, lse=True, err=None):
    P = _paged()
    handle = handle or P.PrefixAttention(b.nq, b.nkv, b.dim, DEV, b.tokens, len(b.spec), dtype=b.dtype)
    out = torch.full((b.tokens, b.nq, b.dim), 7.0, dtype=b.dtype, device=DEV)
    z = torch.full((b.tokens, b.nq), 7.0, dtype=torch.float32, device=DEV) if lse else None
    handle(b.on("q"), b.on("k_pages"), b.on("v_pages"), b.on("cu"), b.on("kv_len"), b.on("table"), b.on("cu_groups"),
           b.on("prefix_len"), out, lse=z, scale=scale, err=err)
    torch.cuda.synchronize()
    return out, z


GROUPS = {
    "one-request": [(512, [(1, 70)])],
    "two-requests": [(128, [(1, 1), (1, 200)])],
    "decode": [(640, [(1, 1 + 37 * i % 300) for i in range(20)])],
    "decode-many": [(1024, [(1, 5 + i) for i in range(70)])],
    "no-common-block": [(96, [(1, 3)] * 9)],
    "nothing-common": [(0, [(1, 40)] * 5)],
    "groups": [(256, [(1, 9)] * 7), (0, [(1, 300)]), (1280, [(1, 130), (0, 60), (1, 1), (1, 129), (1, 2)] * 2), (512, [(0, 0)] * 3)],
    "chunks": [(512, [(9, 9), (70, 200), (33, 33), (1, 500)])],
    "long-chunks": [(768, [(150, 150), (131, 260), (200, 201)])],
    "few-rows": [(2048, [(1, 3), (2, 5), (1, 700)])],
}


@pytest.mark.parametrize("page", [16, 64, 128])
@pytest.mark.parametrize("groups", list(GROUPS))
def test_prefix_groups(groups, page):
    if any(p % page for p, _ in GROUPS[groups]):  # (common are whole pages)
        page = 32
    b = Groups(GROUPS[groups], 8, 2, 128, page, seed=len(groups) + page, device=DEV, pad_tokens=2)
    err = _err()
    out, lse = _attend(b, err=err)
    _check(b, out, lse)
    assert int(err.item()) == 0


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("nq,nkv,dim,page", [(4, 4, 64, 32), (14, 2, 64, 16), (6, 2, 128, 16), (5, 1, 128, 32), (32, 8, 128, 128),
                                             (33, 1, 128, 16), (128, 1, 64, 16)])
def test_prefix_head_layouts_and_types(nq, nkv, dim, page, dtype):
    b = Groups([(1024, [(1, 130), (19, 150), (3, 3), (1, 64), (1, 1), (1, 9)]), (384, [(1, 5)] * 11)], nq, nkv, dim, page, dtype,
               seed=nq + dim, device=DEV)
    out, lse = _attend(b)
    _check(b, out, lse)


@pytest.mark.parametrize("told", [[300, 1024], [129, 0], [-5, 1000], [512, 127]])
def test_prefix_length_told(told):
    """A length that ends inside a block, that is none, and that is less than what the pages have in common."""
    b = Groups([(512, [(1, 30), (40, 44), (1, 300)] * 3), (1024, [(1, 1)] * 12)], 8, 2, 128, 32, seed=3, device=DEV, told=told)
    _check(b, *_attend(b))


def test_prefix_reaches_into_new_tokens():
    """New tokens inside the common pages: a request that is answered for a second time has all its positions in them."""
    b = Groups([(640, [(1, 0), (1, 0), (3, 0), (1, 20), (1, 128)])], 8, 2, 128, 64, seed=5, device=DEV)
    _check(b, *_attend(b))


def test_prefix_requests_outside_any_group():
    b = Groups([(512, [(1, 30)] * 9), (256, [(1, 7), (5, 80)]), (128, [(60, 200)])], 8, 2, 128, 16, seed=6, device=DEV, alone=2)
    _check(b, *_attend(b))
    b = Groups([(512, [(1, 30)] * 4)], 8, 2, 128, 16, seed=6, device=DEV, alone=1)
    _check(b, *_attend(b))


@pytest.mark.parametrize("groups,nq,nkv,dim,page,dtype", [
    ([(4096, [(1, 1 + 61 * i % 700) for i in range(64)])], 32, 8, 128, 64, BF16),
    ([(8192, [(1, 300)] * 4)] * 4, 32, 8, 128, 64, BF16), ([(2048, [(129 - 4 * i, 129) for i in range(8)])], 16, 4, 128, 16, FP16),
    ([(3008, [(1, 100)] * 30), (1024, [(40, 90)] * 5)], 14, 2, 64, 16, FP16)])
def test_prefix_large(groups, nq, nkv, dim, page, dtype):
    """Both kinds of work on every SM, cut and whole, several times with the same bits, on one object."""
    b = Groups(groups, nq, nkv, dim, page, dtype, seed=17, device=DEV)
    ref, ref_lse, tol, lse_tol = R.attention_on_gpu(b, DEV)
    handle, first, err = _paged().PrefixAttention(nq, nkv, dim, DEV, b.tokens + 7, len(b.spec) + 3, dtype=dtype), None, _err()
    for _ in range(8):
        out, lse = _attend(b, handle, err=err)
        assert int(err.item()) == 0
        d = (out.double() - ref).abs()
        assert bool((d <= tol).all()), (int((~(d <= tol)).sum()), float(d.max()))
        assert bool(((lse.double() - ref_lse).abs() <= lse_tol).all())
        first = out if first is None else first
        assert torch.equal(out, first)


def test_prefix_scale_no_lse_and_strides():
    b = Groups([(512, [(1, 30), (4, 80), (1, 2), (1, 1), (1, 90)])], 8, 2, 128, 32, seed=2, device=DEV, pad_tokens=3)
    out, lse = _attend(b, scale=0.3)
    _check(b, out, lse, scale=0.3)
    out2, none = _attend(b, scale=0.3, lse=False)
    assert none is None and torch.equal(out, out2)
    wide = torch.zeros((b.tokens, 8 * 128 + 64), dtype=BF16, device=DEV)
    wide[:, :1024] = b.on("q").view(b.tokens, -1)
    to = torch.full((b.tokens, 2048), 7.0, dtype=BF16, device=DEV)
    z = torch.full((b.tokens, 11), 7.0, device=DEV)
    pool = torch.stack((b.on("k_pages"), b.on("v_pages")), 1).contiguous()
    P = _paged()
    P.PrefixAttention(8, 2, 128, DEV, b.tokens, 5)(wide[:, :1024], pool[:, 0], pool[:, 1], b.on("cu"), b.on("kv_len"), b.on("table"),
                                                   b.on("cu_groups"), b.on("prefix_len"), to[:, 512:1536], lse=z[:, 1:9])
    torch.cuda.synchronize()
    _check(b, to[:, 512:1536].reshape(-1, 8, 128), z[:, 1:9])
    assert bool((to[:, :512] == 7).all()) and bool((to[:, 1536:] == 7).all())
    assert bool((z[:, 0] == 7).all()) and bool((z[:, 9:] == 7).all())


def test_prefix_common_keys_far_above_and_below_the_own():
    """Rows whose weight is all in the common part, or all in the own."""
    b = Groups([(512, [(1, 100)] * 8)], 4, 1, 128, 64, seed=8, device=DEV)
    for i in range(8):
        own = slice(512, 612)
        b.k[i][:512] = 0.5
        b.k[i][own] = -0.5 if i % 2 else 2.0
        for p in range(612):
            b.k_pages[int(b.table[i, p // 64]), :, p % 64] = b.k[i][p]
    b.q = (b.q.float().abs() * 3).to(BF16)
    _check(b, *_attend(b))


def test_prefix_shows_what_is_not_a_number():
    """A common key of NaN reaches every row of its group and head, an own one its request's rows, and no others."""
    b = Groups([(512, [(1, 100)] * 6), (512, [(1, 90)] * 6)], 8, 2, 128, 64, seed=9, device=DEV)
    clean = Groups([(512, [(1, 100)] * 6), (512, [(1, 90)] * 6)], 8, 2, 128, 64, seed=9)
    b.k_pages[int(b.table[0, 1]), 1, 5] = math.nan
    b.k_pages[int(b.table[8, 9]), 0, 0] = math.nan
    out, lse = (x.cpu() for x in _attend(b))
    ref, ref_lse, tol, lse_tol = R.attention(clean)
    for t in range(12):
        for h in range(8):
            if (t < 6 and h >= 4) or (t == 8 and h < 4):
                assert bool(out[t, h].isnan().all()) and bool(lse[t, h].isnan()), (t, h)
            else:
                assert bool(((out[t, h].double() - ref[t, h]).abs() <= tol[t, h]).all()), (t, h)
                assert float((lse[t, h].double() - ref_lse[t, h]).abs()) <= float(lse_tol[t, h])


def test_prefix_flags_what_it_cannot_reach():
    b = Groups([(256, [(1, 40)] * 6), (128, [(1, 30)])], 4, 1, 128, 32, seed=3, device=DEV)
    b.table[:6, 1] = b.pages  # one past the pool
    err = _err()
    out, _ = _attend(b, err=err)
    assert int(err.item()) == 128
    for i in range(6):
        b.k[i][32:64], b.v[i][32:64] = 0, 0
    _check(b, out, None)
    b = Groups([(256, [(1, 40)] * 6)], 4, 1, 128, 32, seed=3, device=DEV)
    b.table = b.table[:, :9].contiguous()
    err = _err()
    _attend(b, err=err)
    assert int(err.item()) == 128, "a request longer than its table row"


def test_prefix_in_a_graph_follows_the_lengths_and_groups():
    P = _paged()
    shape = [(512, [(1, 400), (2, 300), (1, 64), (1, 65)]), (256, [(1, 20)] * 8)]
    b = Groups(shape, 4, 1, 128, 16, seed=12, device=DEV)
    handle = P.PrefixAttention(4, 1, 128, DEV, b.tokens, 12)
    args = {n: b.on(n) for n in ("q", "k_pages", "v_pages", "cu", "kv_len", "table", "cu_groups", "prefix_len")}
    out = torch.zeros((b.tokens, 4, 128), dtype=BF16, device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        handle(*args.values(), out)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            handle(*args.values(), out)
    for short, told in ((0, [512, 256]), (9, [512, 0]), (19, [130, 256])):
        args["kv_len"].copy_(b.kv_len - short)
        args["prefix_len"].copy_(torch.tensor(told, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        c = Groups(shape, 4, 1, 128, 16, seed=12)
        c.spec = [(n, kv - short) for n, kv in c.spec]
        c.k, c.v = [x[:len(x) - short] for x in c.k], [x[:len(x) - short] for x in c.v]
        ref, _, tol, _ = R.attention(c)
        assert bool(((out.double().cpu() - ref).abs() <= tol).all()), (short, told)


def test_append_then_prefix_attention_on_another_stream():
    """A model layer's calls over a cache whose requests share pages."""
    P = _paged()
    b = Groups([(512, [(1, 90), (17, 40), (1, 1), (1, 7), (1, 300)])], 8, 2, 128, 16, seed=21, device=DEV)
    cos, sin = P.rope_table(1024, 128, 5e6, DEV)
    handle = P.PrefixAttention(8, 2, 128, DEV, b.tokens, 5)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        q = torch.empty((b.tokens, 8, 128), dtype=BF16, device=DEV)
        out = torch.empty_like(q)
        k, v, cu, kv_len, table = b.on("k_pages"), b.on("v_pages"), b.on("cu"), b.on("kv_len"), b.on("table")
        P.rope_append(b.on("qkv"), cu, kv_len, table, 8, 2, cos, sin, q, k, v)
        handle(q, k, v, cu, kv_len, table, b.on("cu_groups"), b.on("prefix_len"), out)
    side.synchronize()
    kc, vc = k.cpu(), v.cpu()
    b.q = q.cpu()
    for i, (_, kv) in enumerate(b.spec):
        at = [(int(b.table[i, p // 16]), p % 16) for p in range(kv)]
        b.k[i], b.v[i] = torch.stack([kc[a, :, r] for a, r in at]), torch.stack([vc[a, :, r] for a, r in at])
    ref, _, tol, _ = R.attention(b)
    assert bool(((out.double().cpu() - ref).abs() <= tol).all())
