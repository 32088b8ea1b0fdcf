"""qd_sample on the GPU against its definition in 64 bits.

The reference orders the tokens and sums their weights in float64, so it knows the kept set and the share of
every token up to the rounding of the fp32 weights: a weight is off by at most 2^-21 of itself (expf within 2
ulps, the rounding of d) + |d| 2^-23 and 2^-41 of the largest (the fixed point). A drawn token is right when
u lies in its interval of the kept running sum, widened by that much; a token is kept rightly when it is
inside, or within that much of, the cut."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def _draw(logits, u, **kw):
    from decode_b200.sample import sample

    rows = logits.shape[0]
    tok = torch.full((rows,), -5, dtype=torch.int64, device=DEV)
    lp = torch.full((rows,), 5.0, device=DEV)
    dt = {"top_k": torch.int32}
    kw = {k: v if v is None or torch.is_tensor(v) and v.is_cuda else
          torch.as_tensor(v).to(dt.get(k, torch.float32)).expand(rows).contiguous().to(DEV) for k, v in kw.items()}
    sample(logits.to(DEV), torch.as_tensor(u, dtype=torch.float32).expand(rows).contiguous().to(DEV), tok, logprob=lp, **kw)
    torch.cuda.synchronize()
    return tok.cpu(), lp.cpu()


def _row_ok(l, u, tok, lp, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """Checks one row's draw; l float64 logits, NaN already -inf."""
    n = len(l)
    top = l.max()
    d = (l - top) / temperature
    w = d.exp()
    order = torch.sort(l, descending=True, stable=True).indices
    ws = w[order]
    rel = 2.0 ** -21 + 2.0 ** -22 * min(40.0, float(-d[w > 2.0 ** -42].min()))
    slack = float(rel * ws.sum() + n * 2.0 ** -41)
    k = top_k if 0 < top_k < n else n
    c = ws.cumsum(0)
    want = top_p * float(c[k - 1])
    sure = maybe = k  # lengths of the surely and of the possibly kept prefix
    if top_p < 1:
        before = c[:k] - ws[:k]
        sure, maybe = max(1, int((before < want - slack).sum())), max(1, int((before < want + slack).sum()))
    if min_p > 0:
        floor = math.log(min(min_p, 1.0))
        near = 2.0 ** -20 * (1 + abs(floor))
        sure, maybe = min(sure, max(1, int((d[order] >= floor + near).sum()))), min(maybe, max(1, int((d[order] >= floor - near).sum())))
    place = int((order == tok).nonzero())
    assert place < maybe, f"token {tok} at place {place} is not among the {maybe} kept"
    lo, hi, shares = math.inf, -math.inf, []
    for kept in {sure, maybe}:  # the interval of the token under either kept set
        x = torch.zeros_like(w)
        x[order[:kept]] = ws[:kept]
        total, upto = float(x.sum()), float(x[:tok + 1].sum())
        lo, hi = min(lo, (upto - float(x[tok]) - slack) / total), max(hi, (upto + slack) / total)
        shares.append(float(d[tok]) - math.log(total))
    if sure == maybe:  # otherwise the cut itself is in doubt by one token or a tie
        assert lo <= u <= hi, f"u {u} is outside [{lo}, {hi}] of token {tok}"
    tol = 2.0 ** -20 * (1 + abs(float(d[tok])) + abs(shares[0])) + slack
    assert min(shares) - tol <= lp <= max(shares) + tol, (lp, shares)


def _check(logits, u, **kw):
    tok, lp = _draw(logits, u, **kw)
    rows = logits.shape[0]
    at = lambda v, i: float(v if not torch.is_tensor(v) else v.reshape(-1)[i if v.numel() > 1 else 0])  # noqa: E731
    for i in range(rows):
        l = logits[i].double().cpu()
        l = torch.where(l.isnan(), -math.inf, l)
        k = {n: at(v, i) for n, v in kw.items() if v is not None}
        if "top_k" in k:
            k["top_k"] = int(k["top_k"])
        if k.get("temperature", 1.0) >= 1e-5:
            _row_ok(l, at(torch.as_tensor(u, dtype=torch.float32), i), int(tok[i]), float(lp[i]), **k)
        else:
            assert int(tok[i]) == int((l == l.max()).nonzero()[0]) and float(lp[i]) == 0
    return tok, lp


def _logits(rows, n, dtype, seed=0, spread=2.5, lead=12.0):
    g = torch.Generator().manual_seed(seed)
    x = spread * torch.randn((rows, n), generator=g)
    hot = torch.randint(0, n, (rows, min(n, 40)), generator=g)
    x.scatter_(1, hot, lead - 8 * torch.rand(hot.shape, generator=g))
    return x.to(dtype), torch.rand((rows,), generator=g)


FILTERS = {"none": {}, "top_k": {"top_k": 20}, "top_p": {"top_p": 0.9}, "min_p": {"min_p": 0.05},
           "all": {"top_k": 50, "top_p": 0.95, "min_p": 0.01}, "k_past_the_row": {"top_k": 10 ** 6}, "one": {"top_k": 1},
           "tiny_p": {"top_p": 1e-9}, "zero_p": {"top_p": 0.0}, "p_near_one": {"top_p": 0.9999}, "min_one": {"min_p": 1.0},
           "min_above_one": {"min_p": 3.0}, "wide_k": {"top_k": 700}}


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("n", [1, 2, 7, 64, 1000, 1025, 5003, 151936])
@pytest.mark.parametrize("name", list(FILTERS))
def test_filters_at_sizes(name, n, dtype):
    rows = 6
    x, u = _logits(rows, n, dtype, seed=n)
    _check(x, u, temperature=0.8, **FILTERS[name])


@pytest.mark.parametrize("rows", [1, 2, 3, 17, 33, 75, 149, 300])
def test_row_counts(rows):
    x, u = _logits(rows, 3001, BF16, seed=rows)
    _check(x, u, temperature=1.2, top_k=30, top_p=0.9)


def test_every_row_with_its_own_settings():
    rows = 48
    g = torch.Generator().manual_seed(3)
    x, u = _logits(rows, 20011, BF16, seed=8)
    t = 0.3 + 1.5 * torch.rand((rows,), generator=g)
    t[::7] = 0
    k = torch.randint(0, 90, (rows,), generator=g)
    k[::5] = -3
    p = 0.3 + 0.8 * torch.rand((rows,), generator=g)
    m = 0.2 * torch.rand((rows,), generator=g)
    m[::3] = 0
    _check(x, u, temperature=t, top_k=k, top_p=p, min_p=m)


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_equal_logits_are_ordered_by_index(dtype):
    """All logits equal, and two levels: the kept ones are the lowest indices, drawn evenly."""
    n, rows = 40000, 64
    u = (torch.arange(rows) + 0.5) / rows
    flat = torch.full((rows, n), 3.0, dtype=dtype)
    tok, lp = _check(flat, u, top_k=1000)
    assert torch.equal(tok, (u * 1000).floor().long())
    assert bool(((lp + math.log(1000)).abs() < 1e-5).all())
    tok, _ = _check(flat, u, top_p=0.25)
    assert torch.equal(tok, (u * 10000).floor().long())
    tok, _ = _check(flat, u)
    assert torch.equal(tok, (u * n).floor().long())
    flat[:, 20000:20010] = 4.0  # ten above the rest
    tok, _ = _check(flat, u, top_k=15)
    assert set(tok.tolist()) <= set(range(5)) | set(range(20000, 20010))
    assert bool((_check(flat, u, temperature=0.0)[0] == 20000).all())


def test_masked_and_broken_logits():
    n = 2000
    x, _ = _logits(8, n, FP32, seed=1)
    x[0, :] = -math.inf                     # nothing to draw from
    x[1, :] = math.nan
    x[2, 5:] = -math.inf                    # five tokens left
    x[3, ::2] = math.nan                    # NaN counts as masked
    x[4, 7] = x[4, 9] = math.inf            # share everything
    x[5, :] = -math.inf
    x[5, 1234] = -3e38                      # one token, however small
    x[6, :] = torch.finfo(FP32).min         # a mask of the type's lowest value, over the whole row
    x[7, 100:] = torch.finfo(FP32).min
    for kw in ({}, {"top_k": 3}, {"top_p": 0.8}, {"min_p": 0.1}, {"top_k": 4, "top_p": 0.9, "min_p": 0.01}, {"temperature": 0.0}):
        tok, lp = _draw(x, 0.6, **kw)
        assert tok[0] == -1 and tok[1] == -1 and lp[0] == -math.inf and lp[1] == -math.inf
        assert 0 <= tok[2] < 5 and tok[3] % 2 == 1 and tok[5] == 1234 and lp[5] == 0 and 0 <= tok[7] < 100
        assert tok[4] == (7 if kw.get("temperature") == 0.0 else 9), kw
        assert 0 <= tok[6] < n
    tok, lp = _draw(x[4:5], 0.4)
    assert tok[0] == 7 and abs(float(lp[0]) + math.log(2)) < 1e-6


def test_extreme_u_and_temperature():
    x, _ = _logits(4, 3000, BF16, seed=9)
    rows = x.repeat(4, 1)
    u = torch.tensor([0.0, 1.0 - 2.0 ** -24, -1.0, math.nan, 1.0, 7.0, 0.0, 0.0, 0.5, 0.5, 0.5, 0.5, 0.5, 0.5, 0.5, 0.5])
    t = torch.tensor([1.0] * 8 + [1e-5, 2e-5, 1e4, math.inf, math.nan, -1.0, 0.0, 1e-30])
    tok, lp = _draw(rows, u, temperature=t, top_k=50)
    assert bool((tok >= 0).all()) and bool((tok < 3000).all())
    order = torch.sort(x.float(), descending=True, stable=True).indices
    for i in (0, 2, 3, 6, 7):  # u at or below 0 (or NaN): the kept token of the lowest index
        assert int(tok[i]) == int(order[i % 4][:50].min())
    for i in (1, 4, 5):        # u at or above 1: the last kept token (of 2^-40 or more, which these all have)
        assert int(tok[i]) == int(order[i % 4][:50].max())
    for i in range(12, 16):    # not a temperature of at least 1e-5: the first of the largest
        assert int(tok[i]) == int(x[i % 4].float().argmax()) and float(lp[i]) == 0
    first = order[3][:50].sort().values
    assert int(tok[11]) == int(first[25])  # an infinite temperature: all kept tokens alike


def test_strided_rows_and_part_of_a_row():
    from decode_b200.sample import sample

    x, u = _logits(5, 1004, BF16, seed=2)
    for shift in (0, 1, 3):
        for width in (1004, 1003):
            wide = torch.full((5, 1111), 99.0, dtype=BF16, device=DEV)
            wide[:, shift:shift + width] = x[:, :width].to(DEV)
            tok = torch.empty((5,), dtype=torch.int64, device=DEV)
            sample(wide[:, shift:], u.to(DEV), tok, vocab=width)
            ref, _ = _draw(x[:, :width].contiguous(), u)
            assert torch.equal(tok.cpu(), ref)
            for i in range(5):
                _row_ok(x[i, :width].double(), float(u[i]), int(tok[i]), float(_draw(x[:, :width].contiguous(), u)[1][i]))


def test_draws_follow_the_distribution():
    """One row drawn with evenly spaced numbers: every token comes up its share of the times, to one draw."""
    x, _ = _logits(1, 500, FP32, seed=5, lead=5.0)
    n = 4096
    u = (torch.arange(n) + 0.5) / n
    tok, _ = _draw(x.expand(n, -1).contiguous(), u, temperature=1.0, top_p=0.9)
    w = torch.softmax(x[0].double(), 0)
    order = torch.sort(x[0], descending=True, stable=True).indices
    kept = int(((w[order].cumsum(0) - w[order]) < 0.9).sum())
    share = torch.zeros_like(w)
    share[order[:kept]] = w[order[:kept]] / w[order[:kept]].sum()
    count = torch.bincount(tok, minlength=500).double()
    assert bool(((count - n * share).abs() <= 1.01).all())
    assert bool((tok[1:] >= tok[:-1]).all()), "a larger number never draws a lower index"


def test_repeats_bit_for_bit_and_in_a_graph():
    x, u = _logits(40, 30011, FP32, seed=6)
    a = _draw(x, u, temperature=0.9, top_p=0.95)
    assert all(torch.equal(p, q) for p, q in zip(a, _draw(x, u, temperature=0.9, top_p=0.95)))
    from decode_b200.sample import sample

    xd, ud, tok = x.to(DEV), u.to(DEV), torch.zeros((40,), dtype=torch.int64, device=DEV)
    t, p = torch.full((40,), 0.9, device=DEV), torch.full((40,), 0.95, device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        sample(xd, ud, tok, temperature=t, top_p=p)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            sample(xd, ud, tok, temperature=t, top_p=p)
    tok.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(tok.cpu(), a[0])


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("n", [3000, 100003])
@pytest.mark.parametrize("spread", [1e-4, 0.02, 0.5])
@pytest.mark.parametrize("kept", [{"top_k": 2000}, {"top_p": 0.6}, {"top_k": 2500, "top_p": 0.5}, {"top_k": 10 ** 6, "top_p": 0.999}])
def test_many_tokens_of_nearly_the_same_weight(kept, spread, n, dtype):
    # thousands within a step of d, so that the cut is refined by value, and more than a short count of them holds
    g = torch.Generator().manual_seed(n)
    x = (spread * torch.randn((4, n), generator=g)).to(dtype)
    x[1, ::3] = -math.inf
    x[2, n // 2:] = x[2, 0]
    _check(x, torch.rand((4,), generator=g), temperature=1.0, **kept)


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("kept", ["none", "top_p", "all"])
def test_largest_vocabulary(kept, dtype):
    x, u = _logits(3, 1 << 18, dtype, seed=5)
    u[0] = 0.9999999  # ends in the last part of the row
    _check(x, u, temperature=1.1, **FILTERS[kept])


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("kept", ["none", "all"])
def test_many_more_clusters_than_fit_the_gpu(kept, dtype):
    """CTAs come and go while others of the same call run; a row's draw does not depend on the rows beside it,
    nor on how many CTAs share it (fewer where there are more rows)."""
    rows = 1200
    x, u = _logits(rows, 30011, dtype, seed=11)
    kw = {k: torch.as_tensor(v).expand(rows) for k, v in FILTERS[kept].items()}
    tok, lp = _draw(x, u, **kw)
    for at in range(0, rows, 100):
        some = slice(at, at + (at // 100) % 3 + 1)
        part, part_lp = _draw(x[some].contiguous(), u[some], **{k: v[some] for k, v in kw.items()})
        assert torch.equal(tok[some], part) and torch.equal(lp[some], part_lp)
    for i in range(0, rows, 97):
        _row_ok(x[i].double(), float(u[i]), int(tok[i]), float(lp[i]), **FILTERS[kept])
