"""The serving operators over a paged K/V cache, as measured: what each call is given, what it returns, and its plain form.

  append   q/k RMSNorm, rotary positions and the K/V append of a ragged batch of new tokens into cache pages
  attn     causal attention of each request's new tokens over its pages (one token, or a chunk of them)
  sample   a token per row of logits: temperature, top-k, top-p and min-p, drawn with a given uniform number

A batch is ragged: request i has n_i new tokens (rows cu_tokens[i] .. cu_tokens[i+1] of the token-major
arrays) and, with them, kv_len[i] cached positions; position p lives in row p % page of the page
page_table[i, p // page]. New token j of request i is at position kv_len[i] - n_i + j.

With `own` false `run` computes the operators in elementary torch operations in 32 bits; with `own` true it
calls the package's entry points.
"""

import math
import os
import sys

import torch

own = False

DEVICE = "cuda"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
EPS = 1e-6
THETA = 5e6
FRACTION_BITS = 40  # sampling weights are whole multiples of 2^-40 of the largest: their sums have no rounding


def package():
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "htn-2026_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    from decode_b200 import paged, sample

    return paged, sample


# ------------------------------------------------------------------------------------ cases
def _batch(op, name, batch, chunks, n, kv, page, heads=(32, 8), dim=128, dtype="bf16", norm=True):
    case = {"op": op, "batch": batch, "chunks": chunks, "n": n, "kv": kv, "page": page, "nq": heads[0],
            "nkv": heads[1], "dim": dim, "dtype": dtype}
    if op == "append":
        case["norm"] = norm
    if name:
        case["name"] = name
    return case


def _sample(name, rows, vocab, filters, dtype="bf16"):
    case = {"op": "sample", "rows": rows, "vocab": vocab, "filters": filters, "dtype": dtype}
    if name:
        case["name"] = name
    return case


def listed():
    return [
        # one user's next token: 32 query and 8 K/V heads of 128, the default model's
        _batch("append", "append-1", 1, 0, 1, 1031, 64),
        # a decode step of a full batch
        _batch("append", "append-64", 64, 0, 1, 1536, 16),
        # the prompts of 16 users at once (about 14 k tokens)
        _batch("append", "append-prompts", 16, 16, 1024, 1024, 64),
        # one user's next token after a chat of about a thousand tokens
        _batch("attn", "attn-1", 1, 0, 1, 1031, 64),
        # a decode step of a full batch, 1 to 1.5 k tokens each, in small pages
        _batch("attn", "attn-64", 64, 0, 1, 1536, 16),
        # a decode step of 8 users with long documents
        _batch("attn", "attn-8-long", 8, 0, 1, 40960, 64),
        # what a server runs at a time: 30 users decode while two prompts come in
        _batch("attn", "attn-mixed", 32, 2, 251, 2049, 32),
        # a chunk of a long prompt, after 8192 cached tokens
        _batch("attn", "attn-chunk", 1, 1, 2048, 10240, 128),
        # FP16, heads of 64, seven query heads to a K/V head: another model's short prompts
        _batch("attn", "attn-fp16", 5, 5, 301, 777, 32, heads=(14, 2), dim=64, dtype="fp16"),
        # one user's token, with the model's recommended top-k 20 and top-p 0.95
        _sample("sample-1", 1, 151936, "top_k top_p"),
        # a full batch, where each user has settings of their own (some take the most likely token)
        _sample("sample-64", 64, 151936, "mixed"),
        # many samples for training: 32-bit logits at temperature 1, nothing cut off
        _sample("sample-256-fp32", 256, 151936, "none", dtype="fp32"),
    ]


def _spread(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.4)))))))


def draw(rng):
    op = rng.choice(["append", "attn", "attn", "sample"])
    if op == "sample":
        dtype = rng.choice(["bf16", "fp16", "fp32"])
        filters = rng.choice(["none", "top_k", "top_p", "min_p", "top_k top_p", "mixed", "greedy"])
        return _sample(None, _spread(rng, 1, 256), _spread(rng, 300, 151936), filters, dtype)
    dtype, dim, page = rng.choice(["bf16", "bf16", "fp16"]), rng.choice([64, 128, 128]), rng.choice([16, 32, 64, 128])
    nkv = rng.choice([1, 2, 4, 8])
    heads = (nkv * rng.choice([1, 2, 3, 4, 5, 6, 7, 8]), nkv)
    heads = heads if heads[0] <= 32 else (32, nkv)
    if op == "append":
        batch = _spread(rng, 1, 64)
        chunks = rng.randint(0, batch)
        n = _spread(rng, 1, max(1, min(2048, 14000 // max(1, chunks))))
        return _batch(op, None, batch, chunks, n, n + _spread(rng, 1, 2048), page, heads, dim, dtype, rng.random() < 0.7)
    kind = rng.choice(["decode", "decode", "chunk", "mixed"])
    if kind == "decode":  # up to the listed long batch's keys
        batch = _spread(rng, 1, 96)
        return _batch(op, None, batch, 0, 1, _spread(rng, 1, min(40960, 200000 // batch)), page, heads, dim, dtype)
    if kind == "chunk":
        batch = _spread(rng, 1, 8)
        n = _spread(rng, 2, 2048 // batch)
        return _batch(op, None, batch, batch, n, n + _spread(rng, 1, 8192 // batch), page, heads, dim, dtype)
    batch = rng.randint(3, 40)
    n = _spread(rng, 2, 192)
    return _batch(op, None, batch, rng.randint(1, 3), n, n + _spread(rng, 1, 1900), page, heads, dim, dtype)


def lengths(case):
    """New tokens and cached positions (the new ones included) of each request, by the case alone."""
    b, n, kv = case["batch"], case["n"], case["kv"]
    new = [max(1, n - i * 37 % (n // 4 + 1)) if i < case["chunks"] else 1 for i in range(b)]
    return new, [max(new[i], kv - i * 7919 % (kv // 3 + 1)) for i in range(b)]


def work(case):
    if case["op"] == "sample":
        size = 4 if case["dtype"] == "fp32" else 2
        return {"bytes": case["rows"] * (case["vocab"] * size + 5 * 4 + 12), "flops": 4 * case["rows"] * case["vocab"]}
    new, kv = lengths(case)
    nq, nkv, dim, tokens = case["nq"], case["nkv"], case["dim"], sum(new)
    if case["op"] == "append":
        tables = min(tokens, max(kv)) * dim * 4
        return {"bytes": 2 * 2 * tokens * (nq + 2 * nkv) * dim + tables + 8 * case["batch"] + 4 * tokens,
                "flops": tokens * (nq + nkv) * dim * 8}
    pairs = sum(n * (k - n) + n * (n + 1) // 2 for n, k in zip(new, kv))
    pages = sum(-(-k // case["page"]) for k in kv)
    return {"bytes": 2 * 2 * tokens * nq * dim + 4 * tokens * nq + 2 * 2 * sum(kv) * nkv * dim + 4 * pages + 8 * case["batch"],
            "flops": 4 * nq * dim * pairs}


# ------------------------------------------------------------------------------------ inputs
def _prepare_batch(case, g):
    new, kv = lengths(case)
    page, nkv, dim, dtype = case["page"], case["nkv"], case["dim"], TYPES[case["dtype"]]
    need = [-(-k // page) for k in kv]
    pages, width = sum(need) + 3, max(need)
    order = torch.randperm(pages, generator=g, device=DEVICE).to(torch.int32)  # pages come in any order
    start = torch.tensor([0] + need, device=DEVICE).cumsum(0)[:-1]
    at = start[:, None] + torch.arange(width, device=DEVICE)[None, :]
    table = order[at.clamp(max=pages - 1)].contiguous()
    cu = torch.tensor([0] + new, device=DEVICE).cumsum(0).to(torch.int32)
    rand = lambda *shape: torch.randn(shape, generator=g, device=DEVICE, dtype=torch.float32).to(dtype)  # noqa: E731
    s = {"op": case["op"], "case": case, "cu_tokens": cu, "kv_len": torch.tensor(kv, dtype=torch.int32, device=DEVICE),
         "page_table": table, "tokens": sum(new), "n_max": max(new), "kv_max": max(kv),
         "k_pages": rand(pages, nkv, page, dim), "v_pages": rand(pages, nkv, page, dim)}
    return s, rand


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    if case["op"] == "sample":
        return _prepare_sample(case, g)
    s, rand = _prepare_batch(case, g)
    nq, nkv, dim = case["nq"], case["nkv"], case["dim"]
    if case["op"] == "append":
        s["qkv"] = rand(s["tokens"], (nq + 2 * nkv) * dim)
        s["q_out"] = torch.empty((s["tokens"], nq, dim), dtype=s["qkv"].dtype, device=DEVICE)
        ones = lambda: (1 + 0.2 * rand(dim).float()).to(s["qkv"].dtype)  # noqa: E731
        s["q_norm"], s["k_norm"] = (ones(), ones()) if case["norm"] else (None, None)
        inv = THETA ** (-torch.arange(0, dim, 2, dtype=torch.float64, device=DEVICE) / dim)
        angle = torch.arange(s["kv_max"], dtype=torch.float64, device=DEVICE)[:, None] * inv[None, :]
        s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
        return s
    s["q"] = (2 * rand(s["tokens"], nq, dim).float()).to(s["k_pages"].dtype)  # scores of deviation 2: some keys stand out
    s["out"] = torch.empty_like(s["q"])
    s["lse"] = torch.empty((s["tokens"], nq), dtype=torch.float32, device=DEVICE)
    if own:  # the workspace that a serving program makes once
        s["handle"] = package()[0].PagedAttention(nq, nkv, dim, DEVICE, dtype=s["q"].dtype)
    return s


def _prepare_sample(case, g):
    rows, vocab, kind = case["rows"], case["vocab"], case["filters"]
    uni = lambda *shape: torch.rand(shape, generator=g, device=DEVICE, dtype=torch.float32)  # noqa: E731
    # a language model's rows: a broad bulk, and some likely tokens whose lead differs from row to row
    logits = 2.5 * torch.randn((rows, vocab), generator=g, device=DEVICE, dtype=torch.float32)
    step = vocab // 64
    likely = torch.randint(0, step, (rows, 64), generator=g, device=DEVICE) + step * torch.arange(64, device=DEVICE)
    lead = 8 + 10 * uni(rows, 1)
    logits.scatter_(1, likely, lead - 8 * uni(rows, 64))
    logits[:, vocab // 2::97] = -math.inf  # tokens that a grammar or a user rules out
    s = {"op": "sample", "logits": logits.to(TYPES[case["dtype"]]), "u": uni(rows),
         "tok": torch.empty((rows,), dtype=torch.int64, device=DEVICE),
         "logprob": torch.empty((rows,), dtype=torch.float32, device=DEVICE)}
    s["temperature"] = 0.6 + 0.8 * uni(rows) if kind not in ("none", "greedy") else torch.full((rows,), float(kind == "none"), device=DEVICE)
    mixed = uni(5, rows)
    if kind == "mixed":  # a tenth of the rows greedy; each filter on in a half of them
        s["temperature"] = torch.where(mixed[0] < 0.1, torch.zeros_like(mixed[0]), s["temperature"])
    k = (1 + 99 * uni(rows)).to(torch.int32)
    p, m = 0.5 + 0.49 * uni(rows), 0.2 * uni(rows)
    off = torch.zeros_like(k)
    s["top_k"] = k if "top_k" in kind else torch.where(mixed[1] < 0.5, k, off) if kind == "mixed" else None
    s["top_p"] = p if "top_p" in kind else torch.where(mixed[2] < 0.5, p, torch.ones_like(p)) if kind == "mixed" else None
    s["min_p"] = m if "min_p" in kind else torch.where(mixed[3] < 0.5, m, torch.zeros_like(m)) if kind == "mixed" else None
    return s


# ------------------------------------------------------------------------------------ one pass
def run(s):
    return (_run_own if own else _run_plain)[s["op"]](s)


def _own_append(s):
    c = s["case"]
    package()[0].rope_append(s["qkv"], s["cu_tokens"], s["kv_len"], s["page_table"], c["nq"], c["nkv"], s["cos"], s["sin"],
                             s["q_out"], s["k_pages"], s["v_pages"], q_norm=s["q_norm"], k_norm=s["k_norm"], eps=EPS)
    return s["q_out"], s["k_pages"], s["v_pages"]


def _own_attn(s):
    s["handle"](s["q"], s["k_pages"], s["v_pages"], s["cu_tokens"], s["kv_len"], s["page_table"], s["out"], lse=s["lse"])
    return s["out"], s["lse"]


def _own_sample(s):
    package()[1].sample(s["logits"], s["u"], s["tok"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"],
                        min_p=s["min_p"], logprob=s["logprob"])
    return s["tok"], s["logprob"]


def _positions(s):
    """Request and position of each new token."""
    cu, t = s["cu_tokens"].long(), torch.arange(s["tokens"], device=DEVICE)
    b = torch.searchsorted(cu[1:], t, right=True)
    return b, t - cu[b], s["kv_len"].long()[b] - cu[b + 1] + t


def _plain_append(s):
    c = s["case"]
    nq, nkv, dim, half = c["nq"], c["nkv"], c["dim"], c["dim"] // 2
    b, _, pos = _positions(s)
    x = s["qkv"].float().view(s["tokens"], nq + 2 * nkv, dim)
    q, k, v = x[:, :nq], x[:, nq:nq + nkv], x[:, nq + nkv:]
    if s["q_norm"] is not None:
        q = q * torch.rsqrt(q.square().mean(-1, keepdim=True) + EPS) * s["q_norm"].float()
        k = k * torch.rsqrt(k.square().mean(-1, keepdim=True) + EPS) * s["k_norm"].float()
    cos, sin = s["cos"][pos][:, None, :], s["sin"][pos][:, None, :]
    turn = lambda h: torch.cat((h[..., :half] * cos - h[..., half:] * sin, h[..., half:] * cos + h[..., :half] * sin), -1)  # noqa: E731
    s["q_out"].copy_(turn(q))
    page, row = s["page_table"][b, pos // c["page"]].long(), pos % c["page"]
    s["k_pages"][page, :, row] = turn(k).to(s["k_pages"].dtype)
    s["v_pages"][page, :, row] = v.to(s["v_pages"].dtype)
    return s["q_out"], s["k_pages"], s["v_pages"]


def _plain_attn(s):
    c = s["case"]
    batch, nq, nkv, dim, n = c["batch"], c["nq"], c["nkv"], c["dim"], s["n_max"]
    b, j, pos = _positions(s)
    q = torch.zeros((batch, n, nq, dim), device=DEVICE)
    q[b, j] = s["q"].float()
    last = torch.full((batch, n), -1, dtype=torch.int64, device=DEVICE)  # the last key that a row sees
    last[b, j] = pos
    rows = lambda x: x[s["page_table"].long()].transpose(1, 2).reshape(batch, nkv, -1, dim).float()  # noqa: E731
    k, v = rows(s["k_pages"]), rows(s["v_pages"])
    key = torch.arange(k.shape[2], device=DEVICE)
    v = torch.where((key[None, :] < s["kv_len"][:, None])[:, None, :, None], v, 0.0)
    q = q.view(batch, n, nkv, nq // nkv, dim).permute(0, 2, 3, 1, 4).reshape(batch, nkv, -1, dim)
    score = torch.matmul(q, k.transpose(2, 3)).mul_(1 / math.sqrt(dim)).view(batch, nq, n, -1)
    score.masked_fill_((key[None, None, :] > last[:, :, None])[:, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    p = score.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(batch, nkv, -1, p.shape[-1]), v).view(batch, nq, n, dim) / torch.where(total == 0, 1.0, total)
    s["out"].copy_(o.transpose(1, 2)[b, j])
    s["lse"].copy_((top + total.log())[..., 0].transpose(1, 2)[b, j])
    return s["out"], s["lse"]


def _plain_sample(s):
    scale = 2.0 ** FRACTION_BITS
    logits = s["logits"].float()
    rows, vocab = logits.shape
    logits = torch.where(logits.isnan(), -math.inf, logits)
    top = logits.amax(-1, keepdim=True)
    greedy = ~(s["temperature"] >= 1e-5)
    inv = torch.where(greedy, 1.0, 1.0 / s["temperature"])[:, None]
    d = torch.where(logits == -math.inf, logits, torch.where(logits == top, 0.0, (logits - top) * inv))
    weight = (d.exp().double() * scale).round().long()  # exact in 64 bits: a 24-bit number times a power of two
    order = torch.sort(logits, dim=-1, descending=True, stable=True).indices  # equal logits: the lower index first
    w, rank = weight.gather(1, order), torch.arange(vocab, device=DEVICE)[None, :]
    keep = torch.ones_like(w, dtype=torch.bool)
    if s["top_k"] is not None:
        k = s["top_k"][:, None]
        keep &= (rank < k) | (k <= 0)
    if s["top_p"] is not None:
        p, inside = s["top_p"][:, None], torch.where(keep, w, 0)
        want = (p.double() * inside.sum(-1, keepdim=True).double()).ceil().long()
        keep &= (inside.cumsum(-1) - inside < want) | ~(p < 1)
    if s["min_p"] is not None:
        m = s["min_p"][:, None]
        keep &= (d.gather(1, order) >= m.clamp(max=1.0).log()) | ~(m > 0)
    keep = (keep & ~greedy[:, None]) | (rank == 0)
    w = torch.zeros_like(weight).scatter_(1, order, torch.where(keep, w, 0))
    total = w.sum(-1)
    at = (s["u"].double() * total.double()).floor().long().clamp(min=0)
    at = torch.minimum(at, total - 1)
    tok = (w.cumsum(-1) <= at[:, None]).sum(-1)
    s["logprob"].copy_(d.gather(1, tok[:, None])[:, 0] - (total.float() / scale).log())
    s["tok"].copy_(tok)
    return s["tok"], s["logprob"]


_run_own = {"append": _own_append, "attn": _own_attn, "sample": _own_sample}
_run_plain = {"append": _plain_append, "attn": _plain_attn, "sample": _plain_sample}


# ------------------------------------------------------------------------------------ from the definitions, in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "attn": _exact_attn, "sample": _exact_sample}[case["op"]](case, s)


def _exact_append(case, s):
    """Each pair (x_r, x_{r + dim/2}) of a head is the complex number that its position's angle turns."""
    nq, nkv, dim, page = case["nq"], case["nkv"], case["dim"], case["page"]
    new, kv = lengths(case)
    pools = [s["k_pages"].double(), s["v_pages"].double()]
    q_out, row = [], 0
    for i, (n, total) in enumerate(zip(new, kv)):
        x = s["qkv"][row:row + n].double().view(n, nq + 2 * nkv, dim)
        row += n
        pos = torch.arange(total - n, total, device=DEVICE)
        turn = torch.complex(s["cos"][pos].double(), s["sin"][pos].double())[:, None, :]
        heads = []
        for part, gain in ((x[:, :nq], s["q_norm"]), (x[:, nq:nq + nkv], s["k_norm"])):
            if gain is not None:
                part = gain.double() * part / (part.pow(2).sum(-1, keepdim=True) / dim + EPS).sqrt()
            z = turn * torch.complex(part[..., :dim // 2].contiguous(), part[..., dim // 2:].contiguous())
            heads.append(torch.cat((z.real, z.imag), -1))
        q_out.append(heads[0])
        where = s["page_table"][i].long()[pos // page] * page + pos % page
        for pool, value in zip(pools, (heads[1], x[:, nq + nkv:])):
            for h in range(nkv):
                pool[where // page, h, where % page] = value[:, h]
    return torch.cat(q_out), pools[0], pools[1]


def _exact_attn(case, s):
    nq, nkv, dim, page = case["nq"], case["nkv"], case["dim"], case["page"]
    new, kv = lengths(case)
    out, lse, row = [], [], 0
    for i, (n, total) in enumerate(zip(new, kv)):
        pages = s["page_table"][i, :-(-total // page)].long()
        seen = torch.ones((n, total), dtype=torch.bool, device=DEVICE).tril(total - n)
        o, z = [], []
        for h in range(nq):
            k, v = (x[pages, h * nkv // nq].reshape(-1, dim)[:total].double() for x in (s["k_pages"], s["v_pages"]))
            score = (s["q"][row:row + n, h].double() @ k.T / dim ** 0.5).masked_fill(~seen, -math.inf)
            o.append(torch.softmax(score, -1) @ v)
            z.append(torch.logsumexp(score, -1))
        out.append(torch.stack(o, 1))
        lse.append(torch.stack(z, 1))
        row += n
    return torch.cat(out), torch.cat(lse)


def _exact_sample(case, s):
    """The logarithm of the drawn token's share; the token itself is a choice at a boundary and has no 64-bit value."""
    logprob = []
    for i in range(case["rows"]):
        t = float(s["temperature"][i])
        x, index = torch.sort(s["logits"][i].double(), descending=True, stable=True)
        w = torch.softmax(x / t, 0) if t > 0 else (torch.arange(len(x), device=DEVICE) == 0).double()
        kept = torch.ones_like(w, dtype=torch.bool)
        if s["top_k"] is not None and int(s["top_k"][i]) > 0:
            kept[int(s["top_k"][i]):] = False
        if s["top_p"] is not None and float(s["top_p"][i]) < 1:
            share = torch.where(kept, w, 0) / w[kept].sum()
            kept &= share.cumsum(0) - share < float(s["top_p"][i])
        if s["min_p"] is not None and t > 0:
            kept &= w >= float(s["min_p"][i]) * w[0]
        w = torch.zeros_like(w).scatter_(0, index, torch.where(kept, w, 0))
        w /= w.sum()
        c = w.cumsum(0)
        tok = int(torch.searchsorted(c, float(s["u"][i]) * c[-1], right=True).clamp(max=len(w) - 1))
        logprob.append(w[tok].log())
    return None, torch.stack(logprob)
