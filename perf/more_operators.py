"""Operators over a cache that is held in 8 bits, or whose requests share a beginning: what each call is given, what it returns, and its plain form.

  append8  q/k RMSNorm, rotary positions and the K/V append of a ragged batch into pages of 8-bit rows
  attn8    causal attention of each request's new tokens over such pages
  prefix   causal attention of requests in groups, each of which begins with the same pages

A batch is ragged: request i has n_i new tokens (rows cu_tokens[i] .. cu_tokens[i+1] of the token-major
arrays) and, with them, kv_len[i] cached positions; position p lives in row p % page of the page
page_table[i, p // page]. New token j of request i is at position kv_len[i] - n_i + j.

A cached row of 8 bits (one position of one K/V head) is E4M3 values and one power of two that they are multiples
of: 2^e, e the least from -15 to 7 with |x| <= 448 * 2^e for the row's largest finite x. What lies beyond (where e
would have to be above 7) is held as +-448 * 2^7, infinities as NaN.

With `own` false `run` computes the operators in elementary torch operations in 32 bits; with `own` true it
calls the package's entry points.
"""

import math
import os
import sys

import torch

own = False

DEVICE = "cuda"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu
EPS = 1e-6
THETA = 5e6
LARGEST, LEAST_E, MOST_E = 448.0, -15, 7  # of E4M3; of a row's exponent


def package():
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "htn-2026_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    from decode_b200 import paged

    return paged


# ------------------------------------------------------------------------------------ cases
def _batch(op, name, batch, chunks, n, kv, page, heads=(32, 8), dim=128, dtype="bf16", norm=True):
    """`batch` requests, the first `chunks` of them with up to n new tokens, the others with one; up to kv positions."""
    case = {"op": op, "batch": batch, "chunks": chunks, "n": n, "kv": kv, "page": page, "nq": heads[0],
            "nkv": heads[1], "dim": dim, "dtype": dtype}
    if op == "append8":
        case["norm"] = norm
    if name:
        case["name"] = name
    return case


def _prefix(name, groups, each, prefix, own_kv, chunks, n, page, heads=(32, 8), dim=128, dtype="bf16"):
    """`groups` groups of `each` requests that begin with up to `prefix` common positions and go on with up to own_kv of their own."""
    case = _batch("prefix", name, groups * each, chunks, n, own_kv, page, heads, dim, dtype)
    return case | {"groups": groups, "prefix": prefix}


def listed():
    return [
        # one user's next token: 32 query and 8 K/V heads of 128, the default model's
        _batch("append8", "append8-1", 1, 0, 1, 1031, 64),
        # a decode step of a full batch
        _batch("append8", "append8-64", 64, 0, 1, 1536, 16),
        # the prompts of 16 users at once (about 14 k tokens)
        _batch("append8", "append8-prompts", 16, 16, 1024, 1024, 64),
        # one user's next token after a chat of about a thousand tokens
        _batch("attn8", "attn8-1", 1, 0, 1, 1031, 64),
        # a decode step of a full batch, 1 to 1.5 k tokens each, in small pages
        _batch("attn8", "attn8-64", 64, 0, 1, 1536, 16),
        # a decode step of 8 users with long documents, for which the cache is held in 8 bits
        _batch("attn8", "attn8-8-long", 8, 0, 1, 40960, 64),
        # what a server runs at a time: 30 users decode while two prompts come in
        _batch("attn8", "attn8-mixed", 32, 2, 251, 2049, 32),
        # a chunk of a long prompt, after 8192 cached tokens
        _batch("attn8", "attn8-chunk", 1, 1, 2048, 10240, 128),
        # FP16, heads of 64, seven query heads to a K/V head: another model's short prompts
        _batch("attn8", "attn8-fp16", 5, 5, 301, 777, 32, heads=(14, 2), dim=64, dtype="fp16"),
        # 64 users of one assistant: a system prompt of 4 k tokens, then chats of their own
        _prefix("prefix-64", 1, 64, 4096, 1000, 0, 1, 64),
        # 4 long documents, 4 answers drawn for each
        _prefix("prefix-documents", 4, 4, 16384, 300, 0, 1, 64),
        # 8 prompts of up to 129 tokens over the same instructions, in FP16
        _prefix("prefix-prompts", 1, 8, 2048, 129, 8, 129, 16, dtype="fp16"),
    ]


def _spread(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.4)))))))


def draw(rng):
    op = rng.choice(["append8", "attn8", "attn8", "prefix"])
    dtype, dim, page = rng.choice(["bf16", "bf16", "fp16"]), rng.choice([64, 128, 128]), rng.choice([16, 32, 64, 128])
    nkv = rng.choice([1, 2, 4, 8])
    heads = (nkv * rng.choice([1, 2, 3, 4, 5, 6, 7, 8]), nkv)
    heads = heads if heads[0] <= 32 else (32, nkv)
    if op == "append8":
        batch = _spread(rng, 1, 64)
        chunks = rng.randint(0, batch)
        n = _spread(rng, 1, max(1, min(2048, 14000 // max(1, chunks))))
        return _batch(op, None, batch, chunks, n, n + _spread(rng, 1, 2048), page, heads, dim, dtype, rng.random() < 0.7)
    if op == "prefix":
        groups, each = _spread(rng, 1, 6), _spread(rng, 1, 32)
        batch = groups * each
        prefix = _spread(rng, 1, min(16384, 260000 // batch))
        chunks = rng.choice([0, 0, batch, rng.randint(0, batch)])
        n = _spread(rng, 1, max(1, min(160, 1024 // max(1, chunks)))) if chunks else 1
        return _prefix(None, groups, each, prefix, n + _spread(rng, 1, 1000), chunks, n, page, heads, dim, dtype)
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


def prefixes(case):
    """Common positions of each group, whole pages, by the case alone."""
    if case["op"] != "prefix":
        return [0] * case["batch"]
    page, most = case["page"], case["prefix"]
    return [(most - g * 4099 % (most // 3 + 1)) // page * page for g in range(case["groups"])]


def lengths(case):
    """New tokens and cached positions (the new ones and the common ones included) of each request, by the case alone."""
    b, n, kv = case["batch"], case["n"], case["kv"]
    new = [max(1, n - i * 37 % (n // 4 + 1)) if i < case["chunks"] else 1 for i in range(b)]
    common, each = prefixes(case), b // case.get("groups", b)
    return new, [common[i // each] + max(new[i], kv - i * 7919 % (kv // 3 + 1)) for i in range(b)]


def work(case):
    new, kv = lengths(case)
    nq, nkv, dim, tokens, b = case["nq"], case["nkv"], case["dim"], sum(new), case["batch"]
    if case["op"] == "append8":
        rows = tokens * nkv * 2  # of the cache
        tables = min(tokens, max(kv)) * dim * 4
        return {"bytes": 2 * tokens * (2 * nq + 2 * nkv) * dim + rows * (dim + 1) + tables + 8 * b + 4 * tokens,
                "flops": tokens * (nq + nkv) * dim * 8 + rows * dim * 2}
    pairs = sum(n * (k - n) + n * (n + 1) // 2 for n, k in zip(new, kv))
    keys, row = sum(kv), 2 * dim + 2 if case["op"] == "attn8" else 4 * dim  # a position of a head, K and V
    if case["op"] == "prefix":  # the common positions count once
        keys -= sum(prefixes(case)) * (b // case["groups"] - 1)
    return {"bytes": 2 * 2 * tokens * nq * dim + 4 * tokens * nq + keys * nkv * row + 4 * keys // case["page"] + 8 * b,
            "flops": 4 * nq * dim * pairs}


# ------------------------------------------------------------------------------------ inputs
def _held(x):
    """Values as a cache of 8 bits holds them: E4M3 codes, and the power of two of each row."""
    size = torch.where(x.isfinite(), x, 0.0).abs().amax(-1, keepdim=True)
    fraction, power = torch.frexp(size)  # size = fraction * 2^power, fraction in [0.5, 1); 448 = 0.875 * 2^9
    e = torch.where(size > 0, power - 9 + (fraction > 0.875).to(power.dtype), LEAST_E).clamp(LEAST_E, MOST_E)
    scaled = torch.ldexp(torch.where(x.isfinite() | x.isnan(), x, math.nan), -e)
    return scaled.clamp(-LARGEST, LARGEST).to(E4M3), torch.ldexp(torch.ones_like(size), e)[..., 0].to(E8M0)


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    new, kv = lengths(case)
    page, nq, nkv, dim, dtype, b = (case[k] for k in ("page", "nq", "nkv", "dim", "dtype", "batch"))
    dtype, common, each = TYPES[dtype], prefixes(case), b // case.get("groups", b)
    shared = [common[i // each] // page for i in range(b)]  # pages that a request has from its group's first
    need = [-(-k // page) for k in kv]
    mine = [need[i] - (shared[i] if i % each else 0) for i in range(b)]
    pages, width = sum(mine) + 3, max(need)
    order = torch.randperm(pages, generator=g, device=DEVICE).to(torch.int32)  # pages come in any order
    start = torch.tensor([0] + mine, device=DEVICE).cumsum(0)[:-1]
    lead = torch.tensor(shared, device=DEVICE)[:, None]
    first = torch.arange(b, device=DEVICE) // each * each  # of each request's group
    at = torch.arange(width, device=DEVICE)[None, :]
    own_at = start[:, None] + at - torch.where((torch.arange(b, device=DEVICE) == first)[:, None], 0, lead)
    table = order[torch.where(at < lead, start[first][:, None] + at, own_at).clamp(max=pages - 1)].contiguous()
    cu = torch.tensor([0] + new, device=DEVICE).cumsum(0).to(torch.int32)
    rand = lambda *shape: torch.randn(shape, generator=g, device=DEVICE, dtype=torch.float32)  # noqa: E731
    s = {"op": case["op"], "case": case, "cu_tokens": cu, "kv_len": torch.tensor(kv, dtype=torch.int32, device=DEVICE),
         "page_table": table, "tokens": sum(new), "n_max": max(new), "kv_max": max(kv)}
    k, v = rand(pages, nkv, page, dim), rand(pages, nkv, page, dim)
    if case["op"] == "prefix":
        s["k_pages"], s["v_pages"] = k.to(dtype), v.to(dtype)
        s["cu_groups"] = torch.arange(0, b + 1, each, device=DEVICE).to(torch.int32)
        s["prefix_len"] = torch.tensor(common, dtype=torch.int32, device=DEVICE)
    else:  # rows of differing size, as a model's positions and heads are
        s["k_pages"], s["k_scale"] = _held(k * (0.5 + rand(pages, nkv, page, 1).abs()))
        s["v_pages"], s["v_scale"] = _held(v * (0.5 + rand(pages, nkv, page, 1).abs()))
    if case["op"] == "append8":
        s["qkv"] = rand(s["tokens"], (nq + 2 * nkv) * dim).to(dtype)
        s["q_out"] = torch.empty((s["tokens"], nq, dim), dtype=dtype, device=DEVICE)
        s["q_norm"], s["k_norm"] = ((1 + 0.2 * rand(dim)).to(dtype) for _ in range(2)) if case["norm"] else (None, None)
        inv = THETA ** (-torch.arange(0, dim, 2, dtype=torch.float64, device=DEVICE) / dim)
        angle = torch.arange(s["kv_max"], dtype=torch.float64, device=DEVICE)[:, None] * inv[None, :]
        s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
        return s
    s["q"] = (2 * rand(s["tokens"], nq, dim)).to(dtype)  # scores of deviation 2 and more: some keys stand out
    s["out"] = torch.empty_like(s["q"])
    s["lse"] = torch.empty((s["tokens"], nq), dtype=torch.float32, device=DEVICE)
    if own:  # the workspace that a serving program makes once
        paged = package()
        if case["op"] == "prefix":
            s["handle"] = paged.PrefixAttention(nq, nkv, dim, DEVICE, max_tokens=s["tokens"], max_requests=b, dtype=dtype)
        else:
            s["handle"] = paged.PagedAttention8(nq, nkv, dim, DEVICE, dtype=dtype)
    return s


# ------------------------------------------------------------------------------------ one pass
def run(s):
    return (_run_own if own else _run_plain)[s["op"]](s)


def _own_append8(s):
    c = s["case"]
    package().rope_append8(s["qkv"], s["cu_tokens"], s["kv_len"], s["page_table"], c["nq"], c["nkv"], s["cos"], s["sin"],
                           s["q_out"], s["k_pages"], s["v_pages"], s["k_scale"], s["v_scale"], q_norm=s["q_norm"],
                           k_norm=s["k_norm"], eps=EPS)
    return s["q_out"], s["k_pages"], s["v_pages"], s["k_scale"], s["v_scale"]


def _own_attn8(s):
    # (n_max: a server knows how many tokens it gave each request)
    s["handle"](s["q"], s["k_pages"], s["v_pages"], s["k_scale"], s["v_scale"], s["cu_tokens"], s["kv_len"], s["page_table"],
                s["out"], lse=s["lse"], max_new=s["n_max"])
    return s["out"], s["lse"]


def _own_prefix(s):
    s["handle"](s["q"], s["k_pages"], s["v_pages"], s["cu_tokens"], s["kv_len"], s["page_table"], s["cu_groups"],
                s["prefix_len"], s["out"], lse=s["lse"])
    return s["out"], s["lse"]


def _positions(s):
    """Request and position of each new token."""
    cu, t = s["cu_tokens"].long(), torch.arange(s["tokens"], device=DEVICE)
    b = torch.searchsorted(cu[1:], t, right=True)
    return b, t - cu[b], s["kv_len"].long()[b] - cu[b + 1] + t


def _plain_append8(s):
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
    byte = lambda t: t.view(torch.uint8)  # noqa: E731
    (kc, ks), (vc, vs) = _held(turn(k)), _held(v)
    for pool, value in (("k_pages", kc), ("v_pages", vc), ("k_scale", ks), ("v_scale", vs)):
        byte(s[pool])[page, :, row] = byte(value)
    return s["q_out"], s["k_pages"], s["v_pages"], s["k_scale"], s["v_scale"]


def _plain_attn(s):
    c = s["case"]
    batch, nq, nkv, dim, n = c["batch"], c["nq"], c["nkv"], c["dim"], s["n_max"]
    b, j, pos = _positions(s)
    q = torch.zeros((batch, n, nq, dim), device=DEVICE)
    q[b, j] = s["q"].float()
    last = torch.full((batch, n), -1, dtype=torch.int64, device=DEVICE)  # the last key that a row sees
    last[b, j] = pos
    table = s["page_table"].long()

    def rows(pool, scale):  # every request's positions, one after the other
        x = pool.view(torch.uint8 if scale is not None else pool.dtype)[table]
        x = x if scale is None else x.view(E4M3).float() * scale.view(torch.uint8)[table].view(E8M0).float()[..., None]
        return x.transpose(1, 2).reshape(batch, nkv, -1, dim).float()

    k, v = rows(s["k_pages"], s.get("k_scale")), rows(s["v_pages"], s.get("v_scale"))
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


_run_own = {"append8": _own_append8, "attn8": _own_attn8, "prefix": _own_prefix}
_run_plain = {"append8": _plain_append8, "attn8": _plain_attn, "prefix": _plain_attn}


# ------------------------------------------------------------------------------------ from the definitions, in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return _exact_append8(case, s) if case["op"] == "append8" else _exact_attn(case, s)


def _exact_append8(case, s):
    """Each pair (x_r, x_{r + dim/2}) of a head is the complex number that its position's angle turns; a cached row is
    divided by its power of two, and not rounded."""
    nq, nkv, dim, page = case["nq"], case["nkv"], case["dim"], case["page"]
    new, kv = lengths(case)
    pools = [s["k_pages"].double(), s["v_pages"].double()]
    scales = [s["k_scale"].float().double(), s["v_scale"].float().double()]
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
        for pool, scale, value in zip(pools, scales, (heads[1], x[:, nq + nkv:])):
            ratio = value.abs().amax(-1) / LARGEST
            two = 2.0 ** ratio.clamp(min=2.0 ** LEAST_E, max=2.0 ** MOST_E).log2().ceil()
            for h in range(nkv):
                pool[where // page, h, where % page] = (value[:, h] / two[:, h, None]).clamp(-LARGEST, LARGEST)
                scale[where // page, h, where % page] = two[:, h]
    return torch.cat(q_out), *pools, *scales


def _exact_attn(case, s):
    nq, nkv, dim, page = case["nq"], case["nkv"], case["dim"], case["page"]
    new, kv = lengths(case)
    out, lse, row = [], [], 0
    for i, (n, total) in enumerate(zip(new, kv)):
        pages = s["page_table"][i, :-(-total // page)].long()
        seen = torch.ones((n, total), dtype=torch.bool, device=DEVICE).tril(total - n)
        o, z, cached = [], [], {}
        for name in ("k", "v"):
            x = s[name + "_pages"].view(torch.uint8 if case["op"] == "attn8" else s["q"].dtype)[pages]
            x = x if case["op"] != "attn8" else x.view(E4M3).float()
            x = x.double()
            if case["op"] == "attn8":
                x *= s[name + "_scale"].view(torch.uint8)[pages].view(E8M0).float().double()[..., None]
            cached[name] = x.transpose(0, 1).reshape(nkv, -1, dim)[:, :total]
        for h in range(nq):
            k, v = cached["k"][h * nkv // nq], cached["v"][h * nkv // nq]
            score = (s["q"][row:row + n, h].double() @ k.T / dim ** 0.5).masked_fill(~seen, -math.inf)
            o.append(torch.softmax(score, -1) @ v)
            z.append(torch.logsumexp(score, -1))
        out.append(torch.stack(o, 1))
        lse.append(torch.stack(z, 1))
        row += n
    return torch.cat(out), torch.cat(lse)
