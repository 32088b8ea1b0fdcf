"""Ragged batches over cache pages for the tests, and the paged operators' definitions in 64 bits (CPU)."""

import math

import torch

UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}  # largest relative error of one rounding
TINY = {torch.bfloat16: 0.0, torch.float16: 2.0 ** -25}  # and, below the normal range, largest absolute one


class Batch:
    """Requests given as (new tokens, cached positions with them): tables with the pages in random order and
    junk in the entries past the last needed one, and pools whose unused rows are NaN."""

    def __init__(self, spec, nq, nkv, dim, page, dtype=torch.bfloat16, seed=0, pad_tokens=0, device="cpu", spread=2.0):
        g = torch.Generator().manual_seed(seed)
        self.spec, self.nq, self.nkv, self.dim, self.page, self.dtype = spec, nq, nkv, dim, page, dtype
        need = [-(-kv // page) for _, kv in spec]
        self.pages = sum(need) + 2
        order = torch.randperm(self.pages, generator=g).tolist()
        width = max(max(need), 1) + 1
        self.table = torch.full((len(spec), width), 2 ** 30, dtype=torch.int32)
        self.table[::2] = -7
        for i, n in enumerate(need):
            for p in range(n):
                self.table[i, p] = order.pop()
        self.cu = torch.tensor([0] + [n for n, _ in spec]).cumsum(0).to(torch.int32)
        self.kv_len = torch.tensor([kv for _, kv in spec], dtype=torch.int32)
        self.tokens = int(self.cu[-1]) + pad_tokens
        rand = lambda *s: torch.randn(s, generator=g).to(dtype)  # noqa: E731
        self.q = (spread * torch.randn((self.tokens, nq, dim), generator=g)).to(dtype)
        self.qkv = rand(self.tokens, (nq + 2 * nkv) * dim)
        self.k = [rand(kv, nkv, dim) for _, kv in spec]
        self.v = [rand(kv, nkv, dim) for _, kv in spec]
        self.k_pages = torch.full((self.pages, nkv, page, dim), math.nan, dtype=dtype)
        self.v_pages = self.k_pages.clone()
        for i, (_, kv) in enumerate(spec):
            for p in range(kv):
                at = int(self.table[i, p // page]), slice(None), p % page
                self.k_pages[at], self.v_pages[at] = self.k[i][p], self.v[i][p]
        self.device = device

    def on(self, name):
        return getattr(self, name).to(self.device)

    def rows(self):
        """(request, token row, position) of every new token."""
        for i, (n, kv) in enumerate(self.spec):
            for j in range(n):
                yield i, int(self.cu[i]) + j, kv - n + j


def attention(b: Batch, scale=None):
    """out, lse and the bound of |out - ours| for one rounding of the probabilities to the element type and
    one of the result, in 64 bits."""
    scale = 1 / math.sqrt(b.dim) if scale is None else scale
    out = torch.zeros((b.tokens, b.nq, b.dim), dtype=torch.float64)
    tol, lse = out.clone(), torch.full((b.tokens, b.nq), -math.inf, dtype=torch.float64)
    lse_tol = torch.zeros_like(lse)
    u = UNIT[b.dtype]
    for i, t, pos in b.rows():
        seen = min(pos + 1, b.spec[i][1])
        if seen <= 0:
            continue
        k, v, q = b.k[i][:seen].double(), b.v[i][:seen].double(), b.q[t].double()
        k, v = (x.repeat_interleave(b.nq // b.nkv, 1) for x in (k, v))
        s = torch.einsum("hd,khd->hk", q, k) * scale
        p = torch.softmax(s, -1)
        out[t] = torch.einsum("hk,khd->hd", p, v)
        lse[t] = torch.logsumexp(s, -1)
        # scores in fp32: dim products and sums of relative error 2^-24 each
        ds = b.dim * 2.0 ** -24 * (torch.einsum("hd,khd->hk", q.abs(), k.abs()) * scale).amax(-1) + 2.0 ** -20
        spread = torch.einsum("hk,khd->hd", p, v.abs())
        tol[t] = u * out[t].abs() + (1.01 * u + 2 * ds[:, None]) * spread + seen * 2.0 ** -25 * v.abs().amax()
        lse_tol[t] = 2 * ds + 2.0 ** -21 * lse[t].abs()
    return out, lse, tol, lse_tol


def append(b: Batch, cos, sin, q_norm, k_norm, eps):
    """q_out, the key and value rows by (request, position), and the bounds of q and k for one rounding."""
    nq, nkv, dim, half = b.nq, b.nkv, b.dim, cos.shape[1]
    x = b.qkv.double().view(b.tokens, nq + 2 * nkv, dim)
    u = UNIT[b.dtype]
    q_out, q_tol, keys, values = {}, {}, {}, {}
    for i, t, pos in b.rows():
        parts = []
        for h, w in ((x[t, :nq], q_norm), (x[t, nq:nq + nkv], k_norm)):
            if w is not None:
                h = h / (h.square().mean(-1, keepdim=True) + eps).sqrt() * w.double()
            c, s = cos[pos].double(), sin[pos].double()
            a, z, rest = h[:, :half], h[:, half:2 * half], h[:, 2 * half:]
            y = torch.cat((a * c - z * s, z * c + a * s, rest), -1)
            size = torch.cat((a.abs() + z.abs(), a.abs() + z.abs(), rest.abs()), -1)
            parts.append((y, u * y.abs() + TINY[b.dtype] + 2.0 ** -20 * size))
        q_out[t], q_tol[t] = parts[0]
        keys[i, pos], values[i, pos] = parts[1], b.qkv.view(b.tokens, -1, dim)[t, nq + nkv:]
    return q_out, q_tol, keys, values


def attention_on_gpu(b: Batch, device):
    """`attention` for large batches: the same sums and bounds, a request at a time on the device."""
    scale, u = 1 / math.sqrt(b.dim), UNIT[b.dtype]
    out = torch.zeros((b.tokens, b.nq, b.dim), dtype=torch.float64, device=device)
    tol, lse = out.clone(), torch.full((b.tokens, b.nq), -math.inf, dtype=torch.float64, device=device)
    lse_tol = torch.zeros_like(lse)
    for i, (n, kv) in enumerate(b.spec):
        t = slice(int(b.cu[i]), int(b.cu[i]) + n)
        last = torch.arange(kv - n, kv, device=device)
        dead = torch.arange(kv, device=device)[None, :] > last[:, None]
        for h in range(b.nq):
            g = h // (b.nq // b.nkv)
            q, k, v = b.q[t, h].to(device).double(), b.k[i][:, g].to(device).double(), b.v[i][:, g].to(device).double()
            s = (q @ k.T * scale).masked_fill(dead, -math.inf)
            p = torch.softmax(s, -1)
            out[t, h], lse[t, h] = p @ v, torch.logsumexp(s, -1)
            ds = b.dim * 2.0 ** -24 * (q.abs() @ k.abs().T * scale).amax(-1) + 2.0 ** -20
            tol[t, h] = u * out[t, h].abs() + (1.01 * u + 2 * ds[:, None]) * (p @ v.abs()) + kv * 2.0 ** -25 * v.abs().amax()
            lse_tol[t, h] = 2 * ds + 2.0 ** -21 * lse[t, h].abs()
    return out, lse, tol, lse_tol
