"""Serving many requests at once: prompts of any lengths come in while others decode, with sampled answers.

`PagedServer` runs an Engine's packed weights over a paged K/V cache (`paged`) and draws tokens with
`sample`. Every step is one ragged forward: one token of each request that is decoding and, within a budget
of tokens, chunks of the prompts that are coming in (no counterpart in the reference, whose batch is fixed
for the whole answer).

    srv = PagedServer(Engine(path), pages=4096)
    a = srv.add([151644, 872, 198], max_new_tokens=64, temperature=0.7, top_p=0.8, top_k=20, seed=1)
    b = srv.add(another_prompt, max_new_tokens=200)            # greedy
    for finished_step in srv.run():                            # {request: token} of every step
        ...
"""

from __future__ import annotations

import random
from dataclasses import dataclass, field

import torch

from . import lib as L
from . import ops, paged
from .sample import sample

BF16 = torch.bfloat16


@dataclass
class Request:
    prompt: list[int]
    max_new_tokens: int
    temperature: float
    top_k: int
    top_p: float
    min_p: float
    rng: random.Random
    u: float = 0.0                     # the number that its next token is drawn with
    cached: int = 0                    # positions in the cache
    pages: list[int] = field(default_factory=list)
    out: list[int] = field(default_factory=list)
    logprobs: list[float] = field(default_factory=list)
    failed: bool = False               # ended because a row of logits had nothing to draw

    def left(self) -> int:
        """Tokens that are not in the cache yet."""
        return len(self.prompt) + len(self.out) - self.cached

    def take(self, n: int) -> list[int]:
        """The first n of them: of the prompt, then of the answer."""
        at, end, p = self.cached, self.cached + n, len(self.prompt)
        return self.prompt[at:end] + self.out[max(at - p, 0):max(end - p, 0)]


class PagedServer:
    """`pages` pages of `page_size` positions for every layer; at most max_tokens tokens a step and
    max_requests requests at a time (others wait)."""

    def __init__(self, eng, pages: int, page_size: int = 64, max_tokens: int = 2048, max_requests: int = 64):
        self.eng, self.page_size, self.max_tokens, self.max_requests = eng, page_size, max_tokens, max_requests
        if min(pages, max_tokens, max_requests) < 1:
            raise ValueError(f"a server of {pages} pages, {max_tokens} tokens a step and {max_requests} requests")
        dev, D, nq, nkv, H = eng.device, eng.head_dim, eng.nq, eng.nkv, eng.hidden
        shape = (eng.n_layers, pages, nkv, page_size, D)
        self.k_pages = torch.zeros(shape, dtype=BF16, device=dev)
        self.v_pages = torch.zeros(shape, dtype=BF16, device=dev)
        self.cos, self.sin = paged.rope_table(pages * page_size, D, eng.theta, dev)
        self.attn = paged.PagedAttention(nq, nkv, D, dev)
        self.free = list(range(pages - 1, -1, -1))
        self.waiting: list[int] = []
        self.active: list[int] = []
        self.requests: dict[int, Request] = {}
        self.err = torch.zeros((1,), dtype=torch.int32, device=dev)
        new = lambda *s: torch.empty(s, dtype=BF16, device=dev)  # noqa: E731
        self.x, self.h, self.qkv = new(max_tokens, H), new(max_tokens, H), new(max_tokens, (nq + 2 * nkv) * D)
        self.q, self.att, self.act = new(max_tokens, nq * D), new(max_tokens, nq * D), new(max_tokens, eng.inter)
        self.vrows = ops.packed_rows(eng.vocab)
        self.logits = new(max_requests, self.vrows)
        self.tok = torch.empty((max_requests,), dtype=torch.int64, device=dev)
        self.logprob = torch.empty((max_requests,), dtype=torch.float32, device=dev)
        self.next_id = 0

    # ------------------------------------------------------------------ requests
    def add(self, prompt, max_new_tokens: int, temperature: float = 0.0, top_k: int = 0, top_p: float = 1.0,
            min_p: float = 0.0, seed: int | None = None) -> int:
        """Queues a request; its number. temperature 0 takes the most likely token. The seed fixes the answer's
        random numbers; without one they are the request number's."""
        prompt = [int(t) for t in prompt]
        if not prompt or max_new_tokens < 1:
            raise ValueError("a request needs a prompt and at least one new token")
        if min(prompt) < 0 or max(prompt) >= self.eng.vocab:
            raise ValueError(f"token ids from {min(prompt)} to {max(prompt)}, the vocabulary has {self.eng.vocab}")
        if not -2 ** 31 <= top_k < 2 ** 31:
            raise ValueError(f"top_k {top_k} does not fit 32 bits")
        need = -(-(len(prompt) + max_new_tokens) // self.page_size)
        if need > self.k_pages.shape[1]:
            raise ValueError(f"request of {len(prompt) + max_new_tokens} positions needs {need} pages, "
                             f"there are {self.k_pages.shape[1]}")
        i, self.next_id = self.next_id, self.next_id + 1
        rng = random.Random(i if seed is None else seed)
        self.requests[i] = Request(prompt, max_new_tokens, temperature, top_k, top_p, min_p, rng, rng.random())
        self.waiting.append(i)
        return i

    def cancel(self, i: int) -> Request:
        """Ends request i wherever it is (waiting, in its prompt, answering, done) and hands it back; its pages are
        free and the server forgets it. For answers that end before max_new_tokens, and for done ones, which are
        kept in `requests` until then."""
        r = self.requests[i]
        if i in self.waiting:
            self.waiting.remove(i)
        elif i in self.active:
            self._end(i)
        return self.requests.pop(i)

    def _admit(self) -> None:
        """A waiting request joins when the pages of its whole answer are free, so no step runs out of them."""
        while self.waiting and len(self.active) < self.max_requests:
            r = self.requests[self.waiting[0]]
            need = -(-(len(r.prompt) + r.max_new_tokens) // self.page_size)
            if need > len(self.free):
                return
            r.pages = [self.free.pop() for _ in range(need)]
            self.active.append(self.waiting.pop(0))

    def _plan(self) -> list[tuple[int, list[int]]]:
        """(request, tokens of this step): the decoding requests' tokens, then chunks of prompts."""
        left, batch = self.max_tokens, []
        for i in sorted(self.active, key=lambda i: self.requests[i].left() > 1):
            n = min(self.requests[i].left(), left)
            if n:
                batch.append((i, self.requests[i].take(n)))
                left -= n
        return batch

    # ------------------------------------------------------------------ a step
    def step(self) -> dict[int, int]:
        """One forward; {request: drawn token} for those whose last pending token was in it. Token -1: its logits
        had nothing above -inf, and the request has ended (`failed`)."""
        self._admit()
        batch = self._plan()
        if not batch:
            return {}
        dev, reqs = self.eng.device, [self.requests[i] for i, _ in batch]
        cu, width = [0], max(len(r.pages) for r in reqs)
        for _, tokens in batch:
            cu.append(cu[-1] + len(tokens))
        ids = torch.tensor([t for _, tokens in batch for t in tokens], dtype=torch.int64).to(dev)
        kv = [r.cached + len(t) for r, (_, t) in zip(reqs, batch)]
        ints = torch.tensor(cu + kv + [p for r in reqs for p in r.pages + [0] * (width - len(r.pages))],
                            dtype=torch.int32).to(dev)
        n = len(batch)
        logits = self.forward(ids, ints[:n + 1], ints[n + 1:2 * n + 1], ints[2 * n + 1:].view(n, width))
        draw = torch.tensor([[r.temperature, r.top_p, r.min_p, r.u] for r in reqs], dtype=torch.float32)
        t, top_p, min_p, u = draw.t().contiguous().to(dev).unbind(0)
        top_k = torch.tensor([r.top_k for r in reqs], dtype=torch.int32).to(dev)
        sample(logits, u, self.tok[:n], temperature=t, top_k=top_k, top_p=top_p, min_p=min_p,
               logprob=self.logprob[:n], vocab=self.eng.vocab)
        tok, logprob, err = self.tok[:n].tolist(), self.logprob[:n].tolist(), int(self.err.item())
        if err:  # nothing of this step counts: it can be taken again
            self.err.zero_()
            self.attn.reset()
            raise RuntimeError(f"serving step reported a device error: {L.describe_device_error(err)}")
        drawn = {}
        for (i, _), r, length, token, lp in zip(batch, reqs, kv, tok, logprob):
            r.cached = length
            if not r.left():  # the whole prompt (or the last token) is in: this row's draw is its next token
                drawn[i] = token
                r.failed = token < 0
                if not r.failed:
                    r.u = r.rng.random()  # (rows in the middle of a prompt draw too, but use up no number)
                    r.out.append(token)
                    r.logprobs.append(lp)
                if r.failed or len(r.out) == r.max_new_tokens:
                    self._end(i)
        return drawn

    def _end(self, i: int) -> None:
        r = self.requests[i]
        self.free += r.pages
        r.pages = []
        self.active.remove(i)

    def run(self):
        """Steps until every request is done; yields each step's {request: token}."""
        while self.waiting or self.active:
            yield self.step()

    def forward(self, ids, cu_tokens, kv_len, page_table):
        """Logits [requests, vocab rows] after each request's last token of the ragged batch."""
        eng, T = self.eng, ids.shape[0]
        H, I, eps, nq, nkv, D = eng.hidden, eng.inter, eng.eps, eng.nq, eng.nkv, eng.head_dim
        x, h, qkv, q, att, act = (b[:T] for b in (self.x, self.h, self.qkv, self.q, self.att, self.act))
        batch = dict(cu_tokens=cu_tokens, kv_len=kv_len, page_table=page_table, err=self.err)
        RES, SWIGLU = ops.Gemv.RES, ops.Gemv.SWIGLU
        ops.embed(ids, eng.e_packed, eng.vocab, x, self.err, pdl=False)
        for i in range(eng.n_layers):
            kp, vp = self.k_pages[i], self.v_pages[i]
            ops.rmsnorm_rows(x, eng.ln1[i], eps, h)
            ops.tc_gemm(h, eng.w_qkv[i], (nq + 2 * nkv) * D, qkv, err=self.err)
            paged.rope_append(qkv, nq=nq, nkv=nkv, cos=self.cos, sin=self.sin, q_out=q, k_pages=kp, v_pages=vp,
                              q_norm=eng.qn[i], k_norm=eng.kn[i], eps=eps, **batch)
            self.attn(q, kp, vp, out=att, **batch)
            ops.tc_gemm(att, eng.w_o[i], H, x, res=x, epilogue=RES, err=self.err)
            ops.rmsnorm_rows(x, eng.ln2[i], eps, h)
            ops.tc_gemm(h, eng.w_gu[i], 2 * I, act, epilogue=SWIGLU, err=self.err)
            ops.tc_gemm(act, eng.w_down[i], H, x, res=x, epilogue=RES, err=self.err)
        last = x.index_select(0, cu_tokens[1:].long() - 1)
        n = last.shape[0]
        ops.rmsnorm_rows(last, eng.final_norm, eps, h[:n])  # (no more requests than tokens)
        ops.tc_gemm(h[:n], eng.e_packed, self.vrows, self.logits[:n], err=self.err)
        return self.logits[:n]
