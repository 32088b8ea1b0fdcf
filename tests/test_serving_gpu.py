"""Serving over the paged cache (decode_b200/serving.py) on a 2-layer Qwen3-4B-shaped synthetic model: the
logits of every step against the CPU oracle, forced to the tokens that were drawn, with the bound that the
engine's own decode paths are held to (4 BF16 ulps at |logit| in [4, 8), twice the reference's own
cached-vs-replay drift)."""

import random

import pytest
import torch

from conftest import synth_state
from oracle import qwen3_cpu as Q

pytestmark = pytest.mark.gpu
BOUND = 0.125


@pytest.fixture(scope="module")
def engine():
    import engine as E

    state, cfg = synth_state(2)
    return E.Engine.from_state_dict(state, cfg, "cuda:0")


def _server(engine, **kw):
    from decode_b200.serving import PagedServer

    return PagedServer(engine, **{**dict(pages=64, page_size=16, max_tokens=32, max_requests=4), **kw})


def _logits_of(srv):
    """Runs the server; {request: logits of its drawn tokens}."""
    seen = {}
    while srv.waiting or srv.active:
        before = {i: len(r.out) for i, r in srv.requests.items()}
        srv._admit()
        order = [i for i, _ in srv._plan()]
        drawn = srv.step()
        for row, i in enumerate(order):
            if i in drawn:
                assert len(srv.requests[i].out) == before[i] + 1
                seen.setdefault(i, []).append(srv.logits[row, :srv.eng.vocab].float().cpu())
    return seen


def test_requests_of_many_lengths_follow_the_oracle(engine):
    """Six requests on four places: prompts longer than a step's budget, shorter than a page, joining while
    others decode; greedy."""
    state, cfg = synth_state(2)
    orc = Q.Qwen3Oracle(state, cfg)
    rng = random.Random(4)
    srv = _server(engine)
    prompts = [[rng.randrange(cfg["vocab_size"]) for _ in range(n)] for n in (70, 3, 17, 32, 1, 45)]
    ids = [srv.add(p, new) for p, new in zip(prompts, (4, 7, 2, 3, 5, 2))]
    logits = _logits_of(srv)
    assert len(srv.free) == 64 and not srv.active
    for i, prompt in zip(ids, prompts):
        out = srv.requests[i].out
        _, ref = orc.generate([prompt], len(out), forced=[out])
        for t, token in enumerate(out):
            assert Q.log_softmax_maxdiff(logits[i][t][None], ref[t]) <= BOUND, (i, t)
            assert Q.token_ok(token, ref[t][0], BOUND), (i, t)
            assert srv.requests[i].logprobs[t] == 0.0


def test_sampled_answers_repeat_and_stay_in_the_kept_set(engine):
    rng = random.Random(6)
    prompts = [[rng.randrange(151936) for _ in range(n)] for n in (20, 33, 5)]
    runs = []
    for _ in range(2):
        srv = _server(engine)
        ids = [srv.add(p, 6, temperature=0.9, top_k=5, top_p=0.9, seed=40 + k) for k, p in enumerate(prompts)]
        logits = _logits_of(srv)
        for i in ids:
            for t, token in enumerate(srv.requests[i].out):
                assert token in torch.sort(logits[i][t], descending=True, stable=True).indices[:5].tolist()
                assert -2 < srv.requests[i].logprobs[t] <= 0
        runs.append([srv.requests[i].out for i in ids])
    assert runs[0] == runs[1]
    srv = _server(engine)
    other = srv.add(prompts[0], 6, temperature=0.9, top_k=5, top_p=0.9, seed=99)
    list(srv.run())
    assert srv.requests[other].out != runs[0][0], "another seed draws other numbers"


def test_requests_wait_for_pages_and_refusals(engine):
    srv = _server(engine, pages=4)  # 3 for the first request, 2 for the second
    first, second = srv.add([5] * 40, 8), srv.add([7] * 20, 8)
    steps = list(srv.run())
    assert [i in s for s in steps for i in (second,)].index(True) >= 9, "the second waits for the first one's pages"
    assert len(srv.requests[first].out) == len(srv.requests[second].out) == 8 and sorted(srv.free) == list(range(4))
    with pytest.raises(ValueError, match="pages"):
        srv.add([1] * 70, 20)
    with pytest.raises(ValueError):
        srv.add([], 3)
    with pytest.raises(ValueError):
        srv.add([1], 0)
