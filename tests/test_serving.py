"""PagedServer's planning on the CPU: which tokens, numbers and pages each step takes. The forward and the draw are
replaced (a draw here is the row's number), so no GPU is needed."""

import types

import pytest
import torch

VOCAB = 1000


@pytest.fixture()
def server(monkeypatch):
    from decode_b200 import serving

    seen = []  # (u of the rows) of every step

    def draw(logits, u, tok, temperature, top_k, top_p, min_p, logprob, vocab):
        assert vocab == VOCAB and logits.shape[0] == u.shape[0] == tok.shape[0]
        seen.append([round(float(x), 6) for x in u])
        tok.copy_((u * VOCAB).long())
        logprob.zero_()

    monkeypatch.setattr(serving, "sample", draw)

    def make(**kw):
        eng = types.SimpleNamespace(device=torch.device("cpu"), head_dim=64, nq=2, nkv=1, hidden=8, inter=8, n_layers=1, theta=1e4,
                                    vocab=VOCAB, eps=1e-6)
        srv = serving.PagedServer(eng, **{**dict(pages=64, page_size=16, max_tokens=32, max_requests=4), **kw})
        srv.seen, srv.fed = seen, {}

        def forward(ids, cu, kv_len, table):
            srv.fed[len(srv.fed)] = ids.tolist()
            return torch.zeros((cu.shape[0] - 1, VOCAB))

        srv.forward = forward
        return srv

    return make


def _answers(srv):
    list(srv.run())
    return {i: r.out for i, r in srv.requests.items()}


def test_a_seed_gives_one_answer_whatever_the_load(server):
    """The numbers of an answer do not depend on how its prompt was cut into steps, nor on the requests beside it."""
    kw = dict(temperature=1.0, seed=7)
    alone = server(max_tokens=64)
    i = alone.add(range(60), 5, **kw)
    ref = _answers(alone)[i]
    assert len(set(ref)) == 5
    for max_tokens in (7, 16, 59, 60):
        srv = server(max_tokens=max_tokens)
        i = srv.add(range(60), 5, **kw)
        assert _answers(srv)[i] == ref, max_tokens
    srv = server(max_tokens=20)
    others = [srv.add(range(n), 9, temperature=1.0, seed=n) for n in (30, 2)]
    i = srv.add(range(60), 5, **kw)
    got = _answers(srv)
    assert got[i] == ref and got[others[0]] != got[others[1]]


def test_requests_without_a_seed_draw_numbers_of_their_own(server):
    srv = server()
    ids = [srv.add([1, 2, 3], 6, temperature=1.0) for _ in range(4)]
    got = _answers(srv)
    assert len({tuple(got[i]) for i in ids}) == 4
    again = server()
    ids2 = [again.add([1, 2, 3], 6, temperature=1.0) for _ in range(4)]
    assert [_answers(again)[i] for i in ids2] == [got[i] for i in ids], "a server's answers repeat"
    seeded = server()
    zero = [seeded.add([1, 2, 3], 6, temperature=1.0, seed=0) for _ in range(2)]
    got = _answers(seeded)
    assert got[zero[0]] == got[zero[1]]


@pytest.mark.parametrize("bad", [dict(prompt=[1, VOCAB]), dict(prompt=[-1]), dict(prompt=[3, 2 ** 70]), dict(prompt=[]),
                                 dict(max_new_tokens=0), dict(top_k=2 ** 31), dict(top_k=-2 ** 31 - 1)])
def test_add_refuses_what_would_stop_a_step(server, bad):
    srv = server()
    good = srv.add([1, 2], 3)
    with pytest.raises(ValueError):
        srv.add(**{**dict(prompt=[1], max_new_tokens=2), **bad})
    assert len(_answers(srv)[good]) == 3 and sorted(srv.free) == list(range(64)) and list(srv.requests) == [good]


def test_add_takes_any_sequence_of_ids(server):
    srv = server()
    a, b = srv.add(torch.arange(5), 2), srv.add((3, 4), 2, top_k=2 ** 31 - 1)
    assert srv.requests[a].prompt == [0, 1, 2, 3, 4]
    assert {i: len(o) for i, o in _answers(srv).items()} == {a: 2, b: 2}


@pytest.mark.parametrize("bad", [dict(max_tokens=0), dict(max_requests=0), dict(pages=0)])
def test_a_server_that_could_never_step_is_refused(server, bad):
    with pytest.raises(ValueError):
        server(**bad)


def test_a_device_error_stops_one_step_only(server):
    """A flagged step raises; the word is cleared, the attention's scratch made ready, and the step can be taken again."""
    ref = server()
    ids = [ref.add(range(40), 4, temperature=1.0), ref.add([5], 6, temperature=1.0)]
    want = _answers(ref)
    srv = server()
    assert [srv.add(range(40), 4, temperature=1.0), srv.add([5], 6, temperature=1.0)] == ids
    forward, fail = srv.forward, [False, True, False, False, True, False]

    def flagged(*a):
        if fail and fail.pop(0):
            srv.err.fill_(16)
            srv.attn.scratch[:8 * srv.attn.grid] = 1
        return forward(*a)

    srv.forward = flagged
    raised = 0
    while srv.waiting or srv.active:
        try:
            srv.step()
        except RuntimeError as e:
            assert "position" in str(e)
            raised += 1
            assert raised <= 2 and int(srv.err) == 0 and int(srv.attn.scratch.max()) == 0
    assert raised == 2 and {i: r.out for i, r in srv.requests.items()} == want


def test_a_row_with_nothing_to_draw_ends_its_request_only(server, monkeypatch):
    """qd_sample's token -1 (no logit above -inf): that request ends, its pages are free, the others go on."""
    from decode_b200 import serving

    ref = server()
    keep, kw = ref.add([5] * 20, 6, temperature=1.0, seed=3), dict(temperature=1.0, seed=4)
    want = _answers(ref)[keep]
    srv = server()
    assert srv.add([5] * 20, 6, temperature=1.0, seed=3) == keep
    bad = srv.add([9] * 30, 8, **kw)
    inner = serving.sample

    def draw(logits, u, tok, **k):
        inner(logits, u, tok, **k)
        if len(srv.requests[bad].out) == 2 and bad in srv.active:
            tok[[i for i, _ in srv._plan()].index(bad)] = -1

    monkeypatch.setattr(serving, "sample", draw)
    steps = list(srv.run())
    assert srv.requests[keep].out == want and not srv.requests[keep].failed
    assert srv.requests[bad].failed and len(srv.requests[bad].out) == 2 and min(srv.requests[bad].out) >= 0
    assert [s[bad] for s in steps if bad in s][-1] == -1
    assert sorted(srv.free) == list(range(64)) and not srv.active


def test_cancel_frees_and_forgets(server):
    """Waiting, in the middle of its prompt, answering or done: the request is handed back and nothing of it stays."""
    ref = server()
    keep = ref.add([5] * 20, 9, temperature=1.0, seed=3)
    want = _answers(ref)[keep]
    srv = server(max_requests=3, max_tokens=24)
    assert srv.add([5] * 20, 9, temperature=1.0, seed=3) == keep
    done, answering, middle, waiting = srv.add([1], 1), srv.add([2], 9), srv.add([3] * 200, 2), srv.add([4], 2)
    for _ in range(3):
        srv.step()
    assert waiting in srv.waiting and {answering, middle} <= set(srv.active) and done not in srv.active
    assert 0 < srv.requests[middle].cached < 200
    for i, tokens in ((done, 1), (answering, 3), (middle, 0), (waiting, 0)):
        assert len(srv.cancel(i).out) == tokens and i not in srv.requests
        with pytest.raises(KeyError):
            srv.cancel(i)
    list(srv.run())
    assert srv.requests[keep].out == want and sorted(srv.free) == list(range(64))
    srv.cancel(keep)
    assert not srv.requests and not srv.active and not srv.waiting


def test_a_step_copies_the_tokens_it_takes(server):
    """A decode step after a long prompt does not copy the prompt; a chunk copies the chunk."""
    class Watched(list):
        copied = 0

        def __getitem__(self, at):
            got = list.__getitem__(self, at)
            Watched.copied += len(got) if isinstance(at, slice) else 1
            return got

        def __iter__(self):
            Watched.copied += len(self)
            return list.__iter__(self)

        def __add__(self, other):
            Watched.copied += len(self) + len(other)
            return list.__add__(self, other)

    n = 500
    srv = server(max_tokens=100)
    i = srv.add(range(n), 20)
    r = srv.requests[i]
    r.prompt, r.out = Watched(r.prompt), Watched()
    for step in range(25):
        Watched.copied = 0
        srv.step()
        assert Watched.copied <= (100 if step < 5 else 1), (step, Watched.copied)
    assert sum(srv.fed.values(), [])[:n] == list(range(n)) and len(r.out) == 20
    assert sum(srv.fed.values(), [])[n:] == r.out[:19]
