"""What the paged-cache and sampling entry points refuse, and with which code: host checks, so no GPU is
needed (every call here must return before its launch). The wrappers' own checks of types and shapes are at
the end."""

import ctypes

import pytest
import torch

P = 1 << 20  # stands for a 16-byte aligned device pointer: never dereferenced on the host


@pytest.fixture(scope="module")
def lib():
    from decode_b200 import build, lib as L

    build.build()
    return L.load()


def _append_args(**kw):
    a = dict(qkv=P, ldqkv=48 * 128, dtype=0, tokens=4, nq=32, nkv=8, dim=128, qn=P, kn=P, eps=1e-6, cos=P, sin=P, ld_cs=64,
             n_pos=100, half=64, cu=P, kv=P, batch=2, table=P, ld_table=3, max_pages=3, q_out=P, ldq=4096, k=P, v=P, pages=9,
             page=16, ps_page=8 * 16 * 128, ps_head=16 * 128, err=None, pdl=0, stream=None)
    assert set(kw) <= set(a)
    return list({**a, **kw}.values())


def _attn_args(**kw):
    a = dict(q=P, ldq=4096, dtype=0, tokens=4, nq=32, nkv=8, dim=128, k=P, v=P, pages=9, page=16, ps_page=8 * 16 * 128,
             ps_head=16 * 128, cu=P, kv=P, batch=2, table=P, ld_table=3, max_pages=3, scale=0.1, out=P, ldo=4096, lse=P, ld_lse=32,
             grid=148, scratch=P, bytes=1 << 40, err=None, pdl=0, stream=None)
    assert set(kw) <= set(a)
    return list({**a, **kw}.values())


def _sample_args(**kw):
    a = dict(logits=P, dtype=0, ld=1000, rows=2, vocab=1000, temperature=None, top_k=None, top_p=None, min_p=None, u=P, tok=P,
             logprob=None, pdl=0, stream=None)
    assert set(kw) <= set(a)
    return list({**a, **kw}.values())


SHARED = [({"dtype": 2}, 4), ({"dtype": 9}, 4), ({"dim": 96}, 4), ({"page": 24}, 4), ({"page": 256}, 4), ({"page": 0}, 4),
          ({"nkv": 0}, 1), ({"nq": 30}, 1), ({"nq": 4}, 1), ({"batch": 0}, 1), ({"max_pages": 0}, 1), ({"ld_table": 2}, 1),
          ({"pages": 0}, 1), ({"tokens": -1}, 1), ({"tokens": 1 << 31}, 1), ({"k": None}, 1), ({"v": P + 8}, 1), ({"cu": None}, 1),
          ({"kv": None}, 1), ({"table": None}, 1), ({"ps_head": 1000}, 1), ({"ps_head": 2052}, 1), ({"ps_page": 17}, 1)]


@pytest.mark.parametrize("change,code", SHARED + [
    ({"qkv": None}, 1), ({"qkv": P + 2}, 1), ({"q_out": None}, 1), ({"ldqkv": 48 * 128 - 8}, 1), ({"ldqkv": 48 * 128 + 4}, 1),
    ({"ldq": 4088}, 1), ({"kn": None}, 1), ({"qn": None}, 1), ({"qn": P + 4}, 1), ({"cos": None}, 1), ({"sin": P + 8}, 1),
    ({"half": 4}, 1), ({"half": 12}, 1), ({"half": 72}, 1), ({"ld_cs": 32}, 1), ({"ld_cs": 66}, 1), ({"n_pos": 0}, 1)])
def test_append_refuses(lib, change, code):
    assert lib.qd_paged_rope_append(*_append_args(**change)) == code, change
    assert lib.qd_last_error()


@pytest.mark.parametrize("change,code", SHARED + [
    ({"q": None}, 1), ({"q": P + 2}, 1), ({"out": None}, 1), ({"out": P + 8}, 1), ({"ldq": 4095}, 1), ({"ldo": 4088}, 1),
    ({"ld_lse": 31}, 1), ({"ps_head": 16 * 128 + 8}, 1), ({"scale": 0.0}, 1), ({"scale": float("nan")}, 1), ({"grid": 0}, 2), ({"scratch": None}, 2),
    ({"bytes": 8}, 2)])
def test_attention_refuses(lib, change, code):
    assert lib.qd_paged_attn(*_attn_args(**change)) == code, change
    assert lib.qd_last_error()


@pytest.mark.parametrize("change,code", [
    ({"dtype": 3}, 4), ({"logits": None}, 1), ({"u": None}, 1), ({"tok": None}, 1), ({"rows": -1}, 1), ({"vocab": 0}, 1),
    ({"ld": 999}, 1), ({"vocab": (1 << 18) + 1, "ld": 1 << 19}, 4), ({"logits": P + 1}, 1), ({"dtype": 2, "logits": P + 2}, 1)])
def test_sample_refuses(lib, change, code):
    assert lib.qd_sample(*_sample_args(**change)) == code, change
    assert lib.qd_last_error()


def test_nothing_to_do_is_not_an_error(lib):
    assert lib.qd_paged_rope_append(*_append_args(tokens=0)) == 0
    assert lib.qd_paged_attn(*_attn_args(tokens=0)) == 0
    assert lib.qd_sample(*_sample_args(rows=0)) == 0


def test_attention_plan(lib):
    grid, nbytes = ctypes.c_int(0), ctypes.c_int64(0)
    assert lib.qd_paged_attn_plan(32, 8, 128, 5, ctypes.byref(grid), ctypes.byref(nbytes)) == 0
    assert grid.value == 5 and nbytes.value > 0
    assert lib.qd_paged_attn_plan(32, 7, 128, 0, ctypes.byref(grid), ctypes.byref(nbytes)) == 4
    assert lib.qd_paged_attn_plan(32, 8, 80, 0, ctypes.byref(grid), ctypes.byref(nbytes)) == 4
    assert lib.qd_paged_attn_plan(32, 8, 128, 0, None, ctypes.byref(nbytes)) == 1


def test_wrappers_refuse_cpu_tensors_and_wrong_types():
    from decode_b200 import paged, sample

    k, v = paged.new_pools(3, 2, 16, 128, "cpu")
    cu, kv, table = torch.tensor([0, 1], dtype=torch.int32), torch.tensor([1], dtype=torch.int32), torch.zeros((1, 1), dtype=torch.int32)
    cos, sin = paged.rope_table(4, 128, 1e4, "cpu")
    qkv, q = torch.zeros((1, 8 * 128), dtype=torch.bfloat16), torch.zeros((1, 4, 128), dtype=torch.bfloat16)
    with pytest.raises(AssertionError):
        paged.rope_append(qkv, cu, kv, table, 4, 2, cos, sin, q, k, v)
    with pytest.raises(AssertionError):
        paged.rope_append(qkv.float(), cu, kv, table, 4, 2, cos, sin, q, k, v)
    with pytest.raises(AssertionError):
        sample.sample(torch.zeros((1, 10)), torch.zeros((1,)), torch.zeros((1,), dtype=torch.int64))
    with pytest.raises(AssertionError):
        sample.sample(torch.zeros((1, 10), dtype=torch.float64), torch.zeros((1,)), torch.zeros((1,), dtype=torch.int64))


def test_rope_table_is_the_angles_in_64_bits():
    from decode_b200 import paged

    cos, sin = paged.rope_table(70000, 128, 5e6, "cpu")
    assert cos.shape == (70000, 64) and cos.dtype == torch.float32
    p, r = 69999, 3
    angle = p * 5e6 ** (-2 * r / 128)
    import math

    assert abs(float(cos[p, r]) - math.cos(angle)) < 1e-7 and abs(float(sin[p, r]) - math.sin(angle)) < 1e-7


# ------------------------------------------------------------------------------------ devices
class Stand:
    """Stands for a tensor on GPU `dev` (-1: the host): what the wrappers ask one for, without a GPU."""

    def __init__(self, shape, dtype, dev=0):
        self.shape, self.dtype, self.dev = torch.Size(shape), dtype, dev

    is_cuda = property(lambda self: self.dev >= 0)
    device = property(lambda self: torch.device("cuda", self.dev) if self.dev >= 0 else torch.device("cpu"))

    def get_device(self):
        return self.dev

    def stride(self):
        out = [1]
        for n in reversed(self.shape[1:]):
            out.append(out[-1] * n)
        return tuple(reversed(out))

    def is_contiguous(self):
        return True

    def numel(self):
        return self.shape.numel()

    def data_ptr(self):
        return P


def _stands():
    B, I, F = torch.bfloat16, torch.int32, torch.float32
    batch = dict(cu_tokens=Stand((3,), I), kv_len=Stand((2,), I), page_table=Stand((2, 4), I), k_pages=Stand((9, 2, 16, 128), B),
                 v_pages=Stand((9, 2, 16, 128), B), err=Stand((1,), I))
    return {"append": dict(batch, qkv=Stand((5, 8 * 128), B), cos=Stand((50, 64), F), sin=Stand((50, 64), F), q_out=Stand((5, 4, 128), B),
                           q_norm=Stand((128,), B), k_norm=Stand((128,), B)),
            "attn": dict(batch, q=Stand((5, 4, 128), B), out=Stand((5, 4, 128), B), lse=Stand((5, 4), F), scratch=Stand((1 << 20,), torch.uint8)),
            "sample": dict(logits=Stand((3, 100), B), u=Stand((3,), F), tok=Stand((3,), torch.int64), temperature=Stand((3,), F),
                           top_k=Stand((3,), I), top_p=Stand((3,), F), min_p=Stand((3,), F), logprob=Stand((3,), F))}


@pytest.mark.parametrize("op", ["append", "attn", "sample"])
def test_wrappers_refuse_tensors_on_other_devices(op, monkeypatch):
    """Every tensor of a call is on the current GPU: a host pointer, or one of another GPU, never reaches a kernel."""
    from decode_b200 import paged
    from decode_b200 import sample as S

    handle = paged.PagedAttention(4, 2, 128, "cpu")
    calls = []
    current = [0]
    for m in (paged, S):
        monkeypatch.setattr(m, "_raw_stream", lambda dev: 0)
        monkeypatch.setattr(m, "_current_device", lambda: current[0], raising=False)
    monkeypatch.setattr(paged.L, "call", lambda name, *a: calls.append(name))

    def run(t):
        if op == "append":
            return paged.rope_append(nq=4, nkv=2, **t)
        if op == "attn":
            handle.scratch = t.pop("scratch")
            return handle(**t)
        return S.sample(**t)

    run(_stands()[op])
    assert len(calls) == 1
    for name in _stands()[op]:
        for dev in (-1, 1):
            t = _stands()[op]
            t[name].dev = dev
            with pytest.raises(AssertionError):
                run(t)
            assert len(calls) == 1, f"{name} on device {dev} reached the kernel"
    current[0] = 1
    with pytest.raises(AssertionError):
        run(_stands()[op])
    assert len(calls) == 1, "a launch goes to the current device"


def test_wrappers_refuse_a_wrong_error_word(monkeypatch):
    from decode_b200 import paged

    monkeypatch.setattr(paged, "_raw_stream", lambda dev: 0)
    monkeypatch.setattr(paged, "_current_device", lambda: 0, raising=False)
    monkeypatch.setattr(paged.L, "call", lambda name, *a: pytest.fail("reached the kernel"))
    for bad in (Stand((0,), torch.int32), Stand((1,), torch.uint8)):
        with pytest.raises(AssertionError):
            paged.rope_append(nq=4, nkv=2, **dict(_stands()["append"], err=bad))


# ------------------------------------------------------------------------------------ nothing to do
def test_empty_calls_may_have_null_arrays(lib):
    """An empty tensor's pointer is null: a step in which no request has a token is not an error."""
    assert lib.qd_paged_rope_append(*_append_args(tokens=0, qkv=None, q_out=None)) == 0
    assert lib.qd_paged_rope_append(*_append_args(tokens=0, qkv=None, q_out=None, batch=0, kv=None, table=None, max_pages=0)) == 0
    assert lib.qd_paged_attn(*_attn_args(tokens=0, q=None, out=None, lse=None)) == 0
    assert lib.qd_paged_attn(*_attn_args(tokens=0, q=None, out=None, lse=None, batch=0, kv=None, table=None, max_pages=0)) == 0
    assert lib.qd_sample(*_sample_args(rows=0, logits=None, u=None, tok=None)) == 0
    # what does not depend on the number of tokens is refused all the same
    for change in ({"dim": 96}, {"page": 24}, {"nkv": 7}, {"batch": -1}, {"max_pages": -1}):
        assert lib.qd_paged_rope_append(*_append_args(tokens=0, **change)) != 0
        assert lib.qd_paged_attn(*_attn_args(tokens=0, **change)) != 0
    assert lib.qd_sample(*_sample_args(rows=0, vocab=0)) == 1


def test_wrappers_take_empty_batches(lib, monkeypatch):
    """No tokens (with and without requests) and no rows, through the wrappers: nothing is launched, so no GPU is
    needed."""
    from decode_b200 import paged
    from decode_b200 import sample as S

    class Empty(Stand):
        def data_ptr(self):
            return P if self.numel() else 0

    for m in (paged, S):
        monkeypatch.setattr(m, "_raw_stream", lambda dev: 0)
        monkeypatch.setattr(m, "_current_device", lambda: 0)
    handle = paged.PagedAttention(4, 2, 128, "cpu")
    handle.scratch = Stand((handle.scratch_bytes,), torch.uint8)
    B, I, F = torch.bfloat16, torch.int32, torch.float32
    for n in (0, 2):
        batch = dict(cu_tokens=Empty((n + 1,), I), kv_len=Empty((n,), I), page_table=Empty((n, 3), I),
                     k_pages=Empty((9, 2, 16, 128), B), v_pages=Empty((9, 2, 16, 128), B))
        paged.rope_append(Empty((0, 1024), B), nq=4, nkv=2, cos=Empty((50, 64), F), sin=Empty((50, 64), F), q_out=Empty((0, 4, 128), B), **batch)
        handle(Empty((0, 512), B), out=Empty((0, 512), B), lse=Empty((0, 4), F), **batch)
    S.sample(Empty((0, 100), B), Empty((0,), F), Empty((0,), torch.int64), top_k=Empty((0,), I))


def test_a_single_row_has_no_row_stride(lib, monkeypatch):
    """One token's row may be a view of any buffer: the stride to a next row, which there is not, is not checked."""
    from decode_b200 import paged

    class View(Stand):
        def stride(self):
            return (self.shape[-1] * self.shape[-2] + 3 if len(self.shape) == 3 else self.shape[-1] + 3,) + super().stride()[1:]

    monkeypatch.setattr(paged, "_raw_stream", lambda dev: 0)
    monkeypatch.setattr(paged, "_current_device", lambda: 0)
    seen = []
    monkeypatch.setattr(paged.L, "call", lambda name, *a: seen.append(a))
    handle = paged.PagedAttention.__new__(paged.PagedAttention)
    handle.nq, handle.nkv, handle.head_dim, handle.dtype, handle.grid, handle.scratch_bytes, handle.scale = 4, 2, 128, torch.bfloat16, 1, 0, 0.1
    handle.scratch = Stand((1,), torch.uint8)
    t = _stands()
    handle(**{**{k: v for k, v in t["attn"].items() if k != "scratch"}, "q": View((1, 4, 128), torch.bfloat16),
              "out": View((1, 512), torch.bfloat16), "lse": Stand((1, 4), torch.float32)})
    assert seen[-1][1] == 512 and seen[-1][21] == 512
    paged.rope_append(nq=4, nkv=2, **{**t["append"], "qkv": View((1, 1024), torch.bfloat16), "q_out": View((1, 4, 128), torch.bfloat16)})
    assert seen[-1][1] == 1024


@pytest.mark.parametrize("change,code", [
    ({"ps_page": 16 * 128}, 1), ({"ps_page": 8 * 16 * 128 - 8}, 1), ({"ps_head": 9 * 16 * 128}, 1),
    ({"ps_page": 16 * 128, "ps_head": 9 * 16 * 128 - 1024}, 1), ({"ps_page": 16 * 128, "ps_head": 1 << 62, "pages": (1 << 31) - 1}, 0),
    ({"ps_page": 16 * 128, "ps_head": 9 * 16 * 128}, 0), ({"ps_page": 2 * 8 * 16 * 128}, 0), ({"ps_page": 8 * 16 * 128, "pages": 1}, 0),
    ({"ps_page": 16 * 128, "nkv": 1, "nq": 4}, 0), ({"ps_page": 1 << 62}, 0)])
def test_pools_whose_rows_overlap_are_refused(lib, change, code):
    """Heads lie inside a page, or pages inside a head; two rows in one place would be written by two tokens at once."""
    for call, args in ((lib.qd_paged_rope_append, _append_args), (lib.qd_paged_attn, _attn_args)):
        for tokens in ((4,) if code else (0,)):  # (an accepted call must not launch here)
            assert call(*args(**{**change, "tokens": tokens})) == code, change
