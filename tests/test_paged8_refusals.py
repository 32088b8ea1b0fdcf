"""What the entry points of 8-bit pages refuse, and with which code (host checks: no GPU), and what the wrappers do."""

import ctypes

import pytest
import torch

from test_paged_refusals import SHARED, P, Stand, lib  # noqa: F401  (lib: the fixture)

POOLS = dict(ps_page=8 * 16 * 128, ps_head=16 * 128, ss_page=8 * 16, ss_head=16)


def _append_args(**kw):
    a = dict(qkv=P, ldqkv=48 * 128, dtype=0, tokens=4, nq=32, nkv=8, dim=128, qn=P, kn=P, eps=1e-6, cos=P, sin=P, ld_cs=64,
             n_pos=100, half=64, cu=P, kv=P, batch=2, table=P, ld_table=3, max_pages=3, q_out=P, ldq=4096, k=P, v=P, ks=P, vs=P,
             pages=9, page=16, **POOLS, err=None, pdl=0, stream=None)
    assert set(kw) <= set(a)
    return list({**a, **kw}.values())


def _attn_args(**kw):
    a = dict(q=P, ldq=4096, dtype=0, tokens=4, nq=32, nkv=8, dim=128, k=P, v=P, ks=P, vs=P, pages=9, page=16, **POOLS, cu=P, kv=P,
             batch=2, table=P, ld_table=3, max_pages=3, max_new=0, scale=0.1, out=P, ldo=4096, lse=P, ld_lse=32, grid=148, scratch=P,
             bytes=1 << 40, err=None, pdl=0, stream=None)
    assert set(kw) <= set(a)
    return list({**a, **kw}.values())


SCALES = [({"ks": None}, 1), ({"vs": None}, 1), ({"ks": P + 8}, 1), ({"ss_page": 7 * 16}, 1), ({"ss_head": 8}, 1),
          ({"ss_head": 24, "ss_page": 8 * 24}, 1), ({"ss_page": 8 * 16 + 8}, 1), ({"ps_head": 16 * 128 + 8}, 1), ({"ps_page": 8 * 16 * 128 + 8}, 1),
          ({"ss_page": 16, "ss_head": 8 * 16}, 1)]


@pytest.mark.parametrize("change,code", SHARED + SCALES + [
    ({"qkv": None}, 1), ({"qkv": P + 2}, 1), ({"q_out": None}, 1), ({"ldqkv": 48 * 128 - 8}, 1), ({"ldqkv": 48 * 128 + 4}, 1),
    ({"ldq": 4088}, 1), ({"kn": None}, 1), ({"qn": P + 4}, 1), ({"cos": None}, 1), ({"half": 12}, 1), ({"ld_cs": 32}, 1), ({"n_pos": 0}, 1)])
def test_append8_refuses(lib, change, code):  # noqa: F811
    assert lib.qd_paged_rope_append8(*_append_args(**change)) == code, change
    assert lib.qd_last_error()


@pytest.mark.parametrize("change,code", SHARED + SCALES + [
    ({"q": None}, 1), ({"q": P + 2}, 1), ({"out": None}, 1), ({"out": P + 8}, 1), ({"ldq": 4095}, 1), ({"ldo": 4088}, 1),
    ({"ld_lse": 31}, 1), ({"scale": 0.0}, 1), ({"scale": float("nan")}, 1), ({"grid": 0}, 2), ({"scratch": None}, 2), ({"bytes": 8}, 2)])
def test_attention8_refuses(lib, change, code):  # noqa: F811
    assert lib.qd_paged_attn8(*_attn_args(**change)) == code, change
    assert lib.qd_last_error()


def test_nothing_to_do_is_not_an_error(lib):  # noqa: F811
    for empty in ({}, {"k": None, "v": None, "ks": None, "vs": None, "batch": 0, "kv": None, "table": None, "max_pages": 0}):
        assert lib.qd_paged_rope_append8(*_append_args(tokens=0, qkv=None, q_out=None, **empty)) == 0
        assert lib.qd_paged_attn8(*_attn_args(tokens=0, q=None, out=None, lse=None, **empty)) == 0
    for change in ({"dim": 96}, {"page": 24}, {"ss_head": 8}):
        assert lib.qd_paged_rope_append8(*_append_args(tokens=0, **change)) != 0
        assert lib.qd_paged_attn8(*_attn_args(tokens=0, **change)) != 0


@pytest.mark.parametrize("change", [{"ss_page": 16, "ss_head": 9 * 16}, {"ss_page": 1 << 40}, {"ss_page": 8 * 16, "pages": 1}])
def test_scales_in_other_orders_are_taken(lib, change):  # noqa: F811
    assert lib.qd_paged_attn8(*_attn_args(tokens=0, **change)) == 0


def test_attention8_plan(lib):  # noqa: F811
    grid, nbytes = ctypes.c_int(0), ctypes.c_int64(0)
    assert lib.qd_paged_attn8_plan(32, 8, 128, 5, ctypes.byref(grid), ctypes.byref(nbytes)) == 0
    assert grid.value == 5 and nbytes.value > 0
    assert lib.qd_paged_attn8_plan(32, 7, 128, 0, ctypes.byref(grid), ctypes.byref(nbytes)) == 4
    assert lib.qd_paged_attn8_plan(32, 8, 80, 0, ctypes.byref(grid), ctypes.byref(nbytes)) == 4
    assert lib.qd_paged_attn8_plan(32, 8, 128, 0, None, ctypes.byref(nbytes)) == 1


def _stands():
    B, I, F = torch.bfloat16, torch.int32, torch.float32
    E4, E8 = torch.float8_e4m3fn, torch.float8_e8m0fnu
    batch = dict(cu_tokens=Stand((3,), I), kv_len=Stand((2,), I), page_table=Stand((2, 4), I), k_pages=Stand((9, 2, 16, 128), E4),
                 v_pages=Stand((9, 2, 16, 128), E4), k_scale=Stand((9, 2, 16), E8), v_scale=Stand((9, 2, 16), E8), err=Stand((1,), I))
    return {"append": dict(batch, qkv=Stand((5, 8 * 128), B), cos=Stand((50, 64), F), sin=Stand((50, 64), F), q_out=Stand((5, 4, 128), B),
                           q_norm=Stand((128,), B), k_norm=Stand((128,), B)),
            "attn": dict(batch, q=Stand((5, 4, 128), B), out=Stand((5, 4, 128), B), lse=Stand((5, 4), F), scratch=Stand((1 << 20,), torch.uint8))}


@pytest.fixture
def caller(monkeypatch):
    """run(op, tensors) through the wrappers, and the entry points' calls that reach the library."""
    from decode_b200 import paged

    handle, calls = paged.PagedAttention8(4, 2, 128, "cpu"), []
    monkeypatch.setattr(paged, "_raw_stream", lambda dev: 0)
    monkeypatch.setattr(paged, "_current_device", lambda: 0)
    monkeypatch.setattr(paged.L, "call", lambda name, *a: calls.append((name, len(a))))

    def run(op, t):
        if op == "append":
            return paged.rope_append8(nq=4, nkv=2, **t)
        handle.scratch = t.pop("scratch")
        return handle(**t)

    return run, calls


@pytest.mark.parametrize("op", ["append", "attn"])
def test_wrappers_refuse_other_devices_types_and_shapes(op, caller):
    from decode_b200 import lib as L

    run, calls = caller
    run(op, _stands()[op])
    (name, n), = calls
    assert name == {"append": "qd_paged_rope_append8", "attn": "qd_paged_attn8"}[op] and n == len(L.PROTOTYPES[name][1])
    for name in _stands()[op]:
        for dev in (-1, 1):
            t = _stands()[op]
            t[name].dev = dev
            with pytest.raises(AssertionError):
                run(op, t)
    for name, shape, dtype in (("k_pages", (9, 2, 16, 128), torch.bfloat16), ("k_scale", (9, 2, 16), torch.uint8), ("v_scale", (9, 2, 16), torch.float32),
                               ("k_scale", (9, 2, 32), torch.float8_e8m0fnu), ("v_scale", (8, 2, 16), torch.float8_e8m0fnu)):
        t = _stands()[op]
        t[name] = Stand(shape, dtype)
        with pytest.raises(AssertionError):
            run(op, t)
    assert len(calls) == 1, "a refused call reached the library"


def test_new_pools8_and_what_they_hold():
    from decode_b200 import paged

    k, v, ks, vs = paged.new_pools8(3, 2, 16, 64, "cpu")
    assert k.dtype == v.dtype == torch.float8_e4m3fn and ks.dtype == vs.dtype == torch.float8_e8m0fnu
    assert k.shape == (3, 2, 16, 64) and vs.shape == (3, 2, 16)
    assert bool((paged.held_values(k, ks) == 0).all())
    k.view(torch.uint8)[0, 0, 0, 0], ks.view(torch.uint8)[0, 0, 0] = 0x7e, 134
    k.view(torch.uint8)[0, 0, 1, 0], ks.view(torch.uint8)[0, 0, 1] = 0x01, 112
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        x = paged.held_values(k, ks, dtype)
        assert x.dtype == dtype and float(x[0, 0, 0, 0]) == 57344.0 and float(x[0, 0, 1, 0]) == 2.0 ** -24


def test_max_new_does_not_wrap(caller, monkeypatch):
    """A bound larger than 32 bits is no bound, and not a small one."""
    from decode_b200 import paged

    run, _ = caller
    seen = []
    monkeypatch.setattr(paged.L, "call", lambda name, *a: seen.append(a))
    for given in (None, 0, 1, 5, 2 ** 32 + 1):
        t = _stands()["attn"]
        t["max_new"] = given
        run("attn", t)
    assert [a[23] for a in seen] == [0, 0, 1, 5, 5], "never more than the call's tokens"
