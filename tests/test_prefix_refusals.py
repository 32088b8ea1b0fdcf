"""What the attention over shared beginnings refuses, and with which code (host checks: no GPU)."""

import ctypes

import pytest
import torch

from test_paged_refusals import SHARED, P, Stand, lib  # noqa: F401  (lib: the fixture)


def _args(**kw):
    a = dict(q=P, ldq=4096, dtype=0, tokens=4, nq=32, nkv=8, dim=128, k=P, v=P, pages=9, page=16, ps_page=8 * 16 * 128,
             ps_head=16 * 128, cu=P, kv=P, batch=2, table=P, ld_table=3, max_pages=3, groups=P, prefix=P, n_groups=1, scale=0.1,
             out=P, ldo=4096, lse=P, ld_lse=32, grid=148, scratch=P, bytes=1 << 40, err=None, pdl=0, stream=None)
    assert set(kw) <= set(a)
    return list({**a, **kw}.values())


@pytest.mark.parametrize("change,code", SHARED + [
    ({"q": None}, 1), ({"q": P + 2}, 1), ({"out": None}, 1), ({"out": P + 8}, 1), ({"ldq": 4095}, 1), ({"ldo": 4088}, 1),
    ({"ld_lse": 31}, 1), ({"ps_head": 16 * 128 + 8}, 1), ({"scale": 0.0}, 1), ({"scale": float("nan")}, 1), ({"grid": 0}, 2),
    ({"scratch": None}, 2), ({"bytes": 8}, 2), ({"groups": None}, 1), ({"prefix": None}, 1), ({"n_groups": -1}, 1), ({"n_groups": 3}, 1)])
def test_prefix_refuses(lib, change, code):  # noqa: F811
    assert lib.qd_prefix_attn(*_args(**change)) == code, change
    assert lib.qd_last_error()


def test_nothing_to_do_is_not_an_error(lib):  # noqa: F811
    assert lib.qd_prefix_attn(*_args(tokens=0, q=None, out=None, lse=None)) == 0
    assert lib.qd_prefix_attn(*_args(tokens=0, batch=0, n_groups=0, cu=None, kv=None, table=None, max_pages=0, groups=None, prefix=None)) == 0
    assert lib.qd_prefix_attn(*_args(tokens=0, dim=96)) == 4


def _plan(lib, *args):  # noqa: F811
    grid, nbytes = ctypes.c_int(0), ctypes.c_int64(0)
    rc = lib.qd_prefix_attn_plan(*args, ctypes.byref(grid), ctypes.byref(nbytes))
    return rc, grid.value, nbytes.value


def test_prefix_plan(lib):  # noqa: F811
    rc, grid, small = _plan(lib, 32, 8, 128, 64, 64, 5)
    assert rc == 0 and grid == 5
    rc, _, large = _plan(lib, 32, 8, 128, 2048, 64, 5)
    assert rc == 0 and large - small == (2048 - 64) * (2 * 32 * (128 + 1) * 4 + 8 * 8)
    assert _plan(lib, 32, 8, 128, 1 << 31, 64, 0)[0] == 1 and _plan(lib, 32, 8, 128, -1, 64, 0)[0] == 1
    assert _plan(lib, 32, 8, 128, 64, -1, 0)[0] == 1 and _plan(lib, 32, 7, 128, 64, 64, 0)[0] == 4
    # scratch for fewer tokens, or requests, than a call has
    bytes_for = lambda tokens, requests: _plan(lib, 32, 8, 128, tokens, requests, 148)[2]  # noqa: E731
    assert lib.qd_prefix_attn(*_args(tokens=100, bytes=bytes_for(50, 2))) == 2
    assert lib.qd_prefix_attn(*_args(batch=900, n_groups=900, bytes=bytes_for(4, 2))) == 2
    assert lib.qd_prefix_attn(*_args(tokens=0, batch=2, bytes=bytes_for(0, 2))) == 0


def _stands():
    B, I, F = torch.bfloat16, torch.int32, torch.float32
    return dict(cu_tokens=Stand((3,), I), kv_len=Stand((2,), I), page_table=Stand((2, 4), I), k_pages=Stand((9, 2, 16, 128), B),
                v_pages=Stand((9, 2, 16, 128), B), cu_groups=Stand((2,), I), prefix_len=Stand((1,), I), err=Stand((1,), I),
                q=Stand((5, 4, 128), B), out=Stand((5, 4, 128), B), lse=Stand((5, 4), F), scratch=Stand((1 << 20,), torch.uint8))


def test_wrapper_refuses_other_devices_types_and_shapes(monkeypatch):
    from decode_b200 import lib as L
    from decode_b200 import paged

    handle, calls = paged.PrefixAttention(4, 2, 128, "cpu", 5, 2), []
    monkeypatch.setattr(paged, "_raw_stream", lambda dev: 0)
    monkeypatch.setattr(paged, "_current_device", lambda: 0)
    monkeypatch.setattr(paged.L, "call", lambda name, *a: calls.append((name, len(a))))

    def run(t):
        handle.scratch = t.pop("scratch")
        return handle(**t)

    run(_stands())
    assert calls == [("qd_prefix_attn", len(L.PROTOTYPES["qd_prefix_attn"][1]))]
    for name in _stands():
        for dev in (-1, 1):
            t = _stands()
            t[name].dev = dev
            with pytest.raises(AssertionError):
                run(t)
    for name, shape, dtype in (("cu_groups", (3,), torch.int32), ("cu_groups", (2,), torch.int64), ("prefix_len", (1,), torch.int64),
                               ("q", (5, 4, 128), torch.float16), ("lse", (5, 3), torch.float32)):
        t = _stands()
        t[name] = Stand(shape, dtype)
        with pytest.raises(AssertionError):
            run(t)
    assert len(calls) == 1, "a refused call reached the library"
