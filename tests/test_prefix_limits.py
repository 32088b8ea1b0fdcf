"""What the attention over shared beginnings refuses beyond tests/test_prefix_refusals.py (host checks: no GPU)."""

import pytest
import torch

from test_paged_refusals import Stand, lib  # noqa: F401  (lib: the fixture)
from test_prefix_refusals import _args, _stands

MANY = (1 << 31) - 1


@pytest.mark.parametrize("change", [
    dict(tokens=MANY, nq=65536, nkv=512, dim=64, ldq=65536 * 64, ldo=65536 * 64, ld_lse=65536, ps_page=512 * 16 * 64, ps_head=16 * 64),
    dict(batch=MANY, n_groups=1), dict(batch=1 << 30, n_groups=1 << 30)])
def test_prefix_refuses_what_is_too_large_before_it_launches(lib, change):  # noqa: F811
    """More warps of the last launch than a grid has, and more rows of work than 32 bits count."""
    assert lib.qd_prefix_attn(*_args(bytes=1 << 62, **change)) == 4
    assert lib.qd_last_error()


def test_wrapper_refuses_lengths_that_are_not_one_a_group(monkeypatch):
    from decode_b200 import paged

    handle, calls = paged.PrefixAttention(4, 2, 128, "cpu", 5, 2), []
    monkeypatch.setattr(paged, "_raw_stream", lambda dev: 0)
    monkeypatch.setattr(paged, "_current_device", lambda: 0)
    monkeypatch.setattr(paged.L, "call", lambda name, *a: calls.append(name))
    for shape in ((1, 2), (1, 3)):  # (a second column would be taken for the next groups' lengths)
        t = _stands()
        t["prefix_len"] = Stand(shape, torch.int32)
        handle.scratch = t.pop("scratch")
        with pytest.raises(AssertionError):
            handle(**t)
    assert not calls
