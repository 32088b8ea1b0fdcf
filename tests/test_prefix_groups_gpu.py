"""Groups of the attention over shared beginnings (qd_prefix_attn) in which some requests have nothing to do."""

import pytest
import torch

from test_paged_gpu import _check, _err
from test_prefix_gpu import Groups, _attend

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("empty", [1, 3])
@pytest.mark.parametrize("junk", ["others", "outside"])
def test_prefix_of_a_group_whose_first_requests_have_no_tokens(junk, empty):
    """A slot without new tokens at the head of a group: its table row and its length say nothing (an earlier request's
    pages, or none), and are not read."""
    b = Groups([(512, [(0, 0)] * empty + [(1, 30), (1, 200), (3, 9), (0, 40), (1, 77), (1, 1)]), (256, [(1, 5)] * 8)], 8, 2, 128, 32,
               seed=11 + empty, device=DEV)
    if junk == "others":  # a page of the second group, whose keys are other ones
        b.table[:empty] = b.table[-1, 0].clone()
    else:
        b.table[:empty] = b.pages + 3
    b.kv_len[:empty] = torch.tensor([-9, 7, 2000])[:empty]
    err = _err()
    out, lse = _attend(b, err=err)
    _check(b, out, lse)
    assert int(err.item()) == 0


def test_prefix_of_more_requests_than_threads():
    """More requests than the planning launch has threads, more rows of work than the attention has; groups that share
    among them and behind the last round."""
    few = [(0, [(1, 1 + (7 * i + j) % 19) for j in range(8)]) for i in range(65)]
    groups = few + [(512, [(1, 9 + i) for i in range(12)])] + few + [(640, [(1, 3), (9, 30)] * 6), (0, [(40, 150), (1, 3)])]
    assert sum(len(r) for _, r in groups) > 1024 + 12
    b = Groups(groups, 8, 2, 128, 128, seed=5, device=DEV, pad_tokens=1)
    err = _err()
    out, lse = _attend(b, err=err)
    _check(b, out, lse)
    assert int(err.item()) == 0


def test_prefix_without_any_new_token():
    b = Groups([(128, [(0, 2)] * 3), (0, [(0, 9)])], 8, 2, 128, 32, seed=5, device=DEV, pad_tokens=3)
    err = _err()
    out, lse = _attend(b, err=err)
    assert bool((out == 7).all()) and bool((lse == 7).all()) and int(err.item()) == 0
