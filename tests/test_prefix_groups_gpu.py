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
