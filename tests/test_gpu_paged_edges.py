"""Calls on a paged cache at the edges of what their documentation allows, on the GPU."""
import pytest
import torch

import genesis_b200 as genesis
import genesis_b200.nn.functional as F
from genesis_b200.ops import native as N

import _paged_ref as R

pytestmark = pytest.mark.gpu


def _bits(t):
    return [x.clone().view(torch.uint8) for x in (t.layer.k, t.layer.v)]


@pytest.mark.parametrize("cache", ["bf16", "e4m3"])
@pytest.mark.parametrize("D", [64, 6])           # a row a group of lanes, and a row a warp
def test_rotation_tables_without_a_position(D, cache):
    """Tables of no rows have no address; a call with them still rotates, finds no position, and writes nothing."""
    t = R.Setup([20, 0, 33], 2, D, cache, 16, "cuda")
    y, none = t.tensor(t.normal(3, 2, 8 * D)), t.tensor(torch.zeros(0, D))
    before = _bits(t)
    N.check_status()
    q = F.paged_qkv_rope(y, none, none, t.layer, t.table, t.lens, 4)
    with pytest.raises(IndexError, match="site=9"):
        N.check_status()
    assert torch.all(q._t == 0) and all(torch.equal(a, b) for a, b in zip(_bits(t), before))
    q = F.paged_qkv_rope(y, none, none, t.layer, t.table, t.ints([0, 0, 0]), 4)
    N.check_status()
    assert torch.all(q._t == 0) and all(torch.equal(a, b) for a, b in zip(_bits(t), before))
