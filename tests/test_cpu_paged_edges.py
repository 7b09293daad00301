"""Calls on a paged cache at the edges of what their documentation allows, on the CPU."""
import pytest
import torch

import genesis_b200 as genesis
import genesis_b200.nn.functional as F

import _paged_ref as R


def test_rotation_tables_without_a_position():
    t = R.Setup([20, 0], 2, 8, "fp32")
    y, none = t.tensor(torch.ones(2, 1, 8 * 8)), t.tensor(torch.zeros(0, 8))
    before = R.values(t.layer.k, None)
    with pytest.raises(IndexError, match="rotation tables of 0 positions"):
        F.paged_qkv_rope(y, none, none, t.layer, t.table, t.lens, 4)
    assert torch.equal(R.values(t.layer.k, None).nan_to_num(7e9), before.nan_to_num(7e9))
    q = F.paged_qkv_rope(y, none, none, t.layer, t.table, t.ints([0, 0]), 4)      # no token: nothing to rotate
    assert torch.all(q._t == 0)
