"""Losses on log-probabilities at the edges of what their arguments may be: on the CPU."""
import math

import pytest
import torch

import genesis_b200 as genesis
import genesis_b200.nn.functional as F

T = genesis.Tensor


@pytest.mark.parametrize("dtype", [torch.float32, torch.float64])
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("shape", [(2, 0), (0, 3), (0, 0), (3, 0, 2), (2, 3, 0)])
def test_no_tokens_with_an_advantage_per_sequence(shape, reduction, dtype):
    x = T(torch.zeros(*shape, 7, dtype=dtype), requires_grad=True)
    row = T(torch.zeros(shape))
    loss = F.policy_loss(x, T(torch.zeros(shape, dtype=torch.int64)), row, T(torch.ones(shape[:-1])), row, kl_coef=0.1,
                         reduction=reduction)
    assert tuple(loss.shape) == (shape if reduction == "none" else ()) and not loss._t.any()
    loss.backward(T(torch.ones(loss.shape, dtype=dtype)))
    assert tuple(x.grad.shape) == shape + (7,)
