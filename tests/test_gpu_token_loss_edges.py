"""Losses on log-probabilities at the edges of what their arguments may be: the kernels."""
import math

import pytest
import torch

import genesis_b200 as genesis
import genesis_b200.nn.functional as F
from genesis_b200.ops import dispatch as K

pytestmark = pytest.mark.gpu
T = genesis.Tensor


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("shape", [(2, 0), (0, 3), (0, 0), (3, 0, 2), (2, 3, 0)])
def test_no_tokens(shape, reduction):
    x = T(torch.zeros(*shape, 7, device="cuda"), requires_grad=True)
    row, tok = T(torch.zeros(shape, device="cuda")), T(torch.zeros(shape, dtype=torch.int64, device="cuda"))
    with K.strict_native():
        loss = F.policy_loss(x, tok, row, T(torch.ones(shape[:-1], device="cuda")), row, kl_coef=0.1, reduction=reduction)
        assert tuple(loss.shape) == (shape if reduction == "none" else ()) and not loss._t.any()
        loss.backward(T(torch.ones(loss.shape, device="cuda")))
    assert tuple(x.grad.shape) == shape + (7,)


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("answers,length", [(0, 3), (4, 0), (0, 0)])
def test_no_answers_or_empty_ones(answers, length, reduction):
    x = T(torch.zeros(answers, length, 7, device="cuda"), requires_grad=True)
    ref = torch.tensor([0.0, 1.0, 0.0, 1.0], device="cuda")[:answers]
    with K.strict_native():
        loss, rewards = F.preference_loss(x, T(torch.zeros(answers, length, dtype=torch.int64, device="cuda")), T(ref), beta=0.5,
                                          reduction=reduction, return_rewards=True)
        loss.backward(T(torch.ones(loss.shape, device="cuda")))
    assert torch.equal(rewards._t, -0.5 * ref)
    if answers:
        want = math.log(2) * (2 if reduction == "sum" else 1)            # (rewards of each pair are equal)
        assert bool(((loss._t - want).abs() < 1e-6).all())
    else:
        assert not loss._t.any()
    assert tuple(x.grad.shape) == (answers, length, 7)
