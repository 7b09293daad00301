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


@pytest.mark.parametrize("V", [60, 9000, 40000])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_largest_and_smallest_temperatures(dtype, V):
    """At 1e20 all logits that are not -inf are alike; at 1e-6 the largest one takes all."""
    g = torch.Generator().manual_seed(1)
    z = torch.randn(3, V, generator=g).to(dtype)
    z[:, 5:30] = -math.inf
    z[:, 4] = 6.0
    t = torch.tensor([0, 4, 7])
    x = T(z.cuda(), requires_grad=True)
    with K.strict_native():
        lp = F.token_log_probs(x, T(t.cuda()), temperature=1e20)
        F.sum(lp).backward()
    want = torch.log(torch.tensor(1.0 / (V - 25)))
    assert bool(((lp._t.cpu()[:2] - want).abs() < 4e-6).all()) and lp._t[2] == -math.inf
    assert bool(torch.isfinite(x.grad._t).all()) and not x.grad._t[0, 5:30].any()
    x = T(z.cuda(), requires_grad=True)
    lp = F.token_log_probs(x, T(t.cuda()), temperature=1e-6)
    F.sum(lp[:2]).backward()
    # (z[0] - 6) / 1e-6, rounded once
    ref = (z[0, 0].double() - 6.0) / 1e-6
    assert abs(float(lp._t[0]) / float(ref) - 1) < 2.0 ** -23 and lp._t[1] == 0 and lp._t[2] == -math.inf
    assert bool(torch.isfinite(x.grad._t).all()) if dtype != torch.float16 else True
