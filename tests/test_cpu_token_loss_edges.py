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


def scale(temperature):
    """log2(e) / T as the kernels hold it, a high part rounded down and what is left of it, and the numbers derived from it."""
    import numpy as np
    f32 = np.float32
    with np.errstate(over="ignore", under="ignore", divide="ignore"):
        c = 1.4426950408889634 / temperature
        hi = f32(c)
        if float(hi) >= c:
            hi = np.nextafter(hi, f32(0))
        return hi, f32(c - float(hi)), f32(1.0 / temperature), f32(1.0 / c)


def test_temperatures_that_the_kernels_cannot_hold_are_refused():
    """Above 2.4e38 the slack, T / log2(e) in 32 bits, is infinite, so that a row's maximum would never be taken up and every
    log-probability be infinite.  Over the temperatures that are taken all of these are normal numbers."""
    x, t = T(torch.randn(2, 5)), T(torch.zeros(2, dtype=torch.int64))
    for temperature in (1e39, 1e300, 1e45, 1.1e20):
        with pytest.raises(ValueError):
            F.token_log_probs(x, t, temperature=temperature)
        with pytest.raises(ValueError):
            F.policy_loss(x, t, T(torch.zeros(2)), T(torch.zeros(2)), temperature=temperature)
    hi, lo, inv, slack = scale(1e39)
    assert math.isinf(slack)
    g = torch.Generator().manual_seed(0)
    for temperature in [1e-6, 1.0, 1e20] + [10 ** (26 * float(torch.rand((), generator=g)) - 6) for _ in range(2000)]:
        hi, lo, inv, slack = (float(v) for v in scale(temperature))
        assert min(hi, lo, inv, slack) >= 2.0 ** -126 and math.isfinite(max(hi, lo, inv, slack))
        assert abs(hi + lo - 1.4426950408889634 / temperature) <= 2.0 ** -47 * hi
    F.token_log_probs(x, t, temperature=1e20)


def test_rows_beyond_what_the_kernels_count_are_refused_in_words():
    from genesis_b200.ops import native
    one = torch.zeros(1)
    for shape in ((1, 2 ** 30 + 1), (2, 3, 2 ** 31), (2 ** 28, 4), (2 ** 14, 2 ** 14, 1)):
        with pytest.raises(ValueError, match="2\\^30 logits a row"):
            native.check_token_logits(one.expand(shape))
    for shape in ((1, 2 ** 30), (2 ** 28 - 1, 4), (0, 5), (2, 0, 5)):
        native.check_token_logits(one.expand(shape))


@pytest.mark.parametrize("weight", [math.inf, 1e39, math.nan, -0.1])
def test_weights_that_are_not_finite_in_32_bits_are_refused(weight):
    """0 times infinity would be the loss of tokens that are as likely as the reference's, and of equal answers."""
    x, t, row = T(torch.randn(2, 3, 5)), T(torch.zeros(2, 3, dtype=torch.int64)), T(torch.zeros(2, 3))
    with pytest.raises(ValueError):
        F.policy_loss(x, t, row, row, row, kl_coef=weight)
    with pytest.raises(ValueError):
        F.preference_loss(x, t, T(torch.zeros(2)), beta=weight)
    assert math.isfinite(F.policy_loss(x, t, row, row, clip_high=math.inf).item())
