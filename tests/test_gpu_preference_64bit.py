"""The loss of paired log ratios where rewards are large and their difference is of order one: the kernels."""
import pytest
import torch

import genesis_b200 as genesis
import genesis_b200.nn.functional as F
import _token_loss_ref as R
from genesis_b200.ops import dispatch as K
from test_cpu_preference_64bit import pairs_of_large_rewards, with_digits_beyond_32_bits

pytestmark = pytest.mark.gpu
T = genesis.Tensor

# a row's log-probability in 64 bits: the hardware exponential's 2^-22 and its argument of up to 16 log2(e) rounded to 2^-24
# of itself, weighted by the terms' probabilities
ROW = 2e-6


def test_difference_of_large_rewards():
    z, t, ref = pairs_of_large_rewards(1)
    x = T(z.cuda(), requires_grad=True)
    with K.strict_native():
        loss = F.preference_loss(x, T(t.cuda()), T(ref.cuda()), beta=1.1, label_smoothing=0.1, reduction="none")
        loss.backward(T(torch.ones(3).cuda()))
    r = R.leaf64(z)
    each, _ = R.preference(r, t, ref, 1.1, 0.1)
    each.sum().backward()
    assert float((loss._t.cpu().double() - each.detach()).abs().max()) < 1.1 * 8 * ROW + 2.0 ** -24 * 20
    assert float((x.grad._t.cpu().double() - r.grad).abs().max()) < 1.1 * (1.1 / 4 * 8 * ROW + 1e-6)


def test_a_reference_in_64_bits_is_not_rounded():
    z, t, ref = pairs_of_large_rewards(2)
    ref = with_digits_beyond_32_bits(ref, 3)
    r = R.leaf64(z)
    each, _ = R.preference(r, t, ref, 1.1, 0.1)
    each.sum().backward()
    for given in (ref.cuda(), torch.stack((ref, ref), 1).cuda()[:, 0]):      # (a strided one is laid out, not rounded)
        x = T(z.cuda(), requires_grad=True)
        with K.strict_native():
            loss = F.preference_loss(x, T(t.cuda()), T(given), beta=1.1, label_smoothing=0.1, reduction="none")
            loss.backward(T(torch.ones(3).cuda()))
        assert float((loss._t.cpu().double() - each.detach()).abs().max()) < 1.1 * 8 * ROW + 2.0 ** -24 * 20
        assert float((x.grad._t.cpu().double() - r.grad).abs().max()) < 1.1 * (1.1 / 4 * 8 * ROW + 1e-6)
