"""The loss of paired log ratios where rewards are large and their difference is of order one: on the CPU."""
import torch

import genesis_b200 as genesis
import genesis_b200.nn.functional as F
import _token_loss_ref as R

T = genesis.Tensor


def pairs_of_large_rewards(seed, pairs=3, length=4, V=11):
    """Sums of reference log-probabilities of -18000, a multiple of 4 off for chosen and rejected alike, so that rewards are
    near 18000 beta and their difference is that of the answers themselves."""
    g = torch.Generator().manual_seed(seed)
    z = torch.randn(2 * pairs, length, V, generator=g)
    t = torch.randint(0, V, (2 * pairs, length), generator=g)
    ref = torch.full((2 * pairs,), -18000.0) + 4.0 * torch.arange(pairs).repeat(2)
    return z, t, ref


def test_difference_of_large_rewards():
    """A reward of 1.1 * 18000, rounded to 32 bits, is off by up to 2^-10.  Formed before that, the difference has the errors of
    log-probabilities alone: 8 of them, 1e-6 each (values below 16 rounded to 2^-21, the log-sum's 2^-22), times beta; the
    loss moves by at most that, and is rounded to 2^-24 of itself; the gradient moves by beta / 4 of it."""
    z, t, ref = pairs_of_large_rewards(1)
    x = T(z, requires_grad=True)
    loss = F.preference_loss(x, T(t), T(ref), beta=1.1, label_smoothing=0.1, reduction="none")
    r = R.leaf64(z)
    each, want = R.preference(r, t, ref, 1.1, 0.1)
    w = want.detach()
    assert float(w.abs().min()) > 1.1 * 17900 and float((w[:3] - w[3:]).abs().max()) < 20
    assert float((loss._t.double() - each.detach()).abs().max()) < 1.1 * 8e-6 + 2.0 ** -24 * 20
    loss.backward(T(torch.ones(3)))
    each.sum().backward()
    assert float((x.grad._t.double() - r.grad).abs().max()) < 1.1 * (1.1 / 4 * 8e-6 + 1e-6)


def with_digits_beyond_32_bits(ref, seed):
    return ref.double() + torch.rand(ref.shape, generator=torch.Generator().manual_seed(seed)).double() * 2.0 ** -8


def test_a_reference_in_64_bits_is_not_rounded():
    """Sums near -18000, of which 32 bits hold no more than 2^-10: the loss and the gradient are as near as in the test above."""
    z, t, ref = pairs_of_large_rewards(2)
    ref = with_digits_beyond_32_bits(ref, 3)
    assert float((ref - ref.float().double()).abs().max()) > 4e-4
    x = T(z, requires_grad=True)
    loss = F.preference_loss(x, T(t), T(ref), beta=1.1, label_smoothing=0.1, reduction="none")
    r = R.leaf64(z)
    each, _ = R.preference(r, t, ref, 1.1, 0.1)
    assert float((loss._t.double() - each.detach()).abs().max()) < 1.1 * 8e-6 + 2.0 ** -24 * 20
    loss.backward(T(torch.ones(3)))
    each.sum().backward()
    assert x.grad._t.dtype == torch.float32
    assert float((x.grad._t.double() - r.grad).abs().max()) < 1.1 * (1.1 / 4 * 8e-6 + 1e-6)
