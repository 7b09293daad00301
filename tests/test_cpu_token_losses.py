"""Losses on tokens' log-probabilities on the CPU: values and gradients against the definitions, differences, refusals."""
import math

import pytest
import torch

import genesis_b200 as genesis
import genesis_b200.nn as nn
import genesis_b200.nn.functional as F
import _token_loss_ref as R

T = genesis.Tensor


def make(shape, V, seed=0, dtype=torch.float32, ignored=0.3):
    g = torch.Generator().manual_seed(seed)
    z = (torch.randn(*shape, V, generator=g) * 2).to(dtype)
    t = torch.randint(0, V, shape, generator=g)
    t = torch.where(torch.rand(shape, generator=g) < ignored, torch.full_like(t, -100), t)
    return g, z, t


def policy_inputs(g, z, t, per_sequence):
    lp, _ = R.log_probs(z.double(), t)
    old = (lp + 0.3 * torch.randn(t.shape, generator=g).double()).float()
    ref = (lp + 0.3 * torch.randn(t.shape, generator=g).double()).float()
    adv = torch.randn(t.shape[:-1] if per_sequence else t.shape, generator=g)
    return old, adv, ref


@pytest.mark.parametrize("temperature", [1.0, 0.7])
@pytest.mark.parametrize("shape,V", [((4,), 7), ((2, 5), 33), ((1, 1), 1), ((2, 3, 2), 12), ((0,), 5), ((), 9)])
def test_token_log_probs(shape, V, temperature):
    g, z, t = make(shape, V, 1)
    x = T(z, requires_grad=True)
    lp = F.token_log_probs(x, T(t), temperature=temperature)
    r = R.leaf64(z)
    ref, on = R.log_probs(r, t, temperature)
    assert lp.dtype == genesis.float32 and lp.shape == shape
    assert torch.allclose(lp._t.double(), ref, atol=1e-5, rtol=0)
    gy = torch.randn(shape, generator=g)
    lp.backward(T(gy))
    (ref * gy).sum().backward()
    R.grad_close(x.grad._t, r.grad, gy / temperature)


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("per_sequence,kl", [(True, 0.1), (False, 0.0), (False, 0.05)])
def test_policy_loss(reduction, per_sequence, kl):
    g, z, t = make((3, 6), 21, 2)
    old, adv, ref = policy_inputs(g, z, t, per_sequence)
    x = T(z, requires_grad=True)
    loss = F.policy_loss(x, T(t), T(old), T(adv), T(ref) if kl else None, clip=0.2, clip_high=0.28, kl_coef=kl,
                         reduction=reduction)
    r = R.leaf64(z)
    each, on = R.policy(r, t, old, adv, ref if kl else None, 0.2, 0.28, kl)
    want = {"mean": each.sum() / on.sum(), "sum": each.sum(), "none": each}[reduction]
    assert torch.allclose(loss._t.double(), want, atol=1e-4)
    gy = torch.randn(want.shape, generator=g)
    loss.backward(T(gy))
    want.backward(gy.double())
    R.grad_close(x.grad._t, r.grad, torch.full(t.shape, 4.0))


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("smoothing", [0.0, 0.1])
def test_preference_loss(reduction, smoothing):
    g, z, t = make((6, 5), 19, 3)
    ref = R.log_probs(z.double(), t)[0].sum(1).float() + torch.randn(6, generator=g)
    x = T(z, requires_grad=True)
    loss, rewards = F.preference_loss(x, T(t), T(ref), beta=0.3, label_smoothing=smoothing, reduction=reduction,
                                      return_rewards=True)
    r = R.leaf64(z)
    each, want_rewards = R.preference(r, t, ref, 0.3, smoothing)
    want = {"mean": each.mean(), "sum": each.sum(), "none": each}[reduction]
    assert torch.allclose(loss._t.double(), want, atol=1e-5)
    assert torch.allclose(rewards._t.double(), want_rewards, atol=1e-5) and not rewards.requires_grad
    gy = torch.randn(want.shape, generator=g)
    loss.backward(T(gy))
    want.backward(gy.double())
    R.grad_close(x.grad._t, r.grad, torch.ones(6, 5))


def test_gradients_against_differences():
    """64-bit logits are computed in 64 bits: central differences of the loss agree with the gradient to h^2 and eps / h."""
    g, z, t = make((2, 3), 6, 4, torch.float64, ignored=0.2)
    old, adv, ref = policy_inputs(g, z, t, False)
    seq = R.log_probs(z, t)[0].sum(1).float()

    def losses(x):
        return [F.policy_loss(x, T(t), T(old), T(adv), T(ref), kl_coef=0.1), F.preference_loss(x, T(t), T(seq), beta=0.5),
                F.sum(F.token_log_probs(x, T(t), temperature=0.8) * T(adv.double()))]

    for k in range(3):
        x = T(z.clone(), requires_grad=True)
        losses(x)[k].backward()
        h = 1e-5
        for at in [(0, 0, 1), (0, 2, 3), (1, 1, 5), (1, 2, 0)]:
            up, down = z.clone(), z.clone()
            up[at] += h
            down[at] -= h
            diff = (losses(T(up))[k]._t - losses(T(down))[k]._t) / (2 * h)
            assert abs(float(diff - x.grad._t[at])) < 1e-8


def test_what_does_not_count_reaches_nothing():
    g, z, t = make((2, 4), 10, 5, ignored=0.0)
    t[0, :2] = -100
    old, adv, ref = policy_inputs(g, z, t, False)
    x = T(z, requires_grad=True)
    F.policy_loss(x, T(t), T(old), T(adv), T(ref), kl_coef=0.1).backward()
    z2, old2, adv2, ref2 = z.clone(), old.clone(), adv.clone(), ref.clone()
    z2[0, 0] = math.nan
    z2[0, 1] = -math.inf
    old2[0, 0], adv2[0, 0], ref2[0, 1] = math.nan, math.inf, math.nan
    y = T(z2, requires_grad=True)
    F.policy_loss(y, T(t), T(old2), T(adv2), T(ref2), kl_coef=0.1).backward()
    assert torch.equal(x.grad._t, y.grad._t) and not x.grad._t[0, :2].any()
    # nothing counts at all
    y = T(z2, requires_grad=True)
    loss = F.policy_loss(y, T(torch.full_like(t, -100)), T(old2), T(adv2))
    loss.backward()
    assert loss.item() == 0.0 and not y.grad._t.any()
    y.grad = None
    loss, rewards = F.preference_loss(y, T(torch.full_like(t, -100)), T(torch.zeros(2)), return_rewards=True)
    loss.backward()
    assert abs(loss.item() - math.log(2)) < 1e-6 and not rewards._t.any() and not y.grad._t.any()


def test_kl_of_a_policy_near_its_reference():
    """lp is off by 3e-6 at most (its rounding at |lp| < 16 1e-6, the row's log-sum 2e-6), d by that, and exp(d) - 1 - d by
    |d| of it; exp(d) - 1 has 2^-22 of its own; the loss's rounding 2^-23.  A difference of numbers near one would be off by 1e-7."""
    g, z, t = make((4, 50), 64, 11, ignored=0.1)
    lp, on = R.log_probs(z.double(), t)
    assert float(lp.abs().max()) < 16
    d = torch.where(torch.rand(t.shape, generator=g) < 0.5, 1.0, -1.0) * 10 ** (-3 + torch.rand(t.shape, generator=g).double())
    ref, old = (lp + d).float(), lp.float()
    loss = F.policy_loss(T(z), T(t), T(old), T(torch.zeros(t.shape)), T(ref), kl_coef=0.5, reduction="none")
    r = R.leaf64(z)
    each, _ = R.policy(r, t, old, torch.zeros(t.shape), ref, kl=0.5)
    each = each.detach()
    tol = 0.5 * (d.abs() * 3e-6 + 1e-11 + 2.0 ** -22 * d.abs()) + 2.0 ** -23 * each
    assert bool(((loss._t.double() - each).abs() <= tol).all())
    assert float(tol.max()) < 3e-8


def test_an_answer_of_probability_zero():
    """Pair 0 rejects one, pair 1 chose one, pair 2 has none."""
    g, z, t = make((6, 3), 40, 12, ignored=0.0)
    z[3, 1, t[3, 1]] = -math.inf
    z[1, 2, t[1, 2]] = -math.inf
    x = T(z, requires_grad=True)
    loss, rewards = F.preference_loss(x, T(t), T(torch.zeros(6)), return_rewards=True, reduction="none")
    assert rewards._t[3] == -math.inf and rewards._t[1] == -math.inf and math.isfinite(float(rewards._t[2]))
    assert loss._t[0] == 0 and loss._t[1] == math.inf and 0 < float(loss._t[2]) < 10
    loss.sum().backward()
    gr = x.grad._t
    # the pair that is decided asks for nothing; the gradient of the other's rows is beta (onehot - softmax), all finite
    assert not gr[0].any() and not gr[3].any() and bool(torch.isfinite(gr).all())
    assert abs(float(gr[1, 2, t[1, 2]]) + 0.1) < 1e-6
    smooth = F.preference_loss(x, T(t), T(torch.zeros(6)), label_smoothing=0.1, reduction="none")
    assert smooth._t[0] == math.inf and smooth._t[1] == math.inf


def test_masked_vocabulary():
    """-inf logits have probability 0 and gradient 0; an answer made of one gives a ratio of 0."""
    g, z, t = make((1, 4), 8, 6, ignored=0.0)
    z[..., 3] = -math.inf
    t[:] = torch.tensor([0, 1, 2, 3])
    x = T(z, requires_grad=True)
    lp = F.token_log_probs(x, T(t))
    assert lp._t[0, 3] == -math.inf and torch.isfinite(lp._t[0, :3]).all()
    loss = F.policy_loss(x, T(t), T(torch.zeros(1, 4)), T(torch.ones(1, 4)), reduction="none")
    assert loss._t[0, 3] == 0
    loss.backward(T(torch.ones(1, 4)))
    assert not x.grad._t[..., 3].any() and torch.isfinite(x.grad._t).all()


def test_a_weight_of_zero_leaves_the_reference_out():
    g, z, t = make((2, 4), 10, 9)
    old, adv, ref = policy_inputs(g, z, t, True)
    a = F.policy_loss(T(z), T(t), T(old), T(adv), T(ref * math.nan), kl_coef=0.0)
    assert a.item() == F.policy_loss(T(z), T(t), T(old), T(adv)).item()


def test_modules_and_autocast():
    g, z, t = make((2, 4), 10, 7)
    old, adv, ref = policy_inputs(g, z, t, True)
    a = nn.PolicyLoss(clip=0.1, kl_coef=0.2)(T(z), T(t), T(old), T(adv), T(ref))
    b = F.policy_loss(T(z), T(t), T(old), T(adv), T(ref), clip=0.1, kl_coef=0.2)
    assert a.item() == b.item()
    with genesis.amp.autocast(dtype=genesis.bfloat16):
        c = nn.PolicyLoss(clip=0.1, kl_coef=0.2)(T(z), T(t), T(old), T(adv), T(ref))
    assert c.item() == b.item()
    s = T(torch.zeros(2))
    assert nn.PreferenceLoss(beta=0.2)(T(z), T(t), s).item() == F.preference_loss(T(z), T(t), s, beta=0.2).item()


def test_refusals():
    g, z, t = make((2, 4), 10, 8, ignored=0.0)
    x, tok, row, seq = T(z), T(t), T(torch.zeros(2, 4)), T(torch.zeros(2))
    for call, error in [
        (lambda: F.token_log_probs(z, tok), TypeError),
        (lambda: F.token_log_probs(tok, tok), TypeError),
        (lambda: F.token_log_probs(x, row), TypeError),
        (lambda: F.token_log_probs(x, T(t > 3)), TypeError),
        (lambda: F.token_log_probs(x, T(t[:1])), ValueError),
        (lambda: F.token_log_probs(T(z[..., :0]), tok), ValueError),
        (lambda: F.token_log_probs(x, tok, temperature=0.0), ValueError),
        (lambda: F.token_log_probs(x, tok, temperature=math.nan), ValueError),
        (lambda: F.token_log_probs(x, tok, ignore_index=None), TypeError),
        (lambda: F.token_log_probs(x, T(t + 10)), IndexError),
        (lambda: F.token_log_probs(x, T(t - 20)), IndexError),
        (lambda: F.policy_loss(x, tok, row, row, reduction="max"), ValueError),
        (lambda: F.policy_loss(x, tok, row, T(torch.zeros(4))), ValueError),
        (lambda: F.policy_loss(x, tok, seq, row), ValueError),
        (lambda: F.policy_loss(x, tok, row, tok), TypeError),
        (lambda: F.policy_loss(x, tok, row, row, kl_coef=0.1), ValueError),
        (lambda: F.policy_loss(x, tok, row, row, clip=-0.1), ValueError),
        (lambda: F.policy_loss(x, tok, row, row, clip=1.5), ValueError),
        (lambda: F.policy_loss(x, tok, row, row, clip_high=math.nan), ValueError),
        (lambda: F.policy_loss(x, tok, T(torch.zeros(2, 4), requires_grad=True), row), ValueError),
        (lambda: F.preference_loss(T(z[0]), T(t[0]), seq), ValueError),
        (lambda: F.preference_loss(T(z[:1]), T(t[:1]), T(torch.zeros(1))), ValueError),
        (lambda: F.preference_loss(x, tok, row), ValueError),
        (lambda: F.preference_loss(x, tok, seq, beta=-1), ValueError),
        (lambda: F.preference_loss(x, tok, seq, label_smoothing=1.5), ValueError),
    ]:
        with pytest.raises(error):
            call()


@pytest.mark.parametrize("ignore_index", [2 ** 63, -2 ** 63 - 1, 2 ** 64])
def test_an_ignore_index_that_no_token_can_be_is_refused(ignore_index):
    g, z, t = make((2, 4), 10, 8, ignored=0.0)
    with pytest.raises(ValueError):
        F.token_log_probs(T(z), T(t), ignore_index=ignore_index)


def test_row_map():
    """Rows that lie on two strides are read in place."""
    from genesis_b200.ops.native import _row_map
    z = torch.empty(4, 6, 10)
    for v in (z, z[:, 1:], z[:, ::2], z.transpose(0, 1), z[2], z[2, 3], z.view(2, 2, 6, 10), z.view(2, 2, 6, 10)[:, :, :-1],
              z[:1].expand(3, 6, 10), z[..., 1:]):
        inner, so, si = _row_map(v)
        rows = v.reshape(-1, v.shape[-1])
        base = v.storage_offset()
        for r in range(rows.shape[0]):
            at = base + (r // inner) * so + (r % inner) * si
            idx, k = [], r
            for n in reversed(v.shape[:-1]):
                idx.append(k % n)
                k //= n
            want = base + sum(i * s for i, s in zip(reversed(idx), v.stride()[:-1]))
            assert at == want
    assert _row_map(z.transpose(1, 2)) is None
    assert _row_map(torch.empty(3, 4, 5, 6)[::2, ::3, ::2]) is None
