"""Losses on tokens' log-probabilities: the kernels against the definitions in 64 bits."""
import math

import pytest
import torch

import genesis_b200 as genesis
import genesis_b200.nn.functional as F
import _token_loss_ref as R
from genesis_b200.ops import dispatch as K

pytestmark = pytest.mark.gpu
T = genesis.Tensor
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def make(shape, V, seed=0, dtype=F32, ignored=0.3, std=3.0):
    g = torch.Generator().manual_seed(seed)
    z = (torch.randn(*shape, V, generator=g) * std).to(dtype)
    t = torch.randint(0, V, shape, generator=g)
    t = torch.where(torch.rand(shape, generator=g) < ignored, torch.full_like(t, -100), t)
    return g, z, t


def policy_inputs(g, z, t, per_sequence):
    lp, _ = R.log_probs(z.double(), t)
    delta = 0.3 * torch.randn(t.shape, generator=g).double()
    for border in (math.log(0.8), math.log(1.28)):       # the gradient jumps there: not within the error of lp
        delta = torch.where((delta - border).abs() < 1e-4, delta + 1e-3, delta)
    ref = lp + 0.3 * torch.randn(t.shape, generator=g).double()
    adv = torch.randn(t.shape[:-1] if per_sequence else t.shape, generator=g)
    return (lp - delta).float(), adv, ref.float()


def dev(*xs):
    return [T(x.cuda()) for x in xs]


# log s of a row: the hardware exponential's 2^-22, and arguments of up to 40 log2(e) rounded to 2^-24 of themselves,
# weighted by the terms' probabilities: below 4e-6; (z - m) / T of up to 60 and lp of up to 60, rounded: 4e-6 each
LP_TOL = 1.2e-5

SHAPES = [((1, 1), 1), ((1, 1), 7), ((3, 5), 17), ((9, 40), 64), ((2, 4), 1000), ((2, 3), 1024), ((2, 3), 1025), ((1, 2), 4099),
          ((2, 7), 8192), ((5, 2), 16385), ((2, 2), 50257), ((1, 1), 151936), ((2, 300), 2056), ((0, 3), 5), ((2, 0), 5)]


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("shape,V", SHAPES)
def test_log_probs_and_gradient(shape, V, dtype):
    g, z, t = make(shape, V, 1, dtype)
    temperature = 0.7 if V % 2 else 1.0
    x = T(z.cuda(), requires_grad=True)
    with K.strict_native():
        lp = F.token_log_probs(x, T(t.cuda()), temperature=temperature)
        gy = torch.randn(shape, generator=g)
        lp.backward(T(gy.cuda()))
    r = R.leaf64(z)
    ref, _ = R.log_probs(r, t, temperature)
    assert lp.dtype == genesis.float32
    assert torch.allclose(lp._t.cpu().double(), ref, atol=LP_TOL, rtol=0)
    (ref * gy).sum().backward()
    R.grad_close(x.grad._t, r.grad, gy / temperature)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("view", ["rows", "columns", "step", "transposed", "shifted", "four", "copied"])
def test_layouts(view, dtype):
    """Views whose rows lie on two strides are read in place; others go through a copy."""
    V = {"columns": 1300, "shifted": 1301}.get(view, 1301)
    g, z, _ = make((4, 6), V, 2, dtype)
    full = z.cuda()
    if view == "rows":
        v = full[:, :-1]
    elif view == "columns":
        v = full[..., 3:]
    elif view == "step":
        v = full[:, 1::2]
    elif view == "transposed":
        v = full.transpose(0, 1)
    elif view == "shifted":
        v = torch.empty(full.numel() + 1, dtype=dtype, device="cuda")[1:].view(4, 6, V)
        v.copy_(full)
    elif view == "four":
        v = full.view(2, 2, 6, V)[:, :, 1:]
    else:
        v = full.transpose(1, 2).contiguous().transpose(1, 2)
    t = torch.randint(0, v.shape[-1], v.shape[:-1], generator=g)
    t.view(-1)[::5] = -100
    x = T(v, requires_grad=True)
    lp = F.token_log_probs(x, T(t.cuda().to(torch.int32)))
    gy = torch.randn(t.shape, generator=g)
    lp.backward(T(gy.cuda()))
    r = R.leaf64(v)
    ref, _ = R.log_probs(r, t)
    assert torch.allclose(lp._t.cpu().double(), ref, atol=LP_TOL, rtol=0)
    (ref * gy).sum().backward()
    R.grad_close(x.grad._t, r.grad, gy)
    assert torch.equal(full.cpu(), z)


def test_shifted_view_of_a_graph():
    """The usual shift by one position inside a graph: the gradient reaches the full logits."""
    g, z, t = make((2, 9), 700, 3)
    leaf = T(z.cuda(), requires_grad=True)
    lp = F.token_log_probs((leaf * 2.0)[:, :-1], T(t[:, 1:].cuda()))
    F.sum(lp).backward()
    r = R.leaf64(z)
    R.log_probs((r * 2.0)[:, :-1], t[:, 1:])[0].sum().backward()
    R.grad_close(leaf.grad._t, r.grad, torch.full((2, 9), 2.0))


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("shape,V,per_sequence,kl", [((3, 6), 21, True, 0.1), ((2, 37), 1030, False, 0.0), ((5, 8), 4100, False, 0.05),
                                                     ((2, 3), 50257, True, 0.04), ((7,), 300, False, 0.1), ((1, 1), 9000, True, 0.0)])
def test_policy_loss(shape, V, per_sequence, kl, reduction, dtype):
    g, z, t = make(shape, V, 4, dtype, std=2.0)
    if len(shape) == 1:
        per_sequence = False
    old, adv, ref = policy_inputs(g, z, t, per_sequence)
    x = T(z.cuda(), requires_grad=True)
    tok, o, a, rf = dev(t, old, adv, ref)
    with K.strict_native():
        loss = F.policy_loss(x, tok, o, a, rf if kl else None, clip=0.2, clip_high=0.28, kl_coef=kl, reduction=reduction)
    r = R.leaf64(z)
    each, on = R.policy(r, t, old, adv, ref if kl else None, 0.2, 0.28, kl)
    want = {"mean": each.sum() / on.sum().clamp(min=1), "sum": each.sum(), "none": each}[reduction]
    # a ratio's relative error is that of lp, and the rounding of old (2^-24 of up to 30): 1.5e-5 of A r, of at most 10 here
    assert torch.allclose(loss._t.cpu().double(), want, atol=2e-4 * (on.sum().item() if reduction == "sum" else 1), rtol=1e-5)
    gy = torch.randn(want.shape, generator=g)
    loss.backward(T(gy.cuda()))
    want.backward(gy.double())
    factor = {"mean": gy / on.sum().clamp(min=1), "sum": gy, "none": gy}[reduction].abs()
    R.grad_close(x.grad._t, r.grad, (factor * 10).expand(shape))


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("pairs,length,V", [(1, 1, 5), (3, 5, 19), (2, 33, 1025), (40, 3, 130), (1, 700, 2000), (2, 2, 50257)])
def test_preference_loss(pairs, length, V, reduction, dtype):
    g, z, t = make((2 * pairs, length), V, 5, dtype)
    ref = R.log_probs(z.double(), t)[0].sum(1).float() + 5 * torch.randn(2 * pairs, generator=g)
    x = T(z.cuda(), requires_grad=True)
    tok, rf = dev(t, ref)
    with K.strict_native():
        loss, rewards = F.preference_loss(x, tok, rf, beta=0.3, label_smoothing=0.1, reduction=reduction, return_rewards=True)
    r = R.leaf64(z)
    each, want_rewards = R.preference(r, t, ref, 0.3, 0.1)
    want = {"mean": each.mean(), "sum": each.sum(), "none": each}[reduction]
    # sums of `length` log-probabilities in 64 bits: their errors add up; beta = 0.3
    tol = 0.3 * LP_TOL * length + 1e-5
    assert torch.allclose(rewards._t.cpu().double(), want_rewards, atol=tol)
    assert torch.allclose(loss._t.cpu().double(), want, atol=2 * tol * (pairs if reduction == "sum" else 1), rtol=1e-6)
    assert not rewards.requires_grad
    gy = torch.randn(want.shape, generator=g)
    loss.backward(T(gy.cuda()))
    want.backward(gy.double())
    # the factor beta sigmoid(..) moves by a quarter of beta times the error of h = reward - reward
    factor = (gy.abs() / (pairs if reduction == "mean" else 1)).expand(pairs).repeat(2).unsqueeze(1).expand(t.shape)
    R.grad_close(x.grad._t, r.grad, factor * 0.3 * (1 + tol / 2e-5))


@pytest.mark.parametrize("V", [300, 9000])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_what_does_not_count_reaches_nothing(dtype, V):
    g, z, t = make((2, 4), V, 6, dtype, ignored=0.0)
    t[0, :2] = -100
    old, adv, ref = policy_inputs(g, z, t, False)

    def grad(z, old, adv, ref, t=t):
        x = T(z.cuda(), requires_grad=True)
        tok, o, a, rf = dev(t, old, adv, ref)
        loss = F.policy_loss(x, tok, o, a, rf, kl_coef=0.1)
        loss.backward()
        return loss.item(), x.grad._t

    z2, old2, adv2, ref2 = z.clone(), old.clone(), adv.clone(), ref.clone()
    z2[0, 0] = math.nan
    z2[0, 1] = -math.inf
    old2[0, 0], adv2[0, 0], ref2[0, 1] = math.nan, math.inf, math.nan
    (la, ga), (lb, gb) = grad(z, old, adv, ref), grad(z2, old2, adv2, ref2)
    assert la == lb and torch.equal(ga, gb) and not gb[0, :2].any()
    none = torch.full_like(t, -100)
    lc, gc = grad(z2, old2, adv2, ref2, none)
    assert lc == 0.0 and not gc.any()
    x = T(z2.cuda(), requires_grad=True)
    loss, rewards = F.preference_loss(x, *dev(none, torch.zeros(2)), return_rewards=True)
    loss.backward()
    assert abs(loss.item() - math.log(2)) < 1e-6 and not rewards._t.any() and not x.grad._t.any()


@pytest.mark.parametrize("V", [260, 40000])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_masked_vocabulary_and_extremes(dtype, V):
    """-inf and lowest values: probability 0, gradient 0; whole vectors and whole parts of a row of them; a NaN stays one."""
    g, z, t = make((1, 6), V, 7, dtype, ignored=0.0)
    low = torch.finfo(dtype).min
    z[..., 8:200] = -math.inf
    z[0, 1, :] = -math.inf
    z[0, 1, V - 1] = 2.0
    z[0, 2, : V // 2] = low
    z[0, 3, 220] = math.nan
    z[0, 4, :] = -math.inf
    z[0, 5, 3] = 60000.0                                  # one logit far above all others
    t[0] = torch.tensor([20, V - 1, V - 2, 1, 1, 3])
    x = T(z.cuda(), requires_grad=True)
    lp = F.token_log_probs(x, T(t.cuda()))
    got = lp._t.cpu()
    assert got[0, 0] == -math.inf and got[0, 1] == 0.0 and got[0, 5] == 0.0
    assert math.isnan(got[0, 3]) and math.isnan(got[0, 4])
    want, _ = R.log_probs(z[:, 2].double(), t[:, 2])
    assert torch.allclose(got[:, 2].double(), want, atol=LP_TOL)
    F.sum(lp[:, :3]).backward()
    d = x.grad._t
    assert torch.isfinite(d).all() and not d[0, 0, 8:20].any() and not d[0, 0, 21:200].any() and not d[0, 1].any()
    assert d[0, 0, 20] == 1 and not d[0, 2, : V // 2].any() and not d[0, 3:].any()


@pytest.mark.parametrize("temperature", [0.7, 1.3])
def test_mean_error_at_a_temperature(temperature):
    """0.7 rounded to 32 bits is 1.7e-8 off, which would shift log-probabilities of -30 by 5e-7, all the same way.  What is left:
    the hardware exponential is off by less than 1e-7 on average, and the mean of 8000 roundings of up to 2^-19 (of
    log-probabilities below 64) by 4 * 2^-19 / sqrt(3 * 8000) = 5e-8 at four standard deviations."""
    g, z, t = make((2, 4000), 300, 13, ignored=0.0, std=6.0)
    with genesis.no_grad():
        lp = F.token_log_probs(*dev(z, t), temperature=temperature)
    ref, _ = R.log_probs(z.double(), t, temperature)
    assert -64 < float(ref.min()) < float(ref.mean()) < -12
    assert abs(float((lp._t.cpu().double() - ref).mean())) < 1.5e-7


def test_rewards_of_long_answers():
    """Sums of 1500 log-probabilities of -12.  A row's log-sum is off by 2e-7 at random (39 times that for 1500 of them: 8e-6) and by less
    than 1.5e-8 on average (2.3e-5); nothing is rounded to 32 bits before the difference to the reference's sum, of order one.
    Rounded, every log-probability would be off by up to 2^-21 more."""
    g, z, t = make((4, 1500), 2000, 14, ignored=0.0)
    lp, _ = R.log_probs(z.double(), t)
    ref = (lp.sum(-1) + torch.randn(4, generator=g).double()).float()
    with genesis.no_grad():
        _, rewards = F.preference_loss(*dev(z, t, ref), beta=1.0, return_rewards=True)
    want = lp.sum(-1) - ref.double()
    assert float((rewards._t.cpu().double() - want).abs().max()) < 4e-5 + 2.0 ** -23 * 4


def test_kl_of_a_policy_near_its_reference():
    """lp is off by 4e-6 at most (its rounding at |lp| < 32 2^-19, the row's log-sum 2e-6), ref by its rounding 2e-6, d by
    both, and exp(d) - 1 - d by |d| of it; exp(d) - 1 has 2^-22 of its own; the loss's rounding 2^-23.  A difference of
    numbers near one would be off by 1e-7."""
    g, z, t = make((4, 50), 64, 11, ignored=0.1)
    lp, on = R.log_probs(z.double(), t)
    assert float(lp.abs().max()) < 32
    d = torch.where(torch.rand(t.shape, generator=g) < 0.5, 1.0, -1.0) * 10 ** (-3 + torch.rand(t.shape, generator=g).double())
    ref, old = (lp + d).float(), lp.float()
    loss = F.policy_loss(*dev(z, t, old, torch.zeros(t.shape), ref), kl_coef=0.5, reduction="none")
    r = R.leaf64(z)
    each, _ = R.policy(r, t, old, torch.zeros(t.shape), ref, kl=0.5)
    each = each.detach()
    tol = 0.5 * (d.abs() * 6e-6 + 4e-11 + 2.0 ** -22 * d.abs()) + 2.0 ** -23 * each
    assert bool(((loss._t.cpu().double() - each).abs() <= tol).all())
    assert float(tol.max()) < 4e-8


def test_an_answer_of_probability_zero():
    """Pair 0 rejects one, pair 1 chose one, pair 2 has none."""
    g, z, t = make((6, 3), 40, 12, ignored=0.0)
    z[3, 1, t[3, 1]] = -math.inf
    z[1, 2, t[1, 2]] = -math.inf
    x = T(z.cuda(), requires_grad=True)
    loss, rewards = F.preference_loss(x, *dev(t, torch.zeros(6)), return_rewards=True, reduction="none")
    assert rewards._t[3] == -math.inf and rewards._t[1] == -math.inf and math.isfinite(float(rewards._t[2]))
    assert loss._t[0] == 0 and loss._t[1] == math.inf and 0 < float(loss._t[2]) < 10
    loss.sum().backward()
    gr = x.grad._t
    # the pair that is decided asks for nothing; the gradient of the other's rows is beta (onehot - softmax), all finite
    assert not gr[0].any() and not gr[3].any() and bool(torch.isfinite(gr).all())
    assert abs(float(gr[1, 2, t[1, 2]]) + 0.1) < 1e-6
    smooth = F.preference_loss(x, *dev(t, torch.zeros(6)), label_smoothing=0.1, reduction="none")
    assert smooth._t[0] == math.inf and smooth._t[1] == math.inf


def test_token_outside_the_vocabulary_is_reported():
    from genesis_b200.ops import native
    g, z, t = make((2, 4), 3000, 8, ignored=0.0)
    good, bad = t.clone(), t.clone()
    good[1, 2] = -100
    bad[1, 2] = 3000
    old = torch.zeros(2, 4)
    x = T(z.cuda(), requires_grad=True)
    loss = F.policy_loss(x, *dev(bad, old, old))
    loss.backward()
    torch.cuda.synchronize()
    with pytest.raises(IndexError, match="token"):
        native.check_status()
    y = T(z.cuda(), requires_grad=True)
    F.policy_loss(y, *dev(good, old, old)).backward()
    assert torch.equal(x.grad._t, y.grad._t)


def test_repeats_bit_for_bit_and_on_another_stream():
    g, z, t = make((4, 50), 4096, 9, BF16)
    old, adv, ref = policy_inputs(g, z, t, True)
    tok, o, a, rf = dev(t, old, adv, ref)
    zc = z.cuda()

    def once():
        x = T(zc, requires_grad=True)
        loss = F.policy_loss(x, tok, o, a, rf, kl_coef=0.1)
        loss.backward()
        return loss._t, x.grad._t

    first = once()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = once()
    third = once()
    torch.cuda.synchronize()
    for other in (second, third):
        assert torch.equal(first[0], other[0]) and torch.equal(first[1], other[1])


def test_captured_and_replayed():
    """Forward and backward of all three from one graph, replayed on new inputs."""
    g, z, t = make((4, 20), 2500, 10, BF16)
    old, adv, ref = policy_inputs(g, z, t, True)
    seq = torch.randn(4, generator=g)

    def fn(x, tok, o, a, rf, s):
        outs = []
        for call in (lambda x: F.policy_loss(x, tok, o, a, rf, kl_coef=0.1), lambda x: F.preference_loss(x, tok, s),
                     lambda x: F.sum(F.token_log_probs(x, tok))):
            x = T(x._t, requires_grad=True)
            loss = call(x)
            loss.backward()
            outs += [loss, x.grad]
        return outs

    inputs = dev(z, t, old, adv, ref, seq)
    graphed = genesis.cuda.make_graphed_callable(fn, inputs)
    for seed in (11, 12):
        g, z, t = make((4, 20), 2500, seed, BF16)
        old, adv, ref = policy_inputs(g, z, t, True)
        inputs = dev(z, t, old, adv, ref, seq)
        got = [o._t.clone() for o in graphed(*inputs)]
        for a, b in zip(got, fn(*inputs)):
            assert torch.equal(a, b._t)


def test_retained_graph_and_accumulation():
    g, z, t = make((2, 5), 1500, 13)
    x = T(z.cuda(), requires_grad=True)
    lp = F.token_log_probs(x, T(t.cuda()))
    F.sum(lp).backward()
    once = x.grad._t.clone()
    F.sum(F.token_log_probs(x, T(t.cuda()))).backward()
    assert torch.allclose(x.grad._t, 2 * once)


def test_64_bit_logits_are_computed_in_64_bits():
    g, z, t = make((2, 3), 50, 14, torch.float64)
    lp = F.token_log_probs(T(z.cuda()), T(t.cuda()))
    assert torch.allclose(lp._t.cpu(), R.log_probs(z, t)[0], atol=1e-13)
