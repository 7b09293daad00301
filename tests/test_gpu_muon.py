"""Orthogonalised updates: the tensor-core products against the iteration in 64 bits, and the optimizer's steps."""
import math

import pytest
import torch

import genesis_b200 as genesis
import genesis_b200.nn.functional as F
from genesis_b200.ops import dispatch as K
from test_cpu_muon import reference

pytestmark = pytest.mark.gpu
T = genesis.Tensor


def matrix(*shape, seed=0, kind="normal"):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(*shape, generator=g)
    if kind == "low":       # a few strong directions over a floor of small ones
        x = 0.1 * x + torch.randn(*shape[:-1], 3, generator=g) @ torch.randn(*shape[:-2], 3, shape[-1], generator=g)
    return x


# 2-norm of all errors, absolute.  X = x / |x| has norm 1, and what is rounded in one step grows by up to 3.44 in each
# that follows.  The two fp16 terms of a product hold 22 bits of each operand, the third product (lo lo) is left out: the error
# of A and of B X is at most 3 * 2^-22 of |X|^2 and |B| |X|, with |B| <= 4.8 |A|: 2.3e-6 * 4.8 / 3 in the first step,
# times 3.44^4 = 140: 5e-4; X itself is rounded to 2^-24: 485 * 2^-24 = 3e-5.
TOL = 6e-4

SHAPES = [(1, 1, 1), (1, 1, 40), (1, 40, 1), (1, 16, 16), (1, 64, 64), (1, 63, 65), (1, 128, 128), (1, 129, 127), (3, 100, 300),
          (2, 300, 100), (1, 257, 513), (1, 300, 5000), (1, 5001, 301), (30, 260, 520), (1, 700, 130), (5, 33, 65), (1, 384, 1000), (40, 64, 96), (1, 1000, 1000)]


@pytest.mark.parametrize("kind", ["normal", "low"])
@pytest.mark.parametrize("shape", SHAPES)
def test_orthogonalize(shape, kind):
    x = matrix(*shape, kind=kind)
    with K.strict_native():
        o = genesis.optim.orthogonalize(T(x.cuda()))
    err = torch.linalg.matrix_norm(o._t.cpu().double() - reference(x))
    assert float(err.max()) < TOL, err


def iterated(x, steps=5, coefficients=(3.4445, -4.7750, 2.0315), eps=1e-7):
    """The iteration itself in 64 bits: a decomposition of large matrices takes too long."""
    a, b, c = coefficients
    y = x.double()
    y = y.mT if y.shape[-2] > y.shape[-1] else y
    y = y / (torch.linalg.matrix_norm(y, keepdim=True) + eps)
    for _ in range(steps):
        q = y @ y.mT
        y = a * y + (b * q + c * (q @ q)) @ y
    return y.mT if x.shape[-2] > x.shape[-1] else y


@pytest.mark.parametrize("shape", [(12, 512, 1024), (12, 1000, 500), (2, 2560, 2560), (3, 1100, 2300), (1, 2400, 5100), (9, 896, 896),
                                   (20, 129, 4000), (200, 70, 40)])
def test_large_and_many(shape):
    """Sizes at which tiles are whole, on CTA pairs, or shared by clusters, in each of the three products."""
    x = matrix(*shape, kind="low").cuda()
    with K.strict_native():
        o = genesis.optim.orthogonalize(T(x))
    err = torch.linalg.matrix_norm(o._t.double() - iterated(x))
    assert float(err.max()) < TOL, err


@pytest.mark.parametrize("shape", [(1, 100, 250), (2, 128, 380), (1, 77, 500), (3, 128, 641), (1, 1100, 96), (1, 128, 1500),
                                   (1, 30, 2900), (149, 100, 1300), (160, 24, 4100)])
def test_short_sides(shape):
    """Up to 128 rows: A from one to 33 blocks of the long side by the CTA that goes on with it, or by a launch of its own."""
    x = matrix(*shape, kind="low").cuda()
    with K.strict_native():
        o = genesis.optim.orthogonalize(T(x))
        again = genesis.optim.orthogonalize(T(x))
    err = torch.linalg.matrix_norm(o._t.double() - iterated(x))
    assert float(err.max()) < TOL, err
    assert torch.equal(o._t, again._t)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", [(60, 90), (90, 60), (2, 131, 77), (1, 7)])
def test_types(shape, dtype):
    x = (matrix(*shape) * 1e-2).to(dtype)
    with K.strict_native():
        o = genesis.optim.orthogonalize(T(x.cuda()))
    ref = reference(x)
    assert o._t.dtype == dtype
    # half a step of the type for every element, and the iteration's own error
    tol = torch.finfo(dtype).eps / 2 * ref.abs() + TOL + 2.0 ** -25
    assert ((o._t.cpu().double() - ref).abs() <= tol).all()


@pytest.mark.parametrize("steps,coefficients", [(1, (3.4445, -4.7750, 2.0315)), (2, (1.5, -0.5, 0.0)), (8, (15 / 8, -10 / 8, 3 / 8))])
def test_other_polynomials(steps, coefficients):
    x = matrix(70, 200)
    o = genesis.optim.orthogonalize(T(x.cuda()), steps=steps, coefficients=coefficients)
    ref = reference(x, steps, coefficients)
    assert float(torch.linalg.matrix_norm(o._t.cpu().double() - ref)) < TOL


def test_views_and_degenerate_matrices():
    x = matrix(3, 50, 80).cuda()
    for v in (x.transpose(1, 2), x[:, ::2], x[1], x[..., 3:], x.view(3, 1, 50, 80)):
        o = genesis.optim.orthogonalize(T(v))
        assert o.shape == tuple(v.shape)
        assert float(torch.linalg.matrix_norm(o._t.cpu().double() - reference(v.cpu())).max()) < TOL
    assert not genesis.optim.orthogonalize(T(torch.zeros(2, 30, 40, device="cuda")))._t.any()
    assert genesis.optim.orthogonalize(T(torch.zeros(0, 4, device="cuda")))._t.shape == (0, 4)
    y = x.clone()
    y[0, 3, 3] = math.inf
    y[2, 1, 1] = math.nan
    o = genesis.optim.orthogonalize(T(y))._t
    assert torch.isnan(o[0]).all() and torch.isnan(o[2]).all()
    assert torch.equal(o[1], genesis.optim.orthogonalize(T(x))._t[1])
    for scale in (1e-6, 1e25):           # squares outside the range of 32 bits
        o = genesis.optim.orthogonalize(T(x * scale))._t
        assert float(torch.linalg.matrix_norm(o.cpu().double() - reference((x * scale).cpu())).max()) < TOL


def _model_like(dtype=torch.float32):
    shapes = [(96, 96), (32, 96), (32, 96), (96, 96), (200, 96), (200, 96), (96, 200), (3, 64, 40)]
    ps = [genesis.nn.Parameter(T(matrix(*s, seed=i).cuda() * 0.02)) for i, s in enumerate(shapes)]
    return shapes, ps


def _manual(w, g, u, lr, mu, decay, nesterov):
    u.mul_(mu).add_(g, alpha=1 - mu)
    o = reference(mu * u + (1 - mu) * g if nesterov else u)
    w.mul_(1 - lr * decay).sub_(lr * math.sqrt(max(1.0, w.shape[-2] / w.shape[-1])) * o)


@pytest.mark.parametrize("grad_dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("nesterov", [True, False])
def test_muon_steps(nesterov, grad_dtype):
    shapes, ps = _model_like()
    opt = genesis.optim.Muon(ps, lr=0.1, momentum=0.9, nesterov=nesterov, weight_decay=0.05)
    want = [p._t.cpu().double() for p in ps]
    us = [torch.zeros_like(w) for w in want]
    for step in range(3):
        gs = [matrix(*s, seed=10 * step + i, kind="low").to(grad_dtype) for i, s in enumerate(shapes)]
        for p, g in zip(ps, gs):
            p.grad = T(g.cuda())
        with K.strict_native():
            opt.step()
        for w, g, u in zip(want, gs, us):
            _manual(w, g.double(), u, 0.1, 0.9, 0.05, nesterov)
    for i, (p, w, u) in enumerate(zip(ps, want, us)):
        assert float(torch.linalg.matrix_norm(p._t.cpu().double() - w).max()) < 3 * 0.1 * math.sqrt(3) * TOL + 1e-5
        assert torch.allclose(opt.u[i].cpu().double(), u, atol=1e-6)


def test_repeats_bit_for_bit_and_on_another_stream():
    """Sums have a fixed order: the same call gives the same bits.  A matrix alone may share its contraction among more
    CTAs than in a batch, which is another order, within the tolerance."""
    x = matrix(6, 130, 260).cuda()
    whole = genesis.optim.orthogonalize(T(x))._t
    alone = [genesis.optim.orthogonalize(T(x[i]))._t for i in range(6)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = genesis.optim.orthogonalize(T(x))._t
        single = [genesis.optim.orthogonalize(T(x[i]))._t for i in range(6)]
    torch.cuda.synchronize()
    assert torch.equal(whole, again)
    for i in range(6):
        assert torch.equal(alone[i], single[i])
        assert float(torch.linalg.matrix_norm(whole[i].double() - alone[i].double())) < 2 * TOL


def test_two_streams_at_once_and_a_captured_call():
    """Calls that overlap have workspaces of their own; a captured call replays on new values."""
    xs = [matrix(4, 300, 500, seed=i).cuda() for i in range(4)]
    want = [genesis.optim.orthogonalize(T(x))._t.clone() for x in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    torch.cuda.synchronize()
    got = [None] * 4
    for _ in range(3):
        for i, (x, st) in enumerate(zip(xs, streams)):
            with torch.cuda.stream(st):
                got[i] = genesis.optim.orthogonalize(T(x))._t
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graphed = [genesis.cuda.make_graphed_callable(lambda x: genesis.optim.orthogonalize(x), [T(xs[0])]) for _ in range(2)]
    for i in (1, 2, 3):
        a = graphed[0](T(xs[i]))
        b = graphed[1](T(xs[i - 1]))
        torch.cuda.synchronize()
        assert torch.equal(a._t, want[i]) and torch.equal(b._t, want[i - 1])


def test_a_captured_step_goes_on_with_a_loaded_state():
    w = matrix(3, 60, 90).cuda()
    p = genesis.nn.Parameter(T(w.clone()))
    x = T(torch.randn(5, 60, device="cuda"))
    opt = genesis.optim.Muon([p], lr=0.1)

    def step(x):
        opt.zero_grad()
        loss = (x @ p[0]).sum() + (p * p).sum()
        loss.backward()
        opt.step()
        return loss

    graphed = genesis.cuda.GraphedTrainStep(step, opt, [x])
    graphed(x)
    state = {k: ({i: T(t._t.clone()) for i, t in v.items()} if k == "u" else v) for k, v in opt.state_dict().items()}
    at = p._t.clone()
    graphed(x)
    first = p._t.clone()
    graphed(x)
    opt.load_state_dict(state)
    p._t.copy_(at)
    graphed(x)
    assert torch.equal(p._t, first)


def test_empty_and_zero_gradients():
    ps = [genesis.nn.Parameter(T(matrix(*s).cuda())) for s in ((30, 40), (0, 40), (40, 30), (5, 6))]
    opt = genesis.optim.Muon(ps, lr=0.1, weight_decay=0.5)
    before = [p._t.clone() for p in ps]
    ps[0].grad, ps[1].grad = T(torch.zeros(30, 40).cuda()), T(torch.zeros(0, 40).cuda())
    ps[2].grad = T(matrix(40, 30, seed=1).cuda())
    opt.step()
    assert torch.allclose(ps[0]._t, before[0] * (1 - 0.1 * 0.5)) and torch.equal(ps[3]._t, before[3])
    assert float((ps[2]._t - before[2]).abs().max()) > 1e-3


def test_grad_scaler():
    shapes, ps = _model_like()
    opt = genesis.optim.Muon(ps, lr=0.1)
    scaler = genesis.amp.GradScaler(init_scale=1024.0)
    before = [p._t.clone() for p in ps]
    for p, s in zip(ps, shapes):
        p.grad = T(matrix(*s, seed=3).cuda() * 1024)
    ps[2].grad._t[0, 0] = math.inf
    scaler.step(opt)
    scaler.update()
    assert all(torch.equal(p._t, b) for p, b in zip(ps, before)) and not any(u.any() for u in opt.u.values())
    for p, s in zip(ps, shapes):
        p.grad = T(matrix(*s, seed=3).cuda() * 512)
    scaler.step(opt)
    scaler.update()
    _, qs = _model_like()
    plain = genesis.optim.Muon(qs, lr=0.1)
    for q, s in zip(qs, shapes):
        q.grad = T(matrix(*s, seed=3).cuda())
    plain.step()
    for p, q in zip(ps, qs):
        assert torch.equal(p._t, q._t)                   # (a power of two changes no rounding)


def test_post_training_steps_of_a_model():
    """The operators as they are used together: a reference model scores, the policy's loss trains the matrices with Muon and the
    rest with AdamW; eager and from a graph alike."""
    from genesis_b200.models.transformers import QwenForCausalLM, TransformerConfig
    cfg = TransformerConfig(vocab_size=515, hidden_size=64, intermediate_size=160, num_hidden_layers=2, num_attention_heads=4,
                            num_key_value_heads=2, head_dim=16, max_position_embeddings=32)

    def build():
        genesis.manual_seed(0)
        torch.manual_seed(0)
        model = QwenForCausalLM(cfg).to(genesis.device("cuda"))
        inner = [p for n, p in model.named_parameters() if p._t.dim() == 2 and "layers" in n]
        rest = [p for p in model.parameters() if all(p is not q for q in inner)]
        return model, genesis.optim.Muon(inner, lr=0.02), genesis.optim.AdamW(rest, lr=1e-3)

    g = torch.Generator().manual_seed(1)
    idx = torch.randint(0, 515, (4, 17), generator=g).cuda()
    tok = idx[:, 1:].clone()
    tok[:, :3] = -100
    adv = T(torch.randn(4, generator=g).cuda())
    tok, idx = T(tok), T(idx[:, :-1].contiguous())
    reference_model, _, _ = build()
    with genesis.no_grad():
        old = F.token_log_probs(reference_model(idx), tok)

    def step(model, muon, adam):
        muon.zero_grad()
        adam.zero_grad()
        loss = F.policy_loss(model(idx), tok, old, adv, old, kl_coef=0.05)
        loss.backward()
        muon.step()
        adam.step()
        return loss

    eager = build()
    losses = [step(*eager).item() for _ in range(5)]
    assert all(math.isfinite(x) for x in losses) and len(set(losses)) == 5
    graphed = build()
    run = genesis.cuda.GraphedTrainStep(lambda: step(*graphed), graphed[1:], [], warmup=3)
    again = [run().item() for _ in range(2)]
    # The framework adds up the embedding's gradient in memory in no fixed order, so runs differ in its last bits (eager ones
    # too), and the next step's gradients by some 1e-7 of themselves.  The iteration amplifies that by 485 at most: updates of
    # 2-norm 0.02 * 485 * 1e-7 = 1e-6 for each of the 14 matrices, against gradients of 2-norm 0.5 at most: 7e-6 of the loss.
    assert max(abs(a - b) for a, b in zip(again, losses[3:])) < 1e-5
    assert graphed[1].t == graphed[2].t == 5
    # a learning rate changed between replays counts
    graphed[1].lr, before = 0.0, graphed[1].params[0]._t.clone()
    run()
    assert torch.equal(graphed[1].params[0]._t, before)
    # the gradient of one weight against differences of the loss, along the gradient
    model = build()[0]
    pref = T(torch.zeros(4).cuda())
    F.preference_loss(model(idx), tok, pref, beta=0.5).backward()
    w = model.model.layers[0].mlp.up_proj.weight
    d = w.grad._t / w.grad._t.norm()
    h, vals = 2e-2, []
    start = w._t.clone()
    for sign in (1, -1):
        w.copy_(T(start + sign * h * d))
        with genesis.no_grad():
            vals.append(F.preference_loss(model(idx), tok, pref, beta=0.5).item())
    slope = (vals[0] - vals[1]) / (2 * h)
    # 32-bit losses of order one differ by 2^-23 / h = 6e-6 from rounding, and by h^2 / 6 of the third derivative
    assert abs(slope - float(w.grad._t.norm())) < 0.02 * float(w.grad._t.norm()) + 1e-4
