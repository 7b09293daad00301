"""Orthogonalised updates on the CPU: the iteration against its action on singular values, the optimizer, refusals."""
import math

import pytest
import torch

import genesis_b200 as genesis
from genesis_b200.optim.muon import COEFFICIENTS, _program

T = genesis.Tensor


def reference(x, steps=5, coefficients=COEFFICIENTS, eps=1e-7):
    """Every singular value s of x / (|x| + eps) goes to a s + b s^3 + c s^5, `steps` times; in 64 bits."""
    a, b, c = coefficients
    U, s, V = torch.linalg.svd(x.double(), full_matrices=False)
    s = s / (s.square().sum(-1, keepdim=True).sqrt() + eps)
    for _ in range(steps):
        s = a * s + b * s ** 3 + c * s ** 5
    return (U * s.unsqueeze(-2)) @ V


def matrix(*shape, seed=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed))


@pytest.mark.parametrize("shape", [(1, 1), (1, 9), (7, 1), (5, 8), (8, 5), (16, 16), (3, 6, 10), (2, 2, 9, 4)])
@pytest.mark.parametrize("steps", [1, 5])
def test_orthogonalize(shape, steps):
    x = matrix(*shape)
    o = genesis.optim.orthogonalize(T(x), steps=steps)
    # 32-bit products; the iteration amplifies their roundings up to 3.44^steps = 485 times: 485 * 2^-24 * a few
    assert torch.allclose(o._t.double(), reference(x, steps), atol=2e-4)
    assert o.shape == shape and o.dtype == genesis.float32


def test_types_and_degenerate_matrices():
    x = matrix(6, 9, seed=1)
    o = genesis.optim.orthogonalize(T(x.bfloat16()))
    assert o.dtype == genesis.bfloat16
    assert torch.allclose(o._t.double(), reference(x.bfloat16()), atol=2 ** -8 * 1.3 + 2e-4)
    assert torch.equal(genesis.optim.orthogonalize(T(torch.zeros(3, 4)))._t, torch.zeros(3, 4))
    assert genesis.optim.orthogonalize(T(torch.zeros(0, 4)))._t.shape == (0, 4)
    y = matrix(2, 4, 5)
    y[0, 1, 1] = math.inf
    o = genesis.optim.orthogonalize(T(y))._t
    assert torch.isnan(o[0]).all() and torch.allclose(o[1].double(), reference(y[1]), atol=2e-4)
    # another scale is the same matrix; one far below eps fades
    assert torch.allclose(genesis.optim.orthogonalize(T(x * 1e20))._t, genesis.optim.orthogonalize(T(x))._t, atol=1e-4)
    assert genesis.optim.orthogonalize(T(x * 1e-20))._t.abs().max() < 1e-8


def test_refusals():
    x = T(matrix(4, 5))
    for call, error in [
        (lambda: genesis.optim.orthogonalize(matrix(4, 5)), TypeError),
        (lambda: genesis.optim.orthogonalize(T(torch.ones(4, 5, dtype=torch.int64))), TypeError),
        (lambda: genesis.optim.orthogonalize(T(matrix(5))), ValueError),
        (lambda: genesis.optim.orthogonalize(T(matrix(4, 5), requires_grad=True)), ValueError),
        (lambda: genesis.optim.orthogonalize(x, steps=0), ValueError),
        (lambda: genesis.optim.orthogonalize(x, steps=2.0), ValueError),
        (lambda: genesis.optim.orthogonalize(x, eps=0.0), ValueError),
        (lambda: genesis.optim.orthogonalize(x, coefficients=(1.0, 2.0)), ValueError),
        (lambda: genesis.optim.orthogonalize(x, coefficients=(1.0, math.nan, 2.0)), ValueError),
        (lambda: genesis.optim.orthogonalize(x, coefficients=(9.0, 5.0, 2.0)), ValueError),
        (lambda: genesis.optim.Muon([genesis.nn.Parameter(T(matrix(5)))]), ValueError),
        (lambda: genesis.optim.Muon([genesis.nn.Parameter(T(matrix(4, 5)))] * 2), ValueError),
        (lambda: genesis.optim.Muon([genesis.nn.Parameter(T(matrix(4, 5)))], momentum=1.0), ValueError),
    ]:
        with pytest.raises(error):
            call()


@pytest.mark.parametrize("steps", [1, 2, 3, 4, 5, 7, 8])
@pytest.mark.parametrize("coefficients", [COEFFICIENTS, (1.5, -0.5, 0.0), (15 / 8, -10 / 8, 3 / 8), (2.0, -1.5, 0.5)])
def test_program_of_products(steps, coefficients):
    """The products that the kernels are told to make, carried out on the eigenvalues of X X^T in 64 bits: they give the
    iteration, and every scaled entry stays inside fp16's range."""
    rows = [list(_program(steps, coefficients)[i:i + 12]) for i in range(0, len(_program(steps, coefficients)), 12)]
    a, b, c = coefficients
    s = torch.linspace(0, 1, 20001, dtype=torch.float64)
    want = s.clone()
    for _ in range(steps):
        want = a * want + b * want ** 3 + c * want ** 5
    x, x_scale, slots, kept = s.clone(), rows[0][11], {}, set()

    def fits(v, scale):
        assert math.log2(scale) == int(math.log2(scale)) and float(v.abs().max()) * scale < 32768
        return scale

    fits(x, x_scale)
    assert rows[-1][0] == 3 and rows[0][0] == 0
    i = 0
    while i < len(rows):
        results = []
        for kind, lhs, rhs, out, m1, m2, keep, f_acc, f1, f2, scale, _ in rows[i:i + (2 if rows[i][0] == 2 else 1)]:
            if kind == 0:
                results.append((out, f_acc * (x * x_scale) ** 2, scale, keep))
            elif kind == 3:
                q, qs = slots[lhs]
                x = f_acc * (q * qs) * (x * x_scale) + f1 * x
                x_scale = fits(x, scale) if i + 1 < len(rows) else 1.0
            else:
                (l, ls), (r, rs) = slots[lhs], slots[rhs]
                v = f_acc * (l * ls) * (r * rs)
                for m, f in ((m1, f1), (m2, f2)):
                    if m >= 0:
                        assert m in kept
                        v = v + f * slots[m][0]
                results.append((out, v, scale, keep))
                # a launch reads its operands while it writes its results
                assert out not in (lhs, rhs, m2) and out not in [o[2] for o in rows[i:i + (2 if rows[i][0] == 2 else 1)] if o is not rows[i]]
        for out, v, scale, keep in results:
            slots[out] = (v, fits(v, scale))
            (kept.add if keep else kept.discard)(out)
        i += 2 if rows[i][0] == 2 else 1
    assert float((x - want).abs().max()) < 1e-12


def _manual(ps, gs, us, lr, mu, decay, nesterov):
    for p, g, u in zip(ps, gs, us):
        u.mul_(mu).add_(g, alpha=1 - mu)
        y = mu * u + (1 - mu) * g if nesterov else u
        o = reference(y)
        p.mul_(1 - lr * decay).sub_(lr * math.sqrt(max(1.0, p.shape[-2] / p.shape[-1])) * o)


@pytest.mark.parametrize("nesterov", [True, False])
def test_muon_steps(nesterov):
    shapes = [(6, 9), (9, 6), (6, 9), (3, 5, 4)]
    ps = [genesis.nn.Parameter(T(matrix(*s, seed=i))) for i, s in enumerate(shapes)]
    opt = genesis.optim.Muon(ps, lr=0.1, momentum=0.9, nesterov=nesterov, weight_decay=0.05)
    want = [p._t.double().clone() for p in ps]
    us = [torch.zeros_like(w) for w in want]
    for step in range(3):
        gs = [matrix(*s, seed=10 * step + i) for i, s in enumerate(shapes)]
        for p, g in zip(ps, gs):
            p.grad = T(g)
        before = [p._version for p in ps]
        opt.step()
        assert all(p._version > v for p, v in zip(ps, before))
        _manual(want, [g.double() for g in gs], us, 0.1, 0.9, 0.05, nesterov)
        for p, w in zip(ps, want):
            assert torch.allclose(p._t.double(), w, atol=1e-4)


def test_state_dict_and_missing_gradients():
    ps = [genesis.nn.Parameter(T(matrix(4, 6, seed=i))) for i in range(2)]
    opt = genesis.optim.Muon(ps, lr=0.1)
    ps[0].grad = T(matrix(4, 6, seed=5))
    still = ps[1]._t.clone()
    opt.step()
    assert torch.equal(ps[1]._t, still) and list(opt.u) == [0]
    other = [genesis.nn.Parameter(T(p._t.clone())) for p in ps]
    again = genesis.optim.Muon(other)
    again.load_state_dict(opt.state_dict())
    assert again.lr == 0.1 and again.t == 1
    for o, q in ((opt, ps), (again, other)):
        q[0].grad = T(matrix(4, 6, seed=6))
        o.step()
    assert torch.equal(ps[0]._t, other[0]._t)


def test_momenta_stay_where_they_are_when_a_state_is_loaded():
    ps = [genesis.nn.Parameter(T(matrix(4, 6, seed=i))) for i in range(3)]
    opt = genesis.optim.Muon(ps, lr=0.1)
    for i in (0, 1):
        ps[i].grad = T(matrix(4, 6, seed=5 + i))
    opt.step()
    state = opt.state_dict()
    saved = {i: t._t.clone() for i, t in state["u"].items()}
    state = dict(state, u={0: T(saved[0].clone()), 2: T(saved[1].clone())})
    held = dict(opt.u)
    opt.step()
    opt.load_state_dict(state)
    assert opt.u[0] is held[0] and opt.u[1] is held[1]
    assert torch.equal(opt.u[0], saved[0]) and not opt.u[1].any() and torch.equal(opt.u[2], saved[1])


def test_grad_scaler_skips_overflow():
    p = genesis.nn.Parameter(T(matrix(4, 6)))
    opt = genesis.optim.Muon([p], lr=0.1)
    scaler = genesis.amp.GradScaler(init_scale=8.0)
    w = p._t.clone()
    p.grad = T(matrix(4, 6, seed=1) * 8)
    p.grad._t[0, 0] = math.inf
    scaler.step(opt)
    scaler.update()
    assert torch.equal(p._t, w) and opt.t == 0 and not opt.u.get(0, torch.zeros(1)).any()
    p.grad = T(matrix(4, 6, seed=1) * 4)
    scaler.step(opt)
    scaler.update()
    q = genesis.nn.Parameter(T(w.clone()))
    plain = genesis.optim.Muon([q], lr=0.1)
    q.grad = T(matrix(4, 6, seed=1))
    plain.step()
    assert torch.allclose(p._t, q._t, atol=1e-6)
