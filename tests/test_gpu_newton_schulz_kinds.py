"""Every way in which a Newton-Schulz product is worked on: for each, matrices for which the rule chooses it, asked for on the
device that the test runs on, against the iteration in 64 bits."""
import ctypes
import math

import pytest
import torch

import genesis_b200 as genesis
from genesis_b200.ops import dispatch as K
from genesis_b200.ops import native
from genesis_b200.optim.muon import COEFFICIENTS, _programs

pytestmark = pytest.mark.gpu
T = genesis.Tensor
WHOLE, SHARED, PAIRS = 0, 1, 2

# |error| / |result|: what the documentation of `orthogonalize` says, "some 1e-6 to 2e-5"
TOL = 2.5e-5


def plan(sym, m, n, k, batch, problems=1):
    out = (ctypes.c_int * 3)()
    assert native.lib().gb_ns_plan(1 if sym else 0, m, n, k, batch, problems, ctypes.addressof(out)) == 0
    return tuple(out)


def plans(batch, m, n):
    """(X X^T, one m x m product, two of them in a launch, Q X) of a batch of m x n matrices."""
    return (plan(True, m, n, n, batch), plan(True, m, n, m, batch), plan(True, m, n, m, batch, 2), plan(False, m, n, m, batch))


def one_by_one(batch, m, n, steps=5):
    p = native._programs(_programs(steps, COEFFICIENTS))
    return native.lib().gb_ns_one_by_one(*p, m, n, batch) == 1


def matrix(*shape, seed=0, kind="normal"):
    g = torch.Generator("cuda").manual_seed(seed)
    x = torch.randn(*shape, generator=g, device="cuda")
    if kind == "mixed":     # a gradient's: more strong directions, over larger small ones
        x = 0.3 * x + torch.randn(*shape[:-1], 8, generator=g, device="cuda") @ torch.randn(*shape[:-2], 8, shape[-1], generator=g,
                                                                                          device="cuda")
    if kind == "low":       # a few strong directions over a floor of small ones
        x = 0.1 * x + torch.randn(*shape[:-1], 3, generator=g, device="cuda") @ torch.randn(*shape[:-2], 3, shape[-1], generator=g,
                                                                                          device="cuda")
    return x


def iterated(x, steps=5, coefficients=(3.4445, -4.7750, 2.0315), eps=1e-7, dtype=torch.float64):
    a, b, c = coefficients
    y = x.to(dtype)
    y = y.mT if y.shape[-2] > y.shape[-1] else y
    y = y / (torch.linalg.matrix_norm(y, keepdim=True) + eps)
    for _ in range(steps):
        q = y @ y.mT
        y = a * y + (b * q + c * (q @ q)) @ y
    return y.mT if x.shape[-2] > x.shape[-1] else y


def distance(got, want):
    return float((torch.linalg.matrix_norm(got.double() - want) / torch.linalg.matrix_norm(want)).max())


# whether steps are made one by one, which product of `plans`, (kind, columns of a tile, CTAs that share one), batch, m, n
KINDS = [
    (True, 0, (WHOLE, 128, 1), 200, 130, 201),
    (True, 0, (PAIRS, 256, 1), 56, 131, 1518),
    (True, 0, (SHARED, 128, 2), 1, 131, 199),
    (True, 0, (SHARED, 128, 4), 1, 129, 455),
    (True, 0, (SHARED, 128, 8), 1, 135, 1025),
    (True, 0, (SHARED, 256, 2), 25, 131, 331),
    (True, 0, (SHARED, 256, 4), 13, 129, 474),
    (True, 0, (SHARED, 256, 8), 6, 132, 987),
    (True, 0, (SHARED, 128, 8), 1, 101, 4001),
    (True, 0, (WHOLE, 256, 1), 5, 1033, 1834),
    (True, 1, (WHOLE, 128, 1), 1, 129, 130),
    (True, 1, (SHARED, 128, 2), 1, 271, 272),
    (True, 1, (SHARED, 128, 4), 1, 530, 533),
    (True, 1, (SHARED, 256, 2), 13, 324, 343),
    (True, 1, (SHARED, 256, 4), 4, 454, 467),
    (True, 1, (PAIRS, 256, 1), 2, 1476, 1526),
    (True, 1, (WHOLE, 256, 1), 1, 2857, 2959),
    (True, 3, (WHOLE, 128, 1), 1, 129, 260),
    (True, 3, (PAIRS, 256, 1), 18, 129, 7824),
    (True, 3, (SHARED, 128, 2), 1, 195, 200),
    (True, 3, (SHARED, 128, 4), 1, 449, 461),
    (True, 3, (SHARED, 256, 2), 5, 323, 551),
    (True, 3, (SHARED, 256, 4), 2, 452, 531),
    (True, 3, (WHOLE, 256, 1), 42, 260, 13611),
    (False, 0, (WHOLE, 128, 1), 13, 394, 1446),
    (False, 0, (WHOLE, 256, 1), 26, 329, 1843),
    (False, 0, (SHARED, 128, 2), 10, 329, 1866),
    (False, 0, (SHARED, 128, 4), 3, 389, 3605),
    (False, 0, (SHARED, 128, 8), 1, 324, 9851),
    (False, 0, (SHARED, 256, 2), 15, 330, 1684),
    (False, 0, (SHARED, 256, 4), 4, 388, 2636),
    (False, 0, (SHARED, 256, 8), 3, 324, 4117),
    (False, 0, (PAIRS, 256, 1), 15, 392, 1570),
    (False, 1, (SHARED, 128, 4), 1, 460, 5701),
    (False, 1, (SHARED, 256, 2), 15, 321, 1725),
    (False, 1, (SHARED, 256, 4), 5, 455, 1888),
    (False, 1, (PAIRS, 256, 1), 2, 1474, 3219),
    (False, 1, (WHOLE, 128, 1), 8, 389, 2359),
    (False, 1, (WHOLE, 256, 1), 1, 2838, 4687),
    (False, 1, (SHARED, 128, 2), 1, 324, 9851),
    (False, 2, (SHARED, 128, 4), 1, 460, 5701),
    (False, 2, (SHARED, 256, 2), 7, 331, 2320),
    (False, 2, (SHARED, 256, 4), 1, 642, 3108),
    (False, 2, (PAIRS, 256, 1), 1, 1488, 3227),
    (False, 2, (WHOLE, 128, 1), 4, 388, 2636),
    (False, 2, (SHARED, 128, 2), 1, 324, 9851),
    (False, 3, (WHOLE, 128, 1), 1, 324, 9851),
    (False, 3, (WHOLE, 256, 1), 38, 326, 12107),
    (False, 3, (PAIRS, 256, 1), 5, 705, 1846),
]


@pytest.mark.parametrize("kind", ["normal", "low"])
@pytest.mark.parametrize("one,which,how,batch,m,n", KINDS)
def test_each_kind(one, which, how, batch, m, n, kind):
    assert plans(batch, m, n)[which] == how and one_by_one(batch, m, n) == one
    x = matrix(batch, m, n, seed=m, kind=kind)
    want = iterated(x)
    for tall in (False, True):
        given = x.mT.contiguous() if tall else x
        with K.strict_native():
            o = genesis.optim.orthogonalize(T(given))._t
            again = genesis.optim.orthogonalize(T(given))._t
        assert distance(o.mT if tall else o, want) < TOL
        assert torch.equal(o, again)


@pytest.mark.parametrize("steps,coefficients", [(1, (3.4445, -4.7750, 2.0315)), (2, (1.5, -0.5, 0.0)), (4, (2.0, -1.5, 0.5)),
                                                (8, (15 / 8, -10 / 8, 3 / 8))])
@pytest.mark.parametrize("batch,m,n", [(1, 301, 515), (3, 260, 700), (1, 131, 77), (40, 515, 517), (14, 331, 3320), (8, 330, 6762)])
def test_blocks_of_every_length(batch, m, n, steps, coefficients):
    """One step, blocks of two, of two and two, and of three, three and two; and the same steps one by one."""
    if steps > 1:
        assert one_by_one(batch, min(m, n), max(m, n), steps) == (max(m, n) < 5 * min(m, n))
    x = matrix(batch, m, n, seed=steps)
    with K.strict_native():
        o = genesis.optim.orthogonalize(T(x), steps=steps, coefficients=coefficients)._t
    assert distance(o, iterated(x, steps, coefficients)) < TOL


@pytest.mark.parametrize("shape", [(1, 16, 16), (1, 16, 2000), (1, 16, 16000), (1, 24, 9000), (1, 64, 300), (1, 128, 128), (1, 128, 896),
                                   (1, 130, 600), (1, 256, 1024), (20, 200, 3000), (30, 320, 2000), (1, 400, 4000), (1, 1024, 1024),
                                   (1, 896, 4864), (30, 330, 2500), (24, 512, 2048)])
@pytest.mark.parametrize("kind", ["normal", "mixed", "low"])
def test_beside_products_in_32_bits(shape, kind):
    """As exact as the same iteration in 32-bit products, to within a factor of three on average over inputs, and of 1.5 for the
    spectra that gradients have.  Steps in blocks, which are for long or many matrices of more than 320 rows, keep the second; of
    matrices without strong directions they are up to six times as far off."""
    seeds = range(8 if shape[0] == 1 else 2)
    off = plain = 0.0
    for seed in seeds:
        x = matrix(*shape, seed=seed, kind=kind)
        want = iterated(x)
        plain += distance(iterated(x, dtype=torch.float32), want) / len(seeds)
        with K.strict_native():
            off += distance(genesis.optim.orthogonalize(T(x))._t, want) / len(seeds)
    one = one_by_one(*shape)
    assert one == (shape[1] <= 320 or shape[0] == 1 and shape != (1, 896, 4864))
    most = 1.5 if kind == "mixed" else 3 if one or kind == "low" else 6
    assert off < most * plain + 2.0 ** -24, (off, plain)


# (shapes of one batch, with how the wide matrices' last product is worked on: with one row of tiles and more, remainders of
# rows of one to three elements, weights at addresses that are not multiples of 16)
STEPS = [[(33, 65), (65, 33)], [(131, 77), (77, 131)], [(301, 515), (515, 301)], [(449, 461), (461, 449)], [(323, 551)] * 3 + [(551, 323)] * 2,
         [(452, 531), (531, 452)], [(257, 3001)] * 20, [(129, 7824)] * 12 + [(7824, 129)] * 6, [(1, 7)], [(7, 1), (1, 7)]]


@pytest.mark.parametrize("nesterov", [True, False])
@pytest.mark.parametrize("grad_dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shapes", STEPS)
def test_steps_of_an_optimizer(shapes, grad_dtype, nesterov):
    """Two steps against 64 bits.  An update of norm lr sqrt(tall) |o| is off by TOL of it (in the second step the momentum's
    roundings, 2^-22 of it, times 485, come to it: 1.2e-4 of |o| at worst), a weight by 3 roundings of 2^-24 a step."""
    lr, mu, decay = 0.1, 0.9, 0.05
    if len(shapes) > 10 and (grad_dtype != torch.float32 or not nesterov):
        shapes = shapes[:4] + shapes[-4:]
    store = [torch.full((s[0] * s[1] + 4,), 7.0, device="cuda") for s in shapes]
    ps = []
    for i, s in enumerate(shapes):
        w = store[i][i % 4:i % 4 + s[0] * s[1]].view(s)
        w.copy_(matrix(*s, seed=i) * 0.02)
        ps.append(genesis.nn.Parameter(T(w)))
        assert ps[-1]._t.data_ptr() == w.data_ptr()
    around = [t.clone() for t in store]
    opt = genesis.optim.Muon(ps, lr=lr, momentum=mu, weight_decay=decay, nesterov=nesterov)
    want = [p._t.double() for p in ps]
    us = [torch.zeros_like(w) for w in want]
    moved = [0.0] * len(ps)
    for step in range(2):
        for i, (p, s) in enumerate(zip(ps, shapes)):
            p.grad = T(matrix(*s, seed=100 * step + i, kind="low").to(grad_dtype))
        with K.strict_native():
            opt.step()
        for i, (p, w, u) in enumerate(zip(ps, want, us)):
            g = p.grad._t.double()
            u.mul_(mu).add_(g, alpha=1 - mu)
            o = iterated(mu * u + (1 - mu) * g if nesterov else u)
            size = lr * math.sqrt(max(1.0, w.shape[0] / w.shape[1]))
            w.mul_(1 - lr * decay).sub_(size * o)
            moved[i] += size * float(o.norm())
    for i, (p, w, u) in enumerate(zip(ps, want, us)):
        off = float((p._t.double() - w).norm())
        assert off < (TOL + 1.2e-4) * moved[i] + 6 * 2.0 ** -24 * float(w.norm())
        assert float((opt.u[i].double() - u).norm()) < 2.0 ** -22 * float(u.norm())
        # what lies around the weights is as it was
        a, n = i % 4, shapes[i][0] * shapes[i][1]
        assert torch.equal(store[i][:a], around[i][:a]) and torch.equal(store[i][a + n:], around[i][a + n:])
