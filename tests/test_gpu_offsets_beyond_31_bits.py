"""Logits and matrices of more than 2^31 elements: offsets into them."""
import pytest
import torch

import genesis_b200 as genesis
import genesis_b200.nn.functional as F
from _token_grad_bound import grad_near
from genesis_b200.ops import dispatch as K
from test_gpu_newton_schulz_kinds import TOL
from test_gpu_token_loss_kernels import LP_TOL, exact

pytestmark = pytest.mark.gpu
T = genesis.Tensor


def test_logits():
    """15000 rows of 151936, read through a view that leaves the first position out: rows at both ends, and around 2^31."""
    V, B, L = 151936, 4, 3751
    g = torch.Generator("cuda").manual_seed(0)
    full = torch.empty(B, L, V, dtype=torch.bfloat16, device="cuda").normal_(0.0, 2.0, generator=g)
    t = torch.randint(0, V, (B, L), device="cuda", generator=g)
    gy = torch.randn(B, L - 1, device="cuda", generator=g) * 64
    x = T(full[:, 1:], requires_grad=True)
    assert x._t.numel() > 2 ** 31
    with K.strict_native():
        lp = F.token_log_probs(x, T(t[:, 1:]))
        lp.backward(T(gy))
    rows = (L - 1) * B
    middle = 2 ** 31 // V
    for at in list(range(3)) + list(range(middle - 2, middle + 3)) + list(range(rows - 3, rows)):
        b, i = divmod(at, L - 1)
        z, tok = full[b, i + 1][None], t[b, i + 1][None]
        assert float((lp._t[b, i].double() - exact(z, tok, 1.0)).abs()) < LP_TOL
        grad_near(x.grad._t[b, i][None], z, tok, gy[b, i][None], what=f"row {at}")


@pytest.mark.parametrize("tall", [False, True])
def test_a_matrix(tall):
    """64 x 35 million: the iteration's polynomial in X X^T, which is small, is formed in 64 bits piece by piece."""
    m, n, piece = 64, 35_000_003, 1 << 21
    g = torch.Generator("cuda").manual_seed(1)
    x = torch.empty((n, m) if tall else (m, n), dtype=torch.bfloat16, device="cuda").normal_(generator=g)
    assert x.numel() > 2 ** 31
    w = x.mT if tall else x
    gram = torch.zeros(m, m, dtype=torch.float64, device="cuda")
    for a in range(0, n, piece):
        p = w[:, a:a + piece].double()
        gram += p @ p.mT
    norm = gram.diagonal().sum().sqrt() + 1e-7
    A, P, eye = gram / norm ** 2, None, torch.eye(m, dtype=torch.float64, device="cuda")
    P = eye
    for _ in range(5):
        step = 3.4445 * eye - 4.7750 * A + 2.0315 * (A @ A)
        P, A = step @ P, step @ A @ step
    with K.strict_native():
        o = genesis.optim.orthogonalize(T(x))._t
    o = o.mT if tall else o
    for a in (0, 2 ** 31 // m - 5000, 2 ** 25, n - 10000):
        want = P @ (w[:, a:a + 10000].double() / norm)
        off = (o[:, a:a + 10000].double() - want).abs()
        # half a step of the type for every element, and what the products are off by
        assert bool((off <= 2.0 ** -8 * want.abs() + TOL * want.norm()).all())
        assert float(off.norm()) < 2.0 ** -8 * float(want.norm())
