"""The probabilities in the gradient of 32-bit logits, each against its own size: on the CPU."""
import pytest
import torch

import genesis_b200 as genesis
import genesis_b200.nn.functional as F
import _token_loss_ref as R

T = genesis.Tensor


def fresh_rows(rows, V, seed):
    """Logits near 0, as those of a model that has not been trained: all probabilities are near 1 / V."""
    g = torch.Generator().manual_seed(seed)
    return torch.randn(rows, V, generator=g) * 0.02, torch.randint(0, V, (rows,), generator=g)


def errors(grad, z, t, temperature):
    """Relative errors of the rows' probabilities, from gradients for an incoming 1; the token's own element is left out."""
    r = R.leaf64(z)
    R.log_probs(r, t, temperature)[0].sum().backward()
    rel = grad.cpu().double() / r.grad - 1
    return rel.scatter(-1, t[:, None], 0.0)


# A row's common error: the roundings of its sum (and of additions on the way to it, which a tree of them or 64-bit joins keep
# at one more), of the quotient by it and of 1 / T, 2^-24 each, and the mean error of the exponential, 5e-8: 2.9e-7.  log2 of
# the sum rounded to 32 bits in the exponent is off by up to 2^-20, and a row with it by 6.6e-7.
SHARED = 2.9e-7


@pytest.mark.parametrize("temperature", [1.0, 0.7])
def test_rows_of_a_fresh_model(temperature):
    z, t = fresh_rows(12, 151936, 1)
    x = T(z, requires_grad=True)
    F.sum(F.token_log_probs(x, T(t), temperature=temperature)).backward()
    assert float(errors(x.grad._t, z, t, temperature).mean(-1).abs().max()) < SHARED
