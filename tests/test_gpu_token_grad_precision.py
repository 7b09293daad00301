"""The probabilities in the gradient of logits, each against its own size: the kernels."""
import pytest
import torch

import genesis_b200 as genesis
import genesis_b200.nn.functional as F
from _token_grad_bound import grad_near
from genesis_b200.ops import dispatch as K
from test_cpu_token_grad_precision import SHARED, errors, fresh_rows

pytestmark = pytest.mark.gpu
T = genesis.Tensor


@pytest.mark.parametrize("V", [151936, 2000])
@pytest.mark.parametrize("temperature", [1.0, 0.7])
def test_rows_of_a_fresh_model(temperature, V):
    z, t = fresh_rows(12, V, 1)
    x = T(z.cuda(), requires_grad=True)
    with K.strict_native():
        F.sum(F.token_log_probs(x, T(t.cuda()), temperature=temperature)).backward()
    # (2000 columns: their relative errors, at random up to 3e-7 each, leave 2000^-1/2 of that in the mean, 4 times: 3e-8)
    assert float(errors(x.grad._t, z, t, temperature).mean(-1).abs().max()) < SHARED + (3e-8 if V == 2000 else 0.0)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("std", [0.02, 3.0, 12.0])
@pytest.mark.parametrize("rows,V", [(5, 7), (9, 515), (3, 1025), (4, 16384), (3, 50257), (2, 151936)])
def test_every_probability(rows, V, std, dtype):
    g = torch.Generator().manual_seed(rows * V)
    z = (torch.randn(rows, V, generator=g) * std).to(dtype)
    t = torch.randint(0, V, (rows,), generator=g)
    # (large factors: a 16-bit gradient of 1 / V as it is would be rounded to subnormals in fp16)
    gy = torch.randn(rows, generator=g) * 64
    for temperature in (1.0, 0.7):
        x = T(z.cuda(), requires_grad=True)
        with K.strict_native():
            F.token_log_probs(x, T(t.cuda()), temperature=temperature).backward(T(gy.cuda()))
        grad_near(x.grad._t, z, t, gy / temperature, temperature, what=f"{rows} x {V} T={temperature}")
