"""Muon steps of weights of several types and layouts together."""
import pytest
import torch

import genesis_b200 as genesis
from test_cpu_muon_groups import matrix

pytestmark = pytest.mark.gpu
T = genesis.Tensor


def test_weights_of_other_types_leave_the_others_to_the_kernels():
    def build(kinds):
        ps = [genesis.nn.Parameter(T((matrix(40, 60, seed=i) if k != "transposed" else matrix(60, 40, seed=i).t()).cuda()
                                     .to(torch.bfloat16 if k == "bf16" else torch.float32))) for i, k in kinds]
        for (i, _), p in zip(kinds, ps):
            p.grad = T(matrix(40, 60, seed=10 + i).cuda())
        return ps, genesis.optim.Muon(ps, lr=0.1)

    alone, opt = build([(0, "fp32"), (2, "fp32")])
    opt.step()
    mixed, opt = build([(0, "fp32"), (1, "bf16"), (2, "fp32"), (3, "transposed")])
    before = [p._t.clone() for p in mixed]
    opt.step()
    assert torch.equal(mixed[0]._t, alone[0]._t) and torch.equal(mixed[2]._t, alone[1]._t)
    assert all(float((p._t - b).abs().max()) > 1e-3 for p, b in zip(mixed, before))


@pytest.mark.parametrize("momentum", [0.9, 0.95, 0.3])
@pytest.mark.parametrize("shape", [(40, 60), (7, 9)])
def test_momentum_takes_its_weights_from_64_bits(shape, momentum):
    """u = (1 - mu) g in the first step: the weight rounded once and the product once, 2^-24 of u each.  1 - mu of a mu that had
    been rounded before would be off by 2.4e-7."""
    p = genesis.nn.Parameter(T(matrix(*shape).cuda()))
    p.grad = T(matrix(*shape, seed=1).cuda())
    opt = genesis.optim.Muon([p], lr=0.1, momentum=momentum)
    opt.step()
    want = (1.0 - momentum) * p.grad._t.double()
    assert bool(((opt.u[0].double() - want).abs() <= 2.0 ** -23 * 1.001 * want.abs()).all())
