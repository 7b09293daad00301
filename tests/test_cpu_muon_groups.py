"""Which matrices a Muon step hands to the kernels together."""
import torch

import genesis_b200 as genesis
from genesis_b200.ops import dispatch as K

T = genesis.Tensor


def matrix(*shape, seed=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed))


def calls_of(opt, monkeypatch):
    seen = []
    plain = K.muon_step
    monkeypatch.setattr(K, "muon_step", lambda params, *a, **k: (seen.append([p for p, _ in params]), plain(params, *a, **k))[1])
    opt.step()
    return seen


def test_weights_of_other_types_and_layouts_go_by_themselves(monkeypatch):
    """A 16-bit or transposed weight, which the kernels do not take, leaves the 32-bit ones of its shape with them."""
    ws = [matrix(4, 6), matrix(4, 6).bfloat16(), matrix(6, 4), matrix(6, 4).t(), matrix(4, 6).double(), matrix(4, 6)]
    ps = [genesis.nn.Parameter(T(w)) for w in ws]
    assert not ps[3]._t.is_contiguous()
    for i, p in enumerate(ps):
        p.grad = T(matrix(*p.shape, seed=i))
    opt = genesis.optim.Muon(ps, lr=0.1)
    seen = calls_of(opt, monkeypatch)
    for params in seen:
        assert len({p.dtype for p in params}) == 1 and len({p.is_contiguous() for p in params}) == 1
    assert sorted(len(p) for p in seen) == [1, 1, 1, 3]
