"""A captured training step after a state has been loaded: it reads and writes the loaded moments, not those that were there
when it was captured."""
import pytest
import torch

import genesis_b200 as genesis

pytestmark = pytest.mark.gpu
T = genesis.Tensor


def _copy(state):
    return {k: ({i: T(t._t.clone()) for i, t in v.items()} if k in ("m", "v", "u") else v) for k, v in state.items()}


@pytest.mark.parametrize("with_muon", [False, True])
def test_a_captured_step_goes_on_with_loaded_moments(with_muon):
    g = torch.Generator().manual_seed(0)
    w = genesis.nn.Parameter(T(torch.randn(64, 96, generator=g).cuda()))
    b = genesis.nn.Parameter(T(torch.randn(96, generator=g).cuda()))
    x = T(torch.randn(5, 64, generator=g).cuda())
    adam = genesis.optim.AdamW([b] if with_muon else [w, b], lr=0.05)
    opts = [adam, genesis.optim.Muon([w], lr=0.05)] if with_muon else [adam]

    def step(x):
        for o in opts:
            o.zero_grad()
        y = x @ w + b
        loss = (y * y).mean()
        loss.backward()
        for o in opts:
            o.step()
        return loss

    graphed = genesis.cuda.GraphedTrainStep(step, opts, [x])
    graphed(x)
    states = [_copy(o.state_dict()) for o in opts]
    at = [p._t.clone() for p in (w, b)]
    graphed(x)
    want = [p._t.clone() for p in (w, b)]
    want_states = [_copy(o.state_dict()) for o in opts]
    for _ in range(3):
        graphed(x)
    for o, s in zip(opts, states):
        o.load_state_dict(s)
    for p, t in zip((w, b), at):
        p._t.copy_(t)
    # whatever the moments have been replaced by is written over
    filled = [torch.full((n,), 1e30, device="cuda") for n in (64 * 96, 96) for _ in range(8)]
    graphed(x)
    torch.cuda.synchronize()
    assert all(torch.equal(p._t, t) for p, t in zip((w, b), want))
    for o, s in zip(opts, want_states):
        assert o.t == s["t"]
        for k in ("m", "v", "u"):
            for i, t in (s.get(k) or {}).items():
                assert torch.equal(getattr(o, k)[i], t._t)
    assert all(bool((f == 1e30).all()) for f in filled)
