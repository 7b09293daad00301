"""Loading a state into an optimizer one of whose steps has been captured: its buffers stay where they are."""
import pytest
import torch

import genesis_b200 as genesis

T = genesis.Tensor


def matrix(*shape, seed=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed))


def build(kind):
    ps = [genesis.nn.Parameter(T(matrix(4, 6, seed=i))) for i in range(3)]
    make = {"adamw": lambda: genesis.optim.AdamW(ps, lr=0.1), "adam": lambda: genesis.optim.Adam(ps, lr=0.1),
            "sgd": lambda: genesis.optim.SGD(ps, lr=0.1, momentum=0.9)}[kind]
    return ps, make()


@pytest.mark.parametrize("kind", ["adamw", "adam", "sgd"])
def test_buffers_stay_once_a_step_has_been_captured(kind):
    ps, opt = build(kind)
    names = [n for n in ("m", "v", "u") if hasattr(opt, n)]
    for i in (0, 1):
        ps[i].grad = T(matrix(4, 6, seed=5 + i))
    opt.step()
    saved = {n: {i: t.clone() for i, t in getattr(opt, n).items()} for n in names}
    state = dict(opt.state_dict(), **{n: {0: T(saved[n][0].clone()), 2: T(saved[n][1].clone())} for n in names})
    opt.step()
    opt._state_stays = True                      # (what a captured step sets)
    held = {n: dict(getattr(opt, n)) for n in names}
    opt.load_state_dict(state)
    for n in names:
        now = getattr(opt, n)
        assert now[0] is held[n][0] and now[1] is held[n][1]
        assert torch.equal(now[0], saved[n][0]) and not now[1].any() and torch.equal(now[2], saved[n][1])


@pytest.mark.parametrize("kind", ["adamw", "sgd"])
def test_buffers_are_replaced_otherwise(kind):
    """A state that was taken by reference and put aside keeps its values when another one is loaded."""
    ps, opt = build(kind)
    ps[0].grad = T(matrix(4, 6, seed=5))
    opt.step()
    aside = opt.state_dict()
    name = "m" if kind == "adamw" else "u"
    values = aside[name][0]._t.clone()
    other = build(kind)[1]
    opt.load_state_dict(other.state_dict())
    assert torch.equal(aside[name][0]._t, values) and 0 not in getattr(opt, name)


def test_an_optimizer_listed_twice_is_refused():
    ps, opt = build("adamw")
    with pytest.raises(ValueError, match="twice"):
        genesis.cuda.GraphedTrainStep(lambda: None, [opt, opt], [])
