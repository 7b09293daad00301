"""Which matrices a Muon step hands to the kernels together."""
import pytest
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


def test_scalars_go_to_the_device_of_the_weights(monkeypatch):
    """With weights on several devices, the scale, the overflow flag and the learning rate follow each of them: a kernel that was
    given another device's address would read outside its memory.  ("meta" stands for a second device.)"""
    ps = [genesis.nn.Parameter(T(matrix(4, 6))), genesis.nn.Parameter(T(matrix(4, 6).to("meta")))]
    for p in ps:
        p.grad = T(torch.ones(4, 6, device=p._t.device))
    opt = genesis.optim.Muon(ps, lr=0.1)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    opt._grad_scale, opt._found_inf, opt._dyn_lr_t = torch.ones(1), torch.zeros(1), torch.tensor([0.1])
    seen = {}
    monkeypatch.setattr(K, "muon_step", lambda params, grads, bufs, *a: seen.update({params[0][0].device.type: a[-3:]}))
    opt.step()
    assert set(seen) == {"cpu", "meta"}
    for dev, scalars in seen.items():
        assert all(s.device.type == dev for s in scalars)


def test_sides_beyond_32_bits_do_not_reach_the_kernels():
    """A side of 2^31 and more would arrive there as a negative number, for which nothing is done and the result is whatever the
    memory held.  Such a matrix goes to the library."""
    from genesis_b200.ops import native
    from genesis_b200.optim.muon import _check
    coefficients, eps, program = _check(1, (1.5, -0.5, 0.0), 1e-7)
    for shape in ((1, 1, 2 ** 30 + 1), (1, 2 ** 31 + 5, 1)):
        x = torch.empty(shape, dtype=torch.bfloat16, device="meta")
        assert native.newton_schulz(x, 1, coefficients, eps, program) is NotImplemented
        w = [(torch.empty(shape, device="meta"), 0)]
        assert native.muon_step(w, w, w, (1, max(shape)), 0.1, 0.9, True, 0.0, 1.0, 1, coefficients, eps, program, None, None,
                                None) is NotImplemented


def test_a_norm_beyond_32_bits():
    """Elements near 1e38: the matrix is the same up to scale, and comes out as that of elements near 1."""
    x = matrix(20, 30, seed=2).clamp(-3, 3)
    big = genesis.optim.orthogonalize(T(x * 1e38))._t
    # scaling rounds each element once more, 2^-24 of it, which the iteration amplifies by 485 at most; as much for the products
    assert float((big - genesis.optim.orthogonalize(T(x))._t).abs().max()) < 485 * 2.0 ** -24 * 4


def test_no_result_is_kept_in_32_bits_that_nothing_reads():
    from genesis_b200.optim.muon import COEFFICIENTS, _program
    for steps, longest in [(k, n) for k in (1, 2, 3, 4, 5, 7, 8) for n in (3, 1)]:
        flat = list(_program(steps, COEFFICIENTS, longest))
        rows = [flat[i:i + 12] for i in range(0, len(flat), 12)]
        for i, (kind, _, _, out, _, _, keep, *_) in enumerate(rows):
            if kind == 3:
                continue
            read = False
            for j in range(i + 1, len(rows)):
                # the launch that a row of kind 2 shares with the next one reads before either has written
                read |= out in rows[j][4:6] and not (kind == 2 and j == i + 1)
                if rows[j][0] in (0, 3) or rows[j][3] == out:
                    break
            assert bool(keep) == read, (steps, i)


@pytest.mark.parametrize("steps", [1, 2, 3, 5, 8])
@pytest.mark.parametrize("coefficients", [(3.4445, -4.7750, 2.0315), (1.5, -0.5, 0.0), (15 / 8, -10 / 8, 3 / 8), (2.0, -1.5, 0.5)])
def test_program_of_steps_one_by_one(steps, coefficients, monkeypatch):
    """The same steps without blocks: for each X X^T, the matrix that X is multiplied by, and the product."""
    import test_cpu_muon
    from genesis_b200.optim.muon import _program
    flat = list(_program(steps, coefficients, 1))
    assert [flat[i] for i in range(0, len(flat), 12)] == [0, 1, 3] * steps
    monkeypatch.setattr(test_cpu_muon, "_program", lambda s, c: _program(s, c, 1))
    test_cpu_muon.test_program_of_products(steps, coefficients)
