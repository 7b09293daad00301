"""Every kernel that the losses on log-probabilities choose between, in every type: rows that all count, of even and odd
length, forward and backward.  Shapes follow the rules of `csrc/token_loss.cu` for the number of SMs that the device has."""
import pytest
import torch

import genesis_b200 as genesis
import genesis_b200.nn.functional as F
from _token_grad_bound import grad_near
from genesis_b200.ops import dispatch as K

pytestmark = pytest.mark.gpu
T = genesis.Tensor
SIZE = {torch.float32: 4, torch.bfloat16: 2, torch.float16: 2}

# Log-probabilities of normal logits of deviation 2 (below 10 of the row's maximum apart, below 32 in size): log s through the
# hardware exponential's 2^-22 and arguments of up to 20 log2(e) rounded to 2^-24 of themselves, 2e-6, and lp's own rounding
LP_TOL = 4e-6


def sms():
    return torch.cuda.get_device_properties(0).multi_processor_count


def rows_of(name, dtype):
    """(rows, columns) that the rule gives to the kernel `name`."""
    n, size = sms(), SIZE[dtype]
    return {
        "warp, short rows": (19, 2048 // size - 1),
        "warp, many rows": (32 * n + 5, 8192 // size - 3),
        "128 threads, few rows": (2 * n + 3, 8192 // size - 3),
        "128 threads, many rows": (8 * n + 3, 8192 // size + 805),
        "512 threads": (2 * n, 8192 // size + 5),
        "512 threads, one row": (1, 32767),
        "cluster of 2": (n // 2, 32769),
        "cluster of 4": (n // 4, 65539),
        "cluster of 8": (n // 8, 131073),
        "cluster of 8, one row": (1, 151937),
        "256 threads": (2 * n + 1, 8192 // size + 5),
        "256 threads, long rows": (2 * n + 1, 50257),
        "256 threads, aligned rows": (3 * n, 32768),
    }[name]


NAMES = ["warp, short rows", "warp, many rows", "128 threads, few rows", "128 threads, many rows", "512 threads",
         "512 threads, one row", "cluster of 2", "cluster of 4", "cluster of 8", "cluster of 8, one row", "256 threads",
         "256 threads, long rows", "256 threads, aligned rows"]


def exact(z, t, temperature):
    out = []
    step = max(1, (1 << 25) // z.shape[1])
    for a in range(0, z.shape[0], step):
        d = z[a:a + step].double() / temperature
        out.append(d.gather(1, t[a:a + step, None]).squeeze(1) - torch.logsumexp(d, 1))
    return torch.cat(out)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("name", NAMES)
def test_forward_and_backward(name, dtype):
    rows, V = rows_of(name, dtype)
    g = torch.Generator("cuda").manual_seed(len(name))
    z = (torch.randn(rows, V, device="cuda", generator=g) * 2).to(dtype)
    t = torch.randint(0, V, (rows,), device="cuda", generator=g)
    t[-1] = V - 1
    gy = torch.randn(rows, device="cuda", generator=g) * 64
    x = T(z, requires_grad=True)
    with K.strict_native():
        lp = F.token_log_probs(x, T(t), temperature=0.9)
        lp.backward(T(gy))
    want = exact(z, t, 0.9)
    assert float(want.min()) > -32
    assert float((lp._t.double() - want).abs().max()) < LP_TOL
    grad_near(x.grad._t, z, t, gy / 0.9, 0.9, what=name)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("name", [n for n in NAMES if not n.endswith("one row")])
def test_rows_that_do_not_count_between_others(name, dtype):
    """Rows with the ignored token hold NaN: they reach nothing, and the others come out as if they stood alone."""
    rows, V = rows_of(name, dtype)
    g = torch.Generator("cuda").manual_seed(len(name))
    z = (torch.randn(rows, V, device="cuda", generator=g) * 2).to(dtype)
    t = torch.randint(0, V, (rows,), device="cuda", generator=g)
    off = torch.arange(rows, device="cuda") % 3 == 1
    clean = z.clone()
    z[off] = float("nan")
    ignored = torch.where(off, -100, t)

    def both(z, t):
        x = T(z, requires_grad=True)
        lp = F.token_log_probs(x, T(t))
        F.sum(lp).backward()
        return lp._t, x.grad._t

    lp, grad = both(z, ignored)
    assert not lp[off].any() and not grad[off].any()
    want_lp, want_grad = both(clean, t)
    assert torch.equal(lp[~off], want_lp[~off]) and torch.equal(grad[~off], want_grad[~off])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_warps_write_the_gradient_of_many_rows(dtype):
    """More than 1024 columns, at most 8 KB a row, and rows enough to fill the device: a warp a row in the backward pass."""
    rows, V = 32 * sms() + 1, 8192 // SIZE[dtype] - 5
    assert V > 1024
    g = torch.Generator("cuda").manual_seed(3)
    z = (torch.randn(rows, V, device="cuda", generator=g) * 2).to(dtype)
    t = torch.randint(0, V, (rows,), device="cuda", generator=g)
    gy = torch.randn(rows, device="cuda", generator=g) * 64
    x = T(z, requires_grad=True)
    with K.strict_native():
        F.token_log_probs(x, T(t)).backward(T(gy))
    grad_near(x.grad._t, z, t, gy)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("name", ["warp, many rows", "128 threads, many rows", "cluster of 8", "256 threads, long rows"])
def test_losses_through_each_kernel(name, dtype):
    """The policy and the preference loss over the same kernels: their rows' factors, on the device, times the same gradient."""
    rows, V = rows_of(name, dtype)
    rows -= rows % 2
    g = torch.Generator("cuda").manual_seed(5)
    z = (torch.randn(2, rows // 2, V, device="cuda", generator=g) * 2).to(dtype)
    t = torch.randint(0, V, (2, rows // 2), device="cuda", generator=g)
    lp = exact(z.view(rows, V), t.view(-1), 1.0).view(2, -1)
    old = (lp - 0.05).float()                            # (a ratio of 1.05, inside the clipping range)
    adv = torch.tensor([1.5, -0.5], device="cuda") * 64 * rows
    x = T(z, requires_grad=True)
    with K.strict_native():
        F.policy_loss(x, T(t), T(old), T(adv)).backward()
    ratio = torch.exp(lp - old.double())
    # (the ratio is off by lp's and its own roundings, 1e-5 of itself: more than the bound's 8 * 2^-24, so it is taken from 32 bits)
    with genesis.no_grad():
        ratio32 = torch.exp(F.token_log_probs(T(z), T(t))._t - old)
    assert float((ratio32.double() / ratio - 1).abs().max()) < 1e-5
    factor = -adv[:, None].double() * ratio32.double() / rows
    grad_near(x.grad._t.view(rows, V), z.view(rows, V), t.view(-1), factor.reshape(-1))
    ref = lp.sum(1) + torch.tensor([0.3, -0.2], device="cuda").double()
    x = T(z, requires_grad=True)
    with K.strict_native():
        loss, rewards = F.preference_loss(x, T(t), T(ref), beta=2.0, return_rewards=True)
        loss.backward(T(torch.full((), 64.0, device="cuda")))
    assert float((rewards._t.double() - 2.0 * (lp.sum(1) - ref)).abs().max()) < 2.0 * (rows // 2 * 4e-8 + 1e-4)
    h = (rewards._t[0] - rewards._t[1]).double()
    factor = torch.stack((-torch.sigmoid(-h), torch.sigmoid(-h))) * 2.0 * 64
    grad_near(x.grad._t.view(rows, V), z.view(rows, V), t.view(-1), factor.repeat_interleave(rows // 2))
