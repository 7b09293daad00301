"""The losses on tokens' log-probabilities from their definitions, in 64 bits on the CPU, through torch's own autograd."""
import torch
import torch.nn.functional as TF

IGNORE = -100


def leaf64(logits):
    return logits.detach().cpu().double().requires_grad_()


def log_probs(z, tokens, temperature=1.0, ignore=IGNORE):
    """0 where ignored; rows that do not count take no part at all, whatever they hold."""
    tokens = tokens.cpu().long()
    on = tokens != ignore
    rows = TF.log_softmax(z[on] / temperature, -1)
    lp = torch.zeros(tokens.shape, dtype=torch.float64)
    return lp.masked_scatter(on, rows.gather(-1, tokens[on].unsqueeze(-1)).squeeze(-1)) if on.any() else lp + 0 * z[on].sum(), on


def policy(z, tokens, old, adv, ref=None, clip=0.2, clip_high=None, kl=0.0, temperature=1.0, ignore=IGNORE):
    """Losses per token, and which tokens count."""
    lp, on = log_probs(z, tokens, temperature, ignore)
    adv = adv.cpu().double()
    adv = adv if adv.shape == lp.shape else adv.unsqueeze(-1).expand(lp.shape)

    def put(x):
        return torch.where(on, x.cpu().double(), torch.zeros_like(lp))

    adv = put(adv)
    r = torch.exp(lp - put(old))
    lo, hi = 1 - clip, 1 + (clip if clip_high is None else clip_high)
    # outside the clipping range on the side that the advantage pushes to, the loss does not depend on the ratio
    stuck = ((adv > 0) & (r > hi)) | ((adv < 0) & (r < lo))
    each = -adv * torch.where(stuck, r.clamp(lo, hi).detach(), r)
    if ref is not None:
        d = put(ref) - lp
        each = each + kl * (torch.exp(d) - d - 1)
    return torch.where(on, each, torch.zeros_like(each)), on


def preference(z, tokens, ref, beta=0.1, smoothing=0.0, ignore=IGNORE):
    lp, _ = log_probs(z, tokens, ignore=ignore)
    rewards = beta * (lp.sum(-1) - ref.cpu().double())
    P = rewards.numel() // 2
    h = rewards[:P] - rewards[P:]
    return -(1 - smoothing) * TF.logsigmoid(h) - smoothing * TF.logsigmoid(-h), rewards


def grad_close(got, ref, row_factor, what=""):
    """Elementwise: half a step of the type, plus 2e-5 of the row's factor (errors of a probability: its exponent's rounding,
    up to 40 log2(e) 2^-23, the rounding of log s and the hardware exponential's 2^-22 stay below 1e-5 of it, the factor's own
    error through exp(lp - old) is another 1e-5), plus half of the smallest subnormal."""
    eps = torch.finfo(got.dtype).eps / 2
    ref = ref.double()
    tol = eps * ref.abs() + 2e-5 * row_factor.abs().unsqueeze(-1) + (2.0 ** -25 if got.dtype == torch.float16 else 0.0)
    bad = (got.cpu().double() - ref).abs() > tol
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} elements off, worst " \
                          f"{float(((got.cpu().double() - ref).abs() - tol).max()):.3g} beyond the tolerance"
