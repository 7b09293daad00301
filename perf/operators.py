"""Losses on a language model's logits and the orthogonalised update of a weight matrix, as cases that can be measured.

Four operators of post-training, each beside one that the framework has had before (the cross-entropy, the optimizers):

* `token_log_probs`: log-probabilities of given tokens, forward (scoring samples, the reference model) and with gradient;
* `policy_loss`: the clipped policy objective with a KL term against a reference, forward and backward from the logits;
* `preference_loss`: the loss of paired log ratios of chosen and rejected answers, forward and backward from the logits;
* `orthogonalize` and the `Muon` step: Newton-Schulz products that replace the singular values of an update by about one.

`run` computes each case in plain torch, or with `own` through the framework; `exact` restates it in 64 bits.  Vocabularies
are those of this repository's benchmarks (151936, 65536, 50257, 32000); weight matrices are those of hidden 896 with FFN 4864
(14 query and 2 KV heads of 64).
"""
import math

import torch

own = False

DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}
IGNORE = -100
CLIP, CLIP_HIGH, KL, BETA, SMOOTH = 0.2, 0.28, 0.04, 0.1, 0.05
COEFFICIENTS, STEPS, EPS = (3.4445, -4.7750, 2.0315), 5, 1e-7
LR, MOMENTUM, DECAY = 0.02, 0.95, 0.1
LARGEST = 8192 * 151936          # logits of the largest listed loss


# ------------------------------------------------------------------------------------------------
# the cases
# ------------------------------------------------------------------------------------------------
def listed():
    return [
        # log-probabilities of the 16 tokens that one decoding step of a batch has drawn: few rows, all latency
        dict(name="logp_step", kind="logp", B=16, T=1, V=151936, dtype="bf16", prompt=0, pad=0, train=False, temperature=0.7),
        # a reference model scores a batch of answers, prompts left out
        dict(name="logp_score", kind="logp", B=8, T=1024, V=151936, dtype="bf16", prompt=128, pad=64, train=False,
             temperature=1.0),
        # a user's own loss on log-probabilities: rows of odd length in fp16, gradient per token
        dict(name="logp_train", kind="logp", B=4, T=333, V=50257, dtype="fp16", prompt=20, pad=9, train=True, temperature=1.0),
        # a small policy in fp32: the smallest training call
        dict(name="policy_small", kind="policy", B=4, T=16, V=512, dtype="fp32", prompt=2, pad=3, kl=True, per_token=False),
        # one micro-batch of policy training, a third of it prompt, advantages per sequence
        dict(name="policy_train", kind="policy", B=8, T=1024, V=151936, dtype="bf16", prompt=340, pad=100, kl=True,
             per_token=False),
        # a policy with a critic: advantages per token, fp16 logits, no reference model, all tokens count
        dict(name="policy_critic", kind="policy", B=2, T=1000, V=65536, dtype="fp16", prompt=0, pad=0, kl=False,
             per_token=True),
        # two pairs of short answers, rows of odd length
        dict(name="preference_small", kind="preference", B=4, T=33, V=50257, dtype="bf16", prompt=7, pad=11),
        # four pairs of a thousand tokens
        dict(name="preference_train", kind="preference", B=8, T=1024, V=151936, dtype="bf16", prompt=200, pad=150),
        # the update of one small matrix (a key projection's): a chain of short products
        dict(name="orth_small", kind="orth", count=1, rows=128, cols=896, dtype="fp32"),
        # a down projection's update held in bf16
        dict(name="orth_wide", kind="orth", count=1, rows=896, cols=4864, dtype="bf16"),
        # the up projections of 24 layers together: tall matrices, the largest of all
        dict(name="orth_stack", kind="orth", count=24, rows=4864, cols=896, dtype="fp32"),
        # the optimizer's step over the matrices of four layers
        dict(name="muon_step", kind="muon", layers=4, hidden=896, inner=4864, kv=128, dtype="fp32"),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["logp", "logp", "policy", "policy", "preference", "preference", "orth", "orth", "muon"])
    if kind == "orth":
        m, n = _log(rng, 16, 2048), _log(rng, 16, 5000)
        count = _log(rng, 1, 24)
        while count > 1 and _orth_flops(count, m, n) > _orth_flops(24, 4864, 896):
            count -= 1
        return dict(kind=kind, count=count, rows=m, cols=n, dtype=rng.choice(["fp32", "fp32", "bf16", "fp16"]))
    if kind == "muon":
        hidden = _log(rng, 64, 1024)
        return dict(kind=kind, layers=rng.randint(1, 4), hidden=hidden, inner=_log(rng, hidden, 4 * hidden),
                    kv=_log(rng, 16, hidden), dtype="fp32")
    V = rng.choice([151936, 128256, 65536, 50257, 32000, _log(rng, 300, 160000), _log(rng, 300, 160000)])
    rows = _log(rng, 8, min(16384, LARGEST // V))
    B = 2 * rng.randint(1, 4)
    T = max(1, rows // B)
    case = dict(kind=kind, B=B, T=T, V=V, dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]) if rows * V < LARGEST // 2 else "bf16",
                prompt=rng.randint(0, T // 2), pad=rng.randint(0, T // 3))
    if kind == "logp":
        case.update(train=rng.random() < 0.5, temperature=rng.choice([1.0, 0.7, 1.3]))
    elif kind == "policy":
        case.update(kl=rng.random() < 0.6, per_token=rng.random() < 0.5)
    return case


def _matrices(case):
    """(rows, cols) of the weight matrices of one decoder layer: q, k, v, o, gate, up, down."""
    H, I, kv = case["hidden"], case["inner"], case["kv"]
    return [(H, H), (kv, H), (kv, H), (H, H), (I, H), (I, H), (H, I)] * case["layers"]


def _lengths(case):
    """(first, behind the last) counted position of every sequence: a prompt before the answer, padding behind it."""
    T, P, pad = case["T"], case["prompt"], case["pad"]
    return [(P, T - (i * 7) % (pad + 1)) for i in range(case["B"])]


# ------------------------------------------------------------------------------------------------
# inputs
# ------------------------------------------------------------------------------------------------
def _log_probs64(logits, tokens, temperature):
    """Log-probabilities of `tokens` [N] under logits [N, V], in 64 bits, a block of rows at a time."""
    out = torch.empty(logits.shape[0], dtype=torch.float64, device=DEV)
    step = max(1, (1 << 27) // logits.shape[1])
    for a in range(0, logits.shape[0], step):
        z = logits[a:a + step].double() / temperature
        out[a:a + step] = z.gather(1, tokens[a:a + step, None]).squeeze(1) - torch.logsumexp(z, 1)
    return out


def _inputs(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, device=DEV, generator=g)

    if case["kind"] == "orth":
        # a gradient's spectrum: a few strong directions over a floor of small ones
        E, R, C = case["count"], case["rows"], case["cols"]
        x = normal(E, R, C).mul_(0.3).baddbmm_(normal(E, R, 8), normal(E, 8, C)).mul_(1e-3)
        return dict(x=x.to(TYPES[case["dtype"]]) if E > 1 else x[0].to(TYPES[case["dtype"]]))
    if case["kind"] == "muon":
        d = dict(w=[], g=[], u=[])
        for r, c in _matrices(case):
            d["w"].append(normal(r, c) * 0.02)
            d["g"].append((normal(r, c) * 0.3 + normal(r, 8) @ normal(8, c)) * 1e-3)
            d["u"].append((normal(r, c) * 0.1 + normal(r, 8) @ normal(8, c)) * 1e-3)
        return d
    B, T, V = case["B"], case["T"], case["V"]
    logits = torch.empty(B * T, V, dtype=TYPES[case["dtype"]], device=DEV)
    tokens = torch.empty(B * T, dtype=torch.int64, device=DEV)
    step = max(1, (1 << 27) // V)
    for a in range(0, B * T, step):
        z = normal(min(step, B * T - a), V).mul_(3.0)
        logits[a:a + step] = z
        # tokens that the model itself has drawn: the largest of the logits plus Gumbel noise
        noise = torch.empty_like(z).exponential_(generator=g).log_()
        tokens[a:a + step] = torch.argmax(z.sub_(noise), 1)
    d = dict(logits=logits.view(B, T, V))
    temperature = case.get("temperature", 1.0)
    counted = torch.zeros(B, T, dtype=torch.bool, device=DEV)
    for i, (a, b) in enumerate(_lengths(case)):
        counted[i, a:b] = True
    d["tokens"] = torch.where(counted, tokens.view(B, T), torch.full_like(tokens.view(B, T), IGNORE))
    if case["kind"] == "logp":
        if case["train"]:
            d["gy"] = normal(B, T) / (B * T)
        return d
    lp = _log_probs64(logits, tokens, temperature).view(B, T)
    if case["kind"] == "policy":
        # the log ratio to the policy that drew the tokens, a few updates ago; ratios within a thousandth of a clipping
        # border, where the gradient jumps, are moved off it
        delta = normal(B, T).double() * 0.15
        for border in (math.log(1 - CLIP), math.log(1 + CLIP_HIGH)):
            near = (delta - border).abs() < 1e-3
            delta = torch.where(near, delta + torch.where(delta < border, -2e-3, 2e-3), delta)
        d["old"] = (lp - delta).float()
        d["adv"] = normal(B, T) + 0.25 if case["per_token"] else normal(B) + 0.25
        if case["kl"]:
            d["ref"] = (lp + normal(B, T) * 0.3).float()
        return d
    total = torch.where(counted, lp, torch.zeros_like(lp)).sum(1)
    d["ref"] = (total + normal(B).double() * 8).float()
    return d


def prepare(case, seed):
    s = dict(_inputs(case, seed), case=case)
    if not own:
        return s
    import os
    # torch's own memory statistics, which a timing program may ask for, exist only with torch's own allocator
    os.environ.setdefault("GENESIS_B200_POOL", "0")
    import genesis_b200 as genesis
    if case["kind"] == "muon":
        s["params"] = [genesis.nn.Parameter(genesis.Tensor(w)) for w in s["w"]]
        for p, g in zip(s["params"], s["g"]):
            p.grad = genesis.Tensor(g)
        s["opt"] = genesis.optim.Muon(s["params"], lr=LR, momentum=MOMENTUM, weight_decay=DECAY, steps=STEPS,
                                      coefficients=COEFFICIENTS, eps=EPS)
        s["opt"].load_state_dict({"u": dict(enumerate(s["u"]))})
        return s
    train = case.get("train", case["kind"] in ("policy", "preference"))
    for n in ("x", "tokens", "gy", "old", "adv", "ref"):
        if n in s:
            s[n] = genesis.Tensor(s[n])
    if "logits" in s:
        s["logits"] = genesis.Tensor(s["logits"], requires_grad=train)
    return s


# ------------------------------------------------------------------------------------------------
# one pass
# ------------------------------------------------------------------------------------------------
def _rows(s, temperature):
    """Log-probabilities [B, T] of the counted tokens (0 elsewhere) in 32 bits, and what their gradient needs."""
    z = s["logits"].float() / temperature
    valid = s["tokens"] != IGNORE
    tok = torch.where(valid, s["tokens"], torch.zeros_like(s["tokens"])).unsqueeze(-1)
    z = z - z.max(-1, keepdim=True).values
    e = torch.exp(z)
    total = e.sum(-1, keepdim=True)
    lp = (z.gather(-1, tok) - torch.log(total)).squeeze(-1)
    return torch.where(valid, lp, torch.zeros_like(lp)), (valid, tok, e, total, temperature)


def _logits_grad(s, rows, g):
    """Gradient of the logits from the gradient [B, T] of their tokens' log-probabilities, rounded once."""
    valid, tok, e, total, temperature = rows
    g = torch.where(valid, g, torch.zeros_like(g)).unsqueeze(-1) / temperature
    d = -g * (e / total)
    d.scatter_add_(-1, tok, g)
    return d.to(s["logits"].dtype)


def _newton_schulz(x):
    a, b, c = COEFFICIENTS
    tall = x.shape[-2] > x.shape[-1]
    x = x.float()
    x = x.transpose(-2, -1) if tall else x
    x = x / (x.square().sum((-2, -1), keepdim=True).sqrt() + EPS)
    for _ in range(STEPS):
        A = x @ x.transpose(-2, -1)
        x = a * x + (b * A + c * (A @ A)) @ x
    return x.transpose(-2, -1) if tall else x


def run(s):
    case = s["case"]
    if own:
        return _run_own(s, case)
    kind = case["kind"]
    if kind == "orth":
        return [_newton_schulz(s["x"]).to(s["x"].dtype)]
    if kind == "muon":
        for w, g, u in zip(s["w"], s["g"], s["u"]):
            u.mul_(MOMENTUM).add_(g, alpha=1 - MOMENTUM)
            o = _newton_schulz(g * (1 - MOMENTUM) + u * MOMENTUM)
            w.mul_(1 - LR * DECAY).add_(o, alpha=-LR * math.sqrt(max(1.0, w.shape[0] / w.shape[1])))
        return s["w"] + s["u"]
    lp, rows = _rows(s, case.get("temperature", 1.0))
    valid = rows[0]
    if kind == "logp":
        return [lp, _logits_grad(s, rows, s["gy"])] if case["train"] else [lp]
    if kind == "policy":
        adv = s["adv"] if case["per_token"] else s["adv"].unsqueeze(1)
        count = valid.sum().clamp(min=1)
        r = torch.exp(lp - s["old"])
        plain, clipped = -adv * r, -adv * r.clamp(1 - CLIP, 1 + CLIP_HIGH)
        loss = torch.maximum(plain, clipped)
        g = torch.where(plain >= clipped, plain, torch.zeros_like(plain))
        if case["kl"]:
            d = s["ref"] - lp
            loss = loss + KL * (torch.exp(d) - d - 1)
            g = g + KL * (1 - torch.exp(d))
        loss = torch.where(valid, loss, torch.zeros_like(loss)).sum() / count
        return [loss, _logits_grad(s, rows, g / count)]
    # sums over a whole answer lose the low digits of the difference of two of them in 32 bits
    rewards = (BETA * (lp.double().sum(1) - s["ref"].double())).float()
    h = rewards[:case["B"] // 2] - rewards[case["B"] // 2:]
    P = h.numel()
    loss = ((1 - SMOOTH) * _softplus(-h) + SMOOTH * _softplus(h)).sum() / P
    gh = (SMOOTH - 1 / (1 + torch.exp(h))) * (BETA / P)
    return [loss, rewards, _logits_grad(s, rows, torch.cat([gh, -gh]).unsqueeze(1).expand_as(lp))]


def _softplus(x):
    return x.clamp(min=0) + torch.log1p(torch.exp(-x.abs()))


def _run_own(s, case):
    import genesis_b200 as genesis
    import genesis_b200.nn.functional as F
    kind = case["kind"]
    if kind == "orth":
        return [genesis.optim.orthogonalize(s["x"], steps=STEPS, coefficients=COEFFICIENTS, eps=EPS)._t]
    if kind == "muon":
        s["opt"].step()
        return [p._t for p in s["params"]] + [s["opt"].u[i] for i in range(len(s["params"]))]
    logits = s["logits"]
    logits.grad = None
    if kind == "logp":
        if not case["train"]:
            with genesis.no_grad():
                return [F.token_log_probs(logits, s["tokens"], temperature=case["temperature"])._t]
        lp = F.token_log_probs(logits, s["tokens"], temperature=case["temperature"])
        lp.backward(s["gy"])
        return [lp._t, logits.grad._t]
    if kind == "policy":
        loss = F.policy_loss(logits, s["tokens"], s["old"], s["adv"], s.get("ref"), clip=CLIP, clip_high=CLIP_HIGH,
                             kl_coef=KL if case["kl"] else 0.0)
        loss.backward()
        return [loss._t, logits.grad._t]
    loss, rewards = F.preference_loss(logits, s["tokens"], s["ref"], beta=BETA, label_smoothing=SMOOTH, return_rewards=True)
    loss.backward()
    return [loss._t, rewards._t, logits.grad._t]


# ------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ------------------------------------------------------------------------------------------------
def _orth_flops(count, rows, cols):
    """Two symmetric products (half of each is enough) and one full one a step, on the shorter side."""
    m, n = min(rows, cols), max(rows, cols)
    return count * STEPS * (m * (m + 1) * n + m * m * (m + 1) + 2 * m * m * n)


def work(case):
    kind, e = case["kind"], SIZE[case["dtype"]]
    if kind == "orth":
        n = case["count"] * case["rows"] * case["cols"]
        return dict(bytes=2 * n * e, flops=_orth_flops(case["count"], case["rows"], case["cols"]))
    if kind == "muon":
        sizes = _matrices(case)
        # the gradient is read, momentum and weight are read and written
        return dict(bytes=20 * sum(r * c for r, c in sizes), flops=sum(_orth_flops(1, r, c) for r, c in sizes))
    N, V = case["B"] * case["T"], case["V"]
    counted = sum(max(0, b - a) for a, b in _lengths(case))
    train = case.get("train", True)
    # a row that does not count is not read; its gradient, zeros, is written
    return dict(bytes=counted * V * e + (N * V * e if train else 0) + N * 24, flops=counted * V * (10 if train else 5))


# ------------------------------------------------------------------------------------------------
# the same from the definitions, in 64 bits
# ------------------------------------------------------------------------------------------------
def _exact_orth(x):
    """The iteration acts on the singular values alone: U p(p(...p(s))) V'.  Where a decomposition would take too long, the
    products themselves in 64 bits."""
    a, b, c = COEFFICIENTS
    if x.numel() * min(x.shape[-2:]) > 2e8:
        y = x.double() if x.shape[-2] <= x.shape[-1] else x.double().mT
        y = y / (torch.linalg.matrix_norm(y, keepdim=True) + EPS)
        for _ in range(STEPS):
            q = y @ y.mT
            y = torch.baddbmm(y, (c * (q @ q)).add_(q, alpha=b), y, beta=a) if y.dim() == 3 else a * y + (b * q + c * q @ q) @ y
        return y if x.shape[-2] <= x.shape[-1] else y.mT
    U, S, Vh = torch.linalg.svd(x.double(), full_matrices=False)
    t = S / (S.square().sum(-1, keepdim=True).sqrt() + EPS)
    for _ in range(STEPS):
        t = a * t + b * t ** 3 + c * t ** 5
    return (U * t.unsqueeze(-2)) @ Vh


def exact(case, seed):
    kind, d = case["kind"], _inputs(case, seed)
    if kind == "orth":
        return [_exact_orth(d["x"])]
    if kind == "muon":
        ws, us = [], []
        for w, g, u in zip(d["w"], d["g"], d["u"]):
            g, u = g.double(), MOMENTUM * u.double() + (1 - MOMENTUM) * g.double()
            o = _exact_orth((1 - MOMENTUM) * g + MOMENTUM * u)
            ws.append(w.double() * (1 - LR * DECAY) - LR * math.sqrt(max(1.0, w.shape[0] / w.shape[1])) * o)
            us.append(u)
        return ws + us
    B, T, V = d["logits"].shape
    temperature = case.get("temperature", 1.0)
    flat, tokens = d["logits"].view(B * T, V), d["tokens"].view(-1)
    valid = tokens >= 0
    lp = torch.where(valid, _log_probs64(flat, tokens.clamp(min=0), temperature), 0.0).view(B, T).requires_grad_()
    on = valid.view(B, T).double()
    if kind == "logp":
        outs = [lp.detach()]
        if not case["train"]:
            return outs
        g = d["gy"].double()
    else:
        if kind == "policy":
            adv = d["adv"].double() if case["per_token"] else d["adv"].double()[:, None]
            ratio = (lp - d["old"].double()).exp()
            each = -torch.minimum(adv * ratio, adv * ratio.clamp(1 - CLIP, 1 + CLIP_HIGH))
            if case["kl"]:
                k = d["ref"].double() - lp
                each = each + KL * (k.exp() - k - 1)
            loss = (each * on).sum() / on.sum().clamp(min=1)
            outs = [loss.detach()]
        else:
            rewards = BETA * (lp.sum(1) - d["ref"].double())
            h = rewards[:B // 2] - rewards[B // 2:]
            loss = -((1 - SMOOTH) * torch.nn.functional.logsigmoid(h) + SMOOTH * torch.nn.functional.logsigmoid(-h)).mean()
            outs = [loss.detach(), rewards.detach()]
        loss.backward()
        g = lp.grad
    # onto the logits: g (onehot - softmax) / temperature
    g = (g * on).view(-1, 1) / temperature
    grad = torch.empty(B * T, V, dtype=torch.float64, device=DEV)
    step = max(1, (1 << 27) // V)
    for a in range(0, B * T, step):
        p = torch.softmax(flat[a:a + step].double() / temperature, -1)
        p.scatter_add_(1, tokens[a:a + step].clamp(min=0)[:, None], torch.full((p.shape[0], 1), -1.0, dtype=torch.float64, device=DEV))
        grad[a:a + step] = p.mul_(-g[a:a + step])
    return outs + [grad.view(B, T, V)]
