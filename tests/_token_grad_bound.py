"""Bound of the gradient of logits that goes by each probability's own size."""
import math

import torch


def grad_near(got, z, tokens, row_factor, temperature=1.0, ignore=-100, what=""):
    """`got` [rows, V] against f ([j = t] - p), f = row_factor [rows] (the derivative by the row's log-probability over the
    temperature), 0 where ignored; everything in 64 bits, on got's device.

    With x = (z - max) log2(e) / T: the exponent x is off by the roundings of z - m, of its product (of log2(e) / T too in
    16-bit gradients, and of log2 s there, 2^-20 of up to 32), 2^-24 of |x| + 1 each (m may lie a factor of two below the
    maximum); the exponential by 2^-22; the sum by as much again, weighted by the probabilities; f and the products that
    make it by 6 * 2^-24.  One more rounding of 1 - p at the token, and the result's own."""
    rows, V = z.shape
    step = max(1, (1 << 26) // V)
    worst = 0.0
    for a in range(0, rows, step):
        d = z[a:a + step].to(got.device).double()
        t = tokens[a:a + step].to(got.device).long()
        on = t != ignore
        f = torch.where(on, row_factor[a:a + step].to(got.device).double(), 0.0)[:, None]
        p = torch.softmax(d / temperature, -1)
        x = (d.max(-1, keepdim=True).values - d) * (math.log2(math.e) / temperature) + 1
        mean = (p * x).sum(-1, keepdim=True)
        half = got.dtype != torch.float32
        one = (3 if half else 2) * math.log(2) * 2.0 ** -24
        shift = math.log(2) * (2.0 ** -20 + 2.0 ** -24 * 32) if half else 0.0
        rel = one * (x + mean) + 2 * 2.0 ** -22 + shift + 8 * 2.0 ** -24
        hot = torch.zeros_like(p).scatter_(1, torch.where(on, t, 0)[:, None], 1.0)
        want = torch.where(f == 0, 0.0, f * (hot - p))
        # (differences from -inf: probability 0, nothing to be off by)
        err = torch.where(p > 0, p * rel, 0.0)
        tol = want.abs() * (torch.finfo(got.dtype).eps / 2 + 8 * 2.0 ** -24) + f.abs() * (err + hot * 2.0 ** -24)
        # (the hardware exponential gives 0 for what is below 2^-126, the smallest normal number, and f multiplies that)
        tol = tol + f.abs() * 2.0 ** -126 + (2.0 ** -25 if got.dtype == torch.float16 else 2.0 ** -126)
        over = (got[a:a + step].double() - want).abs() - tol
        worst = max(worst, float(over.max()))
        bad = int((over > 0).sum())
        assert bad == 0, f"{what}: {bad} elements of rows {a}.. off, worst {worst:.3g} beyond the tolerance"
