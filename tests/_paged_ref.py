"""Paged caches restated in 64 bits, a token at a time, and what a test has to build for a call."""
import math

import torch

import genesis_b200 as genesis
from genesis_b200.ops.paged import E4M3

TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16, "e4m3": E4M3}
# a rounding is off by at most half a step
HALF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def e4m3_values(x):
    """x [..., D] in 64 bits as the values that e4m3 numbers with a power of two for each row stand for."""
    fine = torch.isfinite(x)
    top = torch.where(fine, x.abs(), torch.zeros_like(x)).amax(-1, keepdim=True)
    e = torch.full_like(top, -126)
    while bool((top > 448 * torch.ldexp(torch.ones_like(e), e)).any()):
        e = torch.where(top > 448 * torch.ldexp(torch.ones_like(e), e), e + 1, e)
    y = torch.ldexp(torch.where(fine, x, torch.zeros_like(x)), -e)
    step = torch.ldexp(torch.ones_like(y), torch.frexp(y.abs().clamp(min=2.0 ** -6))[1] - 4)
    y = torch.ldexp(torch.round(y / step) * step, e)
    return torch.where(fine, y, torch.full_like(y, math.nan))


def held(x, dtype):
    """Numbers in 64 bits as a cache of `dtype` holds them."""
    return e4m3_values(x) if dtype == E4M3 else x.to(dtype).double()


def values(pool, scale):
    """A pool [pages, Hkv, page, D] as values in 64 bits."""
    x = pool.cpu().view(torch.uint8).view(E4M3).double() if pool.dtype == E4M3 else pool.cpu().double()
    if scale is None:
        return x
    s = scale.cpu().int()
    return torch.ldexp(x, (s - 127).unsqueeze(-1).double())


class Setup:
    """A cache with the given sequences in pages of random numbers; pages out of use and the ends of pages hold NaN."""

    def __init__(self, lengths, Hkv, D, cache="bf16", page=16, device="cpu", seed=0, spare=2, width=0, fill=True, value_scale=1.0):
        self.g = torch.Generator().manual_seed(seed)
        self.lengths, self.page, self.device = list(lengths), page, device
        need = [-(-max(n, 0) // page) for n in lengths]
        P = sum(need) + spare
        self.cache = genesis.nn.PagedKVCache(P, Hkv, D, page_size=page, dtype=str(TYPES[cache]).replace("torch.", ""), device=device)
        self.layer = self.cache[0]
        order = torch.randperm(P, generator=self.g).tolist()
        pages, at = [], 0
        for n in need:
            pages.append(order[at:at + n])
            at += n
        self.pages = pages
        self.table = self.cache.page_table(pages, width=max(max(need, default=0), width))
        self.lens = self.ints(lengths)
        # every place holds NaN (0x7f) until a sequence has it
        for pool, scale in ((self.layer.k, self.layer.k_scale), (self.layer.v, self.layer.v_scale)):
            if scale is None:
                pool.fill_(math.nan)
            else:
                pool.view(torch.uint8).fill_(0x7f)
                scale.fill_(127)
        self.kv = []
        for b, n in enumerate(lengths):
            n = max(n, 0)
            k, v = (torch.randn(n, Hkv, D, generator=self.g, dtype=torch.float64) * value_scale for _ in range(2))
            self.kv.append([held(k, TYPES[cache]) if n else k, held(v, TYPES[cache]) if n else v])
            if fill and n:
                p = torch.tensor(pages[b])[torch.arange(n) // page]
                for x, pool, scale in ((self.kv[b][0], self.layer.k, self.layer.k_scale), (self.kv[b][1], self.layer.v, self.layer.v_scale)):
                    self._place(pool, scale, p, torch.arange(n) % page, x)

    def _place(self, pool, scale, p, at, x):
        p, at = p.to(self.device), at.to(self.device)
        if scale is None:
            pool[p, :, at] = x.to(pool.dtype).to(self.device)
            return
        from genesis_b200.ops.paged import quantise
        y, e = quantise(x.float())
        pool.view(torch.uint8)[p, :, at] = y.view(torch.uint8).to(self.device)
        scale[p, :, at] = e.to(self.device)

    def ints(self, xs):
        return genesis.Tensor(torch.tensor(list(xs), dtype=torch.int32).reshape(len(list(xs))).to(self.device))

    def normal(self, *shape, dtype="bf16"):
        return torch.randn(*shape, generator=self.g).to(TYPES[dtype])

    def tensor(self, t):
        return genesis.Tensor(t.to(self.device))


def attention(q, kv, starts, counts, scale):
    """(o, sum p |v|, largest sum |q k| |scale| of a row) in 64 bits; kv: (k, v) [n, Hkv, D] for each sequence, starts: the
    position of its first query row."""
    B, S, Hq, D = q.shape
    o, size, reach = torch.zeros(B, S, Hq, D, dtype=torch.float64), torch.zeros(B, S, Hq, D, dtype=torch.float64), 0.0
    for b in range(B):
        for s in range(min(counts[b], S)):
            n = starts[b] + s + 1
            if n <= 0:
                continue
            k, v = kv[b][0][:n], kv[b][1][:n]
            g = Hq // k.shape[1]
            k, v = k.repeat_interleave(g, 1), v.repeat_interleave(g, 1)
            x = q[b, s].double()
            z = torch.einsum("hd,nhd->hn", x, k) * scale
            reach = max(reach, float(torch.einsum("hd,nhd->hn", x.abs(), k.abs()).max()) * abs(scale))
            p = torch.softmax(z, -1)
            o[b, s], size[b, s] = torch.einsum("hn,nhd->hd", p, v), torch.einsum("hn,nhd->hd", p, v.abs())
    return o, size, reach


def tolerance(q, o, size, reach, keys, cache):
    """How far a kernel that works in 32 bits may be off, number by number.

    Scores: products of D numbers summed in 32 bits, each addition off by at most 2^-23 of what the sum of magnitudes is (tensor
    cores cut off instead of rounding), the scale and the maximum taken off once each: d = (D + 4) 2^-23 reach.  exp turns that
    into a relative error of each probability, its own is 2^-21 (the exponent's rounding: 2^-24 times up to 2 log2(e) reach).
    Probabilities enter the second product as two 16-bit numbers (2^-17 at most of each), or as one of 11 bits where the
    values are held in 8 bits and the output has 8 (2^-12).  Sums over the keys: as above, 2^-23 for every addition of a
    32-bit accumulator, for the product and for the normaliser; parts are joined with as many roundings as there are parts."""
    t, D = q.dtype, q.shape[-1]
    rel = (D + 8) * 2.0 ** -23 * reach + 2.0 ** -20 + (2 * min(keys, 4096) + 64) * 2.0 ** -23
    if t != torch.float32 or cache == "e4m3":
        rel += 2.0 ** -12 if cache == "e4m3" and t == torch.bfloat16 else 2.0 ** -17
    return HALF[t] * o.abs() + (rel + rel * HALF[t]) * size * 2 + 2.0 ** -24 * (t == torch.float16)
