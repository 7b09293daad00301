"""Muon: momentum whose update is orthogonalised before it is applied, for the weight matrices of a model.

    u <- mu u + (1 - mu) g,   y = mu u + (1 - mu) g (Nesterov) or u,   o = orthogonalize(y)
    w <- w (1 - lr decay) - lr sqrt(max(1, rows / cols)) o

The orthogonalisation (`csrc/newton_schulz.cu`) works on all matrices of one shape, and its transpose, at once.  Vectors, embeddings and
output heads are left to AdamW: `Muon` takes tensors of two and more dimensions, whose last two are the matrix.

On CUDA, contiguous weights in 32 bits take the kernels, with gradients of any floating-point type of up to 32 bits.  Other weights
(16-bit or 64-bit ones, transposed views) are updated by library products, one matrix at a time, and not in a captured step.
A call holds workspace: for m x n matrices, m <= n, 12 bytes for each of m n elements (16 in an optimizer's step) and 40 for each of
m m, for as many matrices at a time as make up 4 GB, or one (8192 x 8192: 3.5 GB, 3.8 in a step).  `Muon` keeps no low-precision
copies of its weights (`enable_shadows` of AdamW); autocast converts them in every step.
"""
import ctypes
import functools
import math

import torch

from .. import grad_mode
from ..ops import dispatch as K
from ..tensor import Tensor
from .optimizer import Optimizer

COEFFICIENTS = (3.4445, -4.7750, 2.0315)


# slots of m x m matrices in the kernels' workspace
_A, _W, _B, _Q = 0, 1, 2, (3, 4)


@functools.lru_cache(maxsize=64)
def _program(steps, coefficients, longest=3):
    """The products that `gb_newton_schulz` makes, as an array of 12 numbers each (see there and the head of
    `csrc/newton_schulz.cu`).

    Steps go one by one (`longest` 1), or in blocks of three, or two, between which X is formed anew.  Every matrix is a polynomial in X X^T, so its
    eigenvalues are followed over all singular values that X may have; the power of two by which its terms are scaled in
    fp16 is the largest that keeps its entries, which no eigenvalue exceeds, below a quarter of fp16's range."""
    a, b, c = coefficients
    rows, top, left = [], 1.001, steps

    def scale(values):
        peak = float(values.abs().max())
        if not peak < 4096.0:
            raise ValueError(f"coefficients {coefficients} let singular values grow without bound")
        return 2.0 ** math.floor(math.log2(16384.0 / max(peak, 2.0 ** -10)))

    def row(kind, lhs, rhs, out, f_acc, out_scale, m1=-1, f1=0.0, m2=-1, f2=0.0, keep=True):
        rows.append([kind, lhs, rhs, out, m1, m2, float(keep), f_acc, f1, f2, out_scale, 0.0])

    while left:
        block = min(longest, left if left < 4 else 2 if left == 4 else 3)
        left -= block
        s = torch.linspace(0.0, top, 4097, dtype=torch.float64)
        x_scale = scale(s)
        lam = s * s
        total = torch.ones_like(s)                       # product of the P's: identity * ident + Q
        scales, ident, q, old_q = {_A: scale(lam)}, 1.0, _Q[0], None
        if rows:
            rows[-1][10] = x_scale                       # the X that the block before has left
        else:
            first = x_scale
        row(0, 0, 0, _A, x_scale ** -2, scales[_A])
        for k in range(block):
            B = b * lam + c * lam * lam
            slot = q if k == 0 else _B
            scales[slot] = scale(B)
            last = k + 1 == block                        # (whose Q goes on to X as terms alone: no 32-bit copy of it)
            row(1, _A, _A, slot, c / scales[_A] ** 2, scales[slot], _A, b, keep=k > 0 or not last)
            if not last:
                scales[_W] = scale((a + B) * lam)
                row(2 if k else 1, slot, _A, _W, 1.0 / (scales[slot] * scales[_A]), scales[_W], _A, a)
            new = total * (a + B)
            if k:
                old_q, q = q, _Q[1 - _Q.index(q)]
                scales[q] = scale(new - ident * a)
                row(1, _B, old_q, q, 1.0 / (scales[_B] * scales[old_q]), scales[q], old_q, a, _B, ident, keep=not last)
            total, ident = new, ident * a
            if not last:
                lam = lam * (a + B) ** 2
                scales[_A] = scale(lam)
                row(1, slot, _W, _A, 1.0 / (scales[slot] * scales[_W]), scales[_A], _W, a)
        row(3, q, 0, 0, 1.0 / (scales[q] * x_scale), 1.0, f1=ident)
        top = max(1.001 * float((s * total).abs().max()), 2.0 ** -10)
    rows[0][11] = first
    flat = [x for r in rows for x in r]
    return (ctypes.c_double * len(flat))(*flat)


def _programs(steps, coefficients):
    return _program(steps, coefficients), _program(steps, coefficients, 1)


def _check(steps, coefficients, eps):
    if isinstance(steps, bool) or not isinstance(steps, int) or not 1 <= steps <= 64:
        raise ValueError(f"steps must be an int from 1 to 64, got {steps!r}")
    coefficients = tuple(float(x) for x in coefficients)
    if len(coefficients) != 3 or not all(map(math.isfinite, coefficients)):
        raise ValueError(f"coefficients must be three finite numbers, got {coefficients}")
    if not 1e-30 <= float(eps) < math.inf:
        raise ValueError(f"eps must be finite and at least 1e-30, got {eps}")
    return coefficients, float(eps), _programs(steps, coefficients)


def orthogonalize(x, steps=5, coefficients=COEFFICIENTS, eps=1e-7):
    """Matrices of x [..., rows, cols] with their singular values driven to about one, in x's type.

    `steps` times X <- a X + (b A + c A A) X with A = X X^T, from X = x / (|x| + eps); a matrix with more rows than columns
    is handled as its transpose.  Whatever the type, products have 22-bit operands and sums 32 bits; on CUDA the result is
    some 1e-6 to 4e-5 of its norm off, before it is rounded to x's type: about as far as 32-bit products; up to six times as far
    where long or many matrices of more than 320 rows, which take the steps in blocks, have no strong directions.  Not differentiable.  A matrix that holds an Inf or
    NaN comes out as NaN; the others of a batch are not touched by it."""
    if not isinstance(x, Tensor) or not x._t.dtype.is_floating_point:
        raise TypeError("orthogonalize: x must be a floating-point Tensor")
    if x._t.dim() < 2:
        raise ValueError(f"orthogonalize: x must have two dimensions or more, got shape {tuple(x.shape)}")
    if x.requires_grad and grad_mode.is_grad_enabled():
        raise ValueError("orthogonalize is not differentiable: pass a detached Tensor, or call it under no_grad()")
    coefficients, eps, program = _check(steps, coefficients, eps)
    t = x._t
    if t.numel() == 0:
        return Tensor._wrap(torch.empty_like(t))
    out = K.newton_schulz(t.reshape(-1, *t.shape[-2:]), steps, coefficients, eps, program)
    return Tensor._wrap(out.reshape(t.shape))


class Muon(Optimizer):
    """Momentum with orthogonalised updates, for matrices; see the module's docstring."""

    _fused_amp = True       # the kernels take grad_scale / found_inf device scalars (see GradScaler.step)
    _state_stays = True

    def __init__(self, params, lr=0.02, momentum=0.95, nesterov=True, weight_decay=0.0, steps=5, coefficients=COEFFICIENTS,
                 eps=1e-7):
        super().__init__(params)
        for p in self.params:
            if p._t.dim() < 2 or not p._t.dtype.is_floating_point:
                raise ValueError(f"Muon takes floating-point matrices; give a parameter of shape {tuple(p.shape)} and type "
                                 f"{p._t.dtype} to another optimizer")
        if len({id(p) for p in self.params}) != len(self.params):
            raise ValueError("a parameter is listed twice")
        if not 0.0 <= float(momentum) < 1.0:
            raise ValueError(f"momentum must be in [0, 1), got {momentum}")
        self.coefficients, self.eps, _ = _check(steps, coefficients, eps)
        self.lr, self.momentum, self.nesterov, self.weight_decay, self.steps = lr, momentum, nesterov, weight_decay, steps
        self.t = 0
        self.u = {}
        self._dyn_lr_t = None       # the learning rate on the device, for steps that are replayed from a CUDA graph
        self._dyn_lr = None

    def make_capturable(self):
        """Move the learning rate to the device. Idempotent; needs CUDA parameters."""
        if self._dyn_lr_t is None:
            dev = self.params[0]._t.device
            if dev.type != "cuda":
                raise RuntimeError("capturable optimizer state needs CUDA parameters")
            self._dyn_lr_t = torch.tensor([self.lr], dtype=torch.float32, device=dev)
            self._dyn_lr = self.lr
        return self

    def _sync_lr(self):
        """Write a changed host learning rate to the device (outside a capture)."""
        if self._dyn_lr_t is not None and self._dyn_lr != self.lr:
            self._dyn_lr_t.fill_(float(self.lr))
            self._dyn_lr = self.lr

    def load_state_dict(self, state_dict):
        super().load_state_dict(state_dict)
        self.coefficients = tuple(self.coefficients)
        self._sync_lr()

    def step(self):
        idx = self._active()
        if not idx:
            return
        if self._found_inf is not None and not self.params[idx[0]]._t.is_cuda and float(self._found_inf.item()) != 0.0:
            return                                # cancelled step (host tensors: the flag is read here)
        # gradients that a data-parallel wrapper left in flight
        for join in {id(f): f for f in (getattr(self.params[i], "_late_join", None) for i in idx) if f is not None}.values():
            join()
        self.t += 1
        if self._dyn_lr_t is not None and not torch.cuda.is_current_stream_capturing():
            self._sync_lr()
        program = _programs(self.steps, self.coefficients)
        groups = {}
        for i in idx:
            p, g = self.params[i]._t, self.params[i].grad._t
            if p.numel() == 0:
                continue
            if g.shape != p.shape or g.device != p.device:
                raise ValueError(f"gradient of shape {tuple(g.shape)} on {g.device} for a parameter of shape "
                                 f"{tuple(p.shape)} on {p.device}")
            # (the type and layout of the weight too: those that the kernels do not take must not keep others from them)
            key = (tuple(sorted(p.shape[-2:])), g.dtype, p.device, p.dtype, p.is_contiguous())
            members = groups.setdefault(key, [])
            g, u = K.contiguous(g), self._state(self.u, i)
            members += [((p, k), (g, k), (u, k)) for k in range(p.numel() // (p.shape[-2] * p.shape[-1]))]
        for (shape, _, dev, *_), members in groups.items():
            ps, gs, us = (list(x) for x in zip(*members))
            # (a kernel reads these on its own device)
            scalars = [s if s is None or s.device == dev else s.to(dev)
                       for s in (self._grad_scale, self._found_inf, self._dyn_lr_t)]
            K.muon_step(ps, gs, us, shape, self.lr, self.momentum, self.nesterov, self.weight_decay,
                        math.sqrt(shape[1] / shape[0]), self.steps, self.coefficients, self.eps, program, *scalars)
        self._touched(idx)
