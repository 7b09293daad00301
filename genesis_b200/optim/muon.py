"""Muon: momentum whose update is orthogonalised before it is applied, for the weight matrices of a model.

    u <- mu u + (1 - mu) g,   y = mu u + (1 - mu) g (Nesterov) or u,   o = orthogonalize(y)
    w <- w (1 - lr decay) - lr sqrt(max(1, rows / cols)) o

The orthogonalisation (`csrc/newton_schulz.cu`) works on all matrices of one shape, and its transpose, at once.  Vectors, embeddings and
output heads are left to AdamW: `Muon` takes tensors of two and more dimensions, whose last two are the matrix.
"""
import functools
import math

import torch

from .. import grad_mode
from ..ops import dispatch as K
from ..tensor import Tensor
from .optimizer import Optimizer

COEFFICIENTS = (3.4445, -4.7750, 2.0315)


@functools.lru_cache(maxsize=64)
def _exponents(steps, coefficients):
    """Powers of two [3 steps] by which X, A = X X^T and B = b A + c A A of every step are scaled before they are rounded to
    fp16 terms: the largest that keep their entries, which no singular value exceeds, below a quarter of fp16's range."""
    a, b, c = coefficients
    out, top = [], 1.001
    for _ in range(steps):
        s = torch.linspace(0.0, top, 4097, dtype=torch.float64)
        second = float((b * s ** 2 + c * s ** 4).abs().max())
        out += [math.floor(math.log2(16384.0 / max(x, 2.0 ** -10))) for x in (top, top * top, second)]
        top = 1.001 * float((a * s + b * s ** 3 + c * s ** 5).abs().max())
        if not top < 64.0 or second > 4096.0:
            raise ValueError(f"coefficients {coefficients} let singular values grow without bound")
        top = max(top, 2.0 ** -10)
    return tuple(out)


def _check(steps, coefficients, eps):
    if isinstance(steps, bool) or not isinstance(steps, int) or not 1 <= steps <= 64:
        raise ValueError(f"steps must be an int from 1 to 64, got {steps!r}")
    coefficients = tuple(float(x) for x in coefficients)
    if len(coefficients) != 3 or not all(map(math.isfinite, coefficients)):
        raise ValueError(f"coefficients must be three finite numbers, got {coefficients}")
    if not 1e-30 <= float(eps) < math.inf:
        raise ValueError(f"eps must be finite and at least 1e-30, got {eps}")
    return coefficients, float(eps), _exponents(steps, coefficients)


def orthogonalize(x, steps=5, coefficients=COEFFICIENTS, eps=1e-7):
    """Matrices of x [..., rows, cols] with their singular values driven to about one, in x's type.

    `steps` times X <- a X + (b A + c A A) X with A = X X^T, from X = x / (|x| + eps); a matrix with more rows than columns
    is handled as its transpose.  float16, bfloat16 and float32 are computed with the precision of float32.  Not
    differentiable.  A matrix that holds an Inf or NaN comes out as NaN; the others of a batch are not touched by it."""
    if not isinstance(x, Tensor) or not x._t.dtype.is_floating_point:
        raise TypeError("orthogonalize: x must be a floating-point Tensor")
    if x._t.dim() < 2:
        raise ValueError(f"orthogonalize: x must have two dimensions or more, got shape {tuple(x.shape)}")
    if x.requires_grad and grad_mode.is_grad_enabled():
        raise ValueError("orthogonalize is not differentiable: pass a detached Tensor, or call it under no_grad()")
    coefficients, eps, exponents = _check(steps, coefficients, eps)
    t = x._t
    if t.numel() == 0:
        return Tensor._wrap(torch.empty_like(t))
    out = K.newton_schulz(t.reshape(-1, *t.shape[-2:]), steps, coefficients, eps, exponents)
    return Tensor._wrap(out.reshape(t.shape))


class Muon(Optimizer):
    """Momentum with orthogonalised updates, for matrices; see the module's docstring."""

    _fused_amp = True       # the kernels take grad_scale / found_inf device scalars (see GradScaler.step)

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
        exponents = _exponents(self.steps, self.coefficients)
        groups = {}
        for i in idx:
            p, g = self.params[i]._t, self.params[i].grad._t
            if p.numel() == 0:
                continue
            if g.shape != p.shape or g.device != p.device:
                raise ValueError(f"gradient of shape {tuple(g.shape)} on {g.device} for a parameter of shape "
                                 f"{tuple(p.shape)} on {p.device}")
            members = groups.setdefault((tuple(sorted(p.shape[-2:])), g.dtype, p.device), [])
            g, u = K.contiguous(g), self._state(self.u, i)
            members += [((p, k), (g, k), (u, k)) for k in range(p.numel() // (p.shape[-2] * p.shape[-1]))]
        for (shape, _, _), members in groups.items():
            ps, gs, us = (list(x) for x in zip(*members))
            K.muon_step(ps, gs, us, shape, self.lr, self.momentum, self.nesterov, self.weight_decay,
                        math.sqrt(shape[1] / shape[0]), self.steps, self.coefficients, self.eps, exponents,
                        self._grad_scale, self._found_inf, self._dyn_lr_t)
        self._touched(idx)
