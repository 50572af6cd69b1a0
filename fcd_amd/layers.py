"""Layer norm and dropout as differentiable functions and modules over the HIP kernels.

``layer_norm`` is one node: norm over the last axis, activation, dropout and residual add in one launch.  Its backward is a
node as well, so a gradient penalty (``autograd.grad(..., create_graph=True)``) can differentiate the input gradient again;
differentiating the parameters' gradients is refused.  Dropout masks are recomputed from ``rng`` and never stored.  No
reference counterpart: the reference's networks have neither.

Capturing a backward pass into a HIP graph: let go of eager graphs over the same parameters first (as for any torch module).
A forward pass that is run a second time (activation checkpointing) draws a new range of a module's generator, so its backward
would belong to another mask: there call the functions, with an ``rng`` taken outside the part that is run again.
"""
from __future__ import annotations

from typing import Optional

import torch
import torch.distributed as dist
import torch.nn as nn
from torch.autograd.function import once_differentiable

from . import ops
from .generator import _act_slope


def _even(t: torch.Tensor) -> torch.Tensor:
    """``t`` itself if its rows are evenly spaced, else a contiguous copy (gradients of sums and slices)."""
    try:
        ops._rows(t, "x")
        return t
    except RuntimeError:
        return t.contiguous()


def _words(rng):
    """(tensor, rest) of an ``rng``: its tensor is saved for the backward pass like an operand, so that autograd refuses one that
    has changed by then."""
    if isinstance(rng, torch.Tensor):
        return rng, None
    return tuple(rng) if rng is not None and isinstance(rng[0], torch.Tensor) else (None, rng)


def _rng(words, rest):
    return rest if words is None else words if rest is None else (words, rest)


class _LayerNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, eps, act, p, rng):
        y, mean, rstd = ops.layernorm_fwd(_even(x), weight, bias, eps, act, p, rng, None if residual is None else _even(residual))
        words, rest = _words(rng)
        ctx.save_for_backward(x, weight, bias, mean, rstd, words)      # (x itself, not a copy: the second backward leads to it)
        ctx.cfg = act, p, rest
        ctx.set_materialize_grads(False)
        return y

    @staticmethod
    def backward(ctx, gy):
        if gy is None:
            return (None,) * 8
        x, weight, bias, mean, rstd, words = ctx.saved_tensors
        act, p, rest = ctx.cfg
        needs = ctx.needs_input_grad
        dx = dw = db = None
        if any(needs[:3]):
            dx, dw, db = _LayerNormBwdFn.apply(gy, x, weight, bias, mean, rstd, (act, p, _rng(words, rest)), bool(needs[1] or needs[2]))
        return (dx if needs[0] else None, dw if needs[1] else None, db if needs[2] else None, gy if needs[3] else None,
                None, None, None, None)


class _LayerNormBwdFn(torch.autograd.Function):
    """(gy, x, weight, bias) -> (dx, dweight, dbias): the first-order backward as a node."""

    @staticmethod
    def forward(ctx, gy, x, weight, bias, mean, rstd, cfg, want_affine):
        gy, x = _even(gy), _even(x)
        act, p, rng = cfg
        words, rest = _words(rng)
        ctx.save_for_backward(gy, x, weight, bias, mean, rstd, words)
        ctx.cfg = act, p, rest
        ctx.set_materialize_grads(False)
        return ops.layernorm_bwd(gy, x, mean, rstd, weight, bias, act, p, rng, want_affine=want_affine)

    @staticmethod
    @once_differentiable
    def backward(ctx, ggx, ggw, ggb):
        if ggw is not None or ggb is not None:
            raise NotImplementedError("differentiating through a layer norm's parameter gradients is not supported")
        if ggx is None:
            return (None,) * 8
        gy, x, weight, bias, mean, rstd, words = ctx.saved_tensors
        act, p, rest = ctx.cfg
        needs = ctx.needs_input_grad
        ggy, gx, dw, db = ops.layernorm_bwd2(_even(ggx), gy, x, mean, rstd, weight, bias, act, p, _rng(words, rest),
                                             want_affine=bool(needs[2] or needs[3]))
        return ggy, gx, dw if needs[2] else None, db if needs[3] else None, None, None, None, None


class _DropoutFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, p, rng, residual):
        words, rest = _words(rng)
        ctx.save_for_backward(words)
        ctx.cfg = p, rest
        return ops.dropout(_even(x), p, rng, None if residual is None else _even(residual))

    @staticmethod
    def backward(ctx, gy):
        p, rest = ctx.cfg
        needs = ctx.needs_input_grad
        rng = _rng(ctx.saved_tensors[0], rest)
        return _DropoutFn.apply(gy, p, rng, None) if needs[0] else None, None, None, gy if needs[3] else None


def _code(activation: Optional[str]) -> float:
    return 1.0 if activation is None else _act_slope(activation)


def layer_norm(x, weight=None, bias=None, eps: float = ops.LN_EPS, activation: Optional[str] = None, p: float = 0.0, rng=None,
               residual=None):
    """``dropout(act((x - mean) * rstd * weight + bias)) (+ residual)`` over the last axis; float32, bfloat16 or float16,
    weight / bias float32 or x's type or None.  ``activation``: None, relu, lrelu, silu, mish; ``rng``: see :func:`dropout`."""
    return _LayerNormFn.apply(x, weight, bias, residual, eps, _code(activation), float(p), rng)


def dropout(x, p: float, rng, residual=None):
    """``x * mask / (1 - p) (+ residual)``.  ``rng``: ``(seed, offset)``, what ``ops.dropout_take`` returned, or that with an
    offset in blocks of 8 elements to add, ``(taken, offset)``."""
    return _DropoutFn.apply(x, float(p), rng, residual)


RANK_BLOCKS = 1 << 48     # generator blocks per rank of a data-parallel job: ranks that share a seed draw other masks


def rank_offset() -> int:
    return RANK_BLOCKS * dist.get_rank() if dist.is_available() and dist.is_initialized() else 0


class _Drops(nn.Module):
    """Dropout probability and the generator's state (a buffer: it moves with the module and resumes from a checkpoint).

    Without a seed a module draws one from torch's CPU generator, so every module has masks of its own and ``manual_seed``
    brings them back.  Modules that are given one seed, and copies of a module, draw the same blocks: the same masks, for equal
    shapes."""

    def __init__(self, p: float):
        super().__init__()
        if not 0.0 <= p <= 1.0:
            raise ValueError(f"dropout probability {p} is not in [0, 1]")
        self.p = float(p)

    def _start(self, seed: Optional[int]) -> None:
        if self.p == 0.0:
            return
        if seed is None:
            seed = int(torch.empty((), dtype=torch.int64, device="cpu").random_())
        self.register_buffer("dropout_state", ops.dropout_state(seed, "cpu"))

    def _draw(self, numel: int):
        """(p, rng) of this call."""
        if not self.training or self.p == 0.0:
            return 0.0, None
        return self.p, (ops.dropout_take(self.dropout_state, numel), rank_offset())


class Dropout(_Drops):
    """Dropout whose mask is recomputed in the backward pass; the identity in eval mode."""

    def __init__(self, p: float = 0.5, seed: Optional[int] = None):
        super().__init__(p)
        self._start(seed)

    def forward(self, x, residual=None):
        p, rng = self._draw(x.numel())
        return x if p == 0.0 and residual is None else dropout(x, p, rng, residual)


class LayerNorm(_Drops):
    """Layer norm over the last axis of size ``dim`` with a fused activation, dropout (training mode) and residual add."""

    def __init__(self, dim: int, eps: float = ops.LN_EPS, affine: bool = True, bias: bool = True,
                 activation: Optional[str] = None, dropout: float = 0.0, seed: Optional[int] = None):
        super().__init__(dropout)
        _code(activation)
        self._start(seed)
        self.dim, self.eps, self.activation = int(dim), float(eps), activation
        self.weight = nn.Parameter(torch.ones(dim)) if affine else None
        self.bias = nn.Parameter(torch.zeros(dim)) if affine and bias else None

    def forward(self, x, residual=None):
        if x.shape[-1] != self.dim:
            raise RuntimeError(f"LayerNorm: last axis of {x.shape[-1]}, expected {self.dim}")
        p, rng = self._draw(x.numel())
        return layer_norm(x, self.weight, self.bias, self.eps, self.activation, p, rng, residual)
