"""Root-mean-square norm with the residual's addition, and its 8-bit output.

The norms around a mixer in a residual block (the reference leaves them to its
host model):

* :func:`rms_norm` -- ``y = x * rstd * weight``, ``rstd = (mean x^2 + eps)^-1/2``;
* :func:`add_rms_norm` -- ``s = x + residual``, rounded to its type as the
  residual stream is stored, and the norm of that ``s``; both are returned;
* :func:`rms_norm_8bit` -- the norm (with or without a residual) as e4m3 codes
  and f32 scales, for an 8-bit product; no gradient.

One kernel each way over the rows (``csrc/norm.cu``).  bf16 or f32 streams, a
weight in f32 or bf16, any leading dimensions and row strides, any width up to
16384.  Sums and statistics are f32.
"""
from __future__ import annotations

from typing import Optional

import torch
from torch import Tensor

from . import _lib

LIB = "thetascan_b200"


@torch.library.custom_op(f"{LIB}::norm_fwd", mutates_args=())
def norm_fwd(x: Tensor, residual: Optional[Tensor], weight: Tensor, eps: float,
             keep: bool) -> tuple[Tensor, Tensor, Tensor]:
    """The norm, the stored sum (empty without a residual) and rstd (empty unless ``keep``)."""
    y, total, rstd = _lib.host().norm_fwd(x, residual, weight, eps, keep)
    return (y, x.new_empty(0) if total is None else total,
            x.new_empty(0, dtype=torch.float32) if rstd is None else rstd)


@norm_fwd.register_fake
def _(x, residual, weight, eps, keep):
    return (x.new_empty(x.shape), x.new_empty(x.shape if residual is not None else (0,)),
            x.new_empty(x.numel() // x.shape[-1] if keep else 0, dtype=torch.float32))


@torch.library.custom_op(f"{LIB}::norm_bwd", mutates_args=())
def norm_bwd(dy: Tensor, dsum: Optional[Tensor], total: Tensor, weight: Tensor, rstd: Tensor,
             eps: float) -> tuple[Tensor, Tensor]:
    """Gradients of the sum's terms (one tensor for both) and of the weight."""
    return _lib.host().norm_bwd(dy, dsum, total, weight, rstd, eps)


@norm_bwd.register_fake
def _(dy, dsum, total, weight, rstd, eps):
    return total.new_empty(total.shape), weight.new_empty(weight.shape)


@torch.library.custom_op(f"{LIB}::norm_8bit", mutates_args=())
def norm_8bit(x: Tensor, residual: Optional[Tensor], weight: Tensor, eps: float,
              group: Optional[int]) -> tuple[Tensor, Tensor, Tensor]:
    """The norm's codes and scales, and the stored sum (empty without a residual)."""
    codes, scales, *total = _lib.host().rms_norm_8bit(x, residual, weight, eps, group)
    return codes, scales, *(total or [x.new_empty(0)])


@norm_8bit.register_fake
def _(x, residual, weight, eps, group):
    n = 1 if group is None else -(-x.shape[-1] // group)
    return (x.new_empty(x.shape, dtype=torch.float8_e4m3fn), x.new_empty((*x.shape[:-1], n), dtype=torch.float32),
            x.new_empty(x.shape if residual is not None else (0,)))


class _TracedNorm(torch.autograd.Function):
    """The autograd node as a tracing compiler sees it; eager calls have theirs in ``csrc/host.cpp``."""

    @staticmethod
    def forward(ctx, x, residual, weight, eps):
        y, total, rstd = norm_fwd(x, residual, weight, eps, True)
        ctx.eps, ctx.added = eps, residual is not None
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(total if ctx.added else x, weight, rstd)
        return (y, total) if ctx.added else y

    @staticmethod
    def backward(ctx, dy, dsum=None):
        total, weight, rstd = ctx.saved_tensors
        if dy is None:
            return dsum, dsum if ctx.added else None, None, None
        dx, dweight = norm_bwd(dy, dsum, total, weight, rstd, ctx.eps)
        return dx, dx if ctx.added else None, dweight, None


def _wants_grad(*tensors):
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def _norm(x, residual, weight, eps):
    if torch.compiler.is_compiling():
        if _wants_grad(x, residual, weight):
            return _TracedNorm.apply(x, residual, weight, float(eps))
        y, total, _ = norm_fwd(x, residual, weight, float(eps), False)
        return y if residual is None else (y, total)
    return _lib.host().rms_norm(x, residual, weight, eps)


def rms_norm(x: Tensor, weight: Tensor, eps: float = 1e-6) -> Tensor:
    """``x * (mean(x^2) + eps)^-1/2 * weight`` over the last dimension, in the type of ``x``."""
    return _norm(x, None, weight, eps)


def add_rms_norm(x: Tensor, residual: Tensor, weight: Tensor, eps: float = 1e-6) -> tuple[Tensor, Tensor]:
    """``s = x + residual`` rounded to their type, and ``rms_norm(s)``: returns ``(norm, s)``."""
    return _norm(x, residual, weight, eps)


def rms_norm_8bit(x: Tensor, weight: Tensor, eps: float = 1e-6, *, residual: Optional[Tensor] = None,
                  group: Optional[int] = None):
    """The norm as ``torch.float8_e4m3fn`` codes and f32 scales (the norm is
    ``codes * scales``): one scale per row (``group=None``) or per 128 columns
    (``group=128``), shape ``[..., n_scales]``.  Each scale maps the largest
    magnitude that it covers to 448, the type's largest value; the norm is
    rounded once, from f32 to the code.  Returns ``(codes, scales)``, and the
    stored sum too where there is a residual.  A NaN makes its scale NaN and
    with it all codes under that scale.  For inference: no gradient."""
    if torch.compiler.is_compiling():
        if _wants_grad(x, residual, weight):
            raise RuntimeError("rms_norm_8bit has no gradient: call it under torch.no_grad()")
        codes, scales, total = norm_8bit(x, residual, weight, float(eps), group)
        return (codes, scales) if residual is None else (codes, scales, total)
    return _lib.host().rms_norm_8bit(x, residual, weight, eps, group)
