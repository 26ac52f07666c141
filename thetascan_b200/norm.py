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

import ctypes
from typing import Optional

import torch
from torch import Tensor

from . import _lib

LIB = "thetascan_b200"
GROUP = 128
_DTYPES = {torch.float32: _lib.TS_DTYPE_F32, torch.bfloat16: _lib.TS_DTYPE_BF16}


def _check(x, weight, eps, residual=None):
    for name, t in (("x", x), ("weight", weight), ("residual", residual)):
        if t is None:
            continue
        if not t.is_cuda:
            raise RuntimeError("b200 backend requires CUDA tensors")
        if t.dtype not in _DTYPES:
            raise ValueError(f"{name} must be float32 or bfloat16, got {t.dtype}")
        if t.device != x.device:
            raise ValueError(f"{name} is on {t.device}, x on {x.device}")
    if x.ndim < 1 or weight.ndim != 1 or weight.shape[0] != x.shape[-1]:
        raise ValueError(f"weight {tuple(weight.shape)} does not match the last dimension of x {tuple(x.shape)}")
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype):
        raise ValueError(f"residual must have the shape and dtype of x ({tuple(x.shape)}, {x.dtype}), got "
                         f"{tuple(residual.shape)}, {residual.dtype}")
    if not eps >= 0:
        raise ValueError(f"eps must be >= 0, got {eps}")


def _rows(t):
    """``t [..., width]`` as rows ``[n, width]`` with contiguous channels: a
    view where the strides allow one, else a copy."""
    t2 = t.reshape(-1, t.shape[-1])
    return t2 if t2.stride(1) == 1 or t2.shape[1] == 1 else t2.contiguous()


def _args(x2, weight, eps):
    a = _lib.NormArgs()
    a.rows, a.width = x2.shape
    a.dtype, a.weight_dtype, a.eps = _DTYPES[x2.dtype], _DTYPES[weight.dtype], eps
    a.x, a.x_stride, a.weight = x2.data_ptr(), x2.stride(0), weight.data_ptr()
    return a


def _norm_fwd_impl(x, residual, weight, eps, need_rstd):
    """(y, stored sum or an empty tensor, rstd or an empty tensor)."""
    with _lib.on_device(x):
        y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        total = torch.empty(x.shape if residual is not None else 0, dtype=x.dtype, device=x.device)
        rows = x.numel() // x.shape[-1] if x.shape[-1] else 0
        rstd = torch.empty(rows if need_rstd else 0, dtype=torch.float32, device=x.device)
        if x.numel():
            x2, weight = _rows(x), weight.contiguous()
            a = _args(x2, weight, eps)
            a.y, a.rstd = y.data_ptr(), rstd.data_ptr() if need_rstd else None
            if residual is not None:
                r2 = _rows(residual)
                a.residual, a.residual_stride, a.sum = r2.data_ptr(), r2.stride(0), total.data_ptr()
            _lib.check(_lib.load().ts_b200_norm_fwd(ctypes.byref(a), _lib.stream()))
        return y, total, rstd


def _norm_bwd_impl(dy, dsum, total, weight, rstd, eps):
    """(dx, dweight): dx is the gradient of x and of the residual."""
    with _lib.on_device(total):
        dx = torch.empty(total.shape, dtype=total.dtype, device=total.device)
        dweight = torch.empty(weight.shape, dtype=weight.dtype, device=weight.device)
        if not total.numel():
            return dx, dweight.zero_()
        lib = _lib.load()
        x2, weight, dy2 = _rows(total), weight.contiguous(), _rows(dy)
        a = _args(x2, weight, eps)
        a.rstd = rstd.data_ptr()
        g = _lib.NormGradArgs()
        g.dy, g.dy_stride = dy2.data_ptr(), dy2.stride(0)
        if dsum is not None:
            ds2 = _rows(dsum)
            g.dsum, g.dsum_stride = ds2.data_ptr(), ds2.stride(0)
        nbytes = lib.ts_b200_norm_bwd_workspace_bytes(ctypes.byref(a))
        ws = torch.empty(nbytes, dtype=torch.uint8, device=total.device)
        g.dx, g.dweight, g.workspace, g.workspace_bytes = dx.data_ptr(), dweight.data_ptr(), ws.data_ptr(), nbytes
        _lib.check(lib.ts_b200_norm_bwd(ctypes.byref(a), ctypes.byref(g), _lib.stream()))
        return dx, dweight


@torch.library.custom_op(f"{LIB}::norm_fwd", mutates_args=())
def norm_fwd(x: Tensor, residual: Optional[Tensor], weight: Tensor, eps: float,
             need_rstd: bool) -> tuple[Tensor, Tensor, Tensor]:
    """The norm, the stored sum (empty without a residual) and rstd (empty unless asked for)."""
    return _norm_fwd_impl(x, residual, weight, eps, need_rstd)


@norm_fwd.register_fake
def _(x, residual, weight, eps, need_rstd):
    return (x.new_empty(x.shape), x.new_empty(x.shape if residual is not None else (0,)),
            x.new_empty(x.numel() // x.shape[-1] if need_rstd else 0, dtype=torch.float32))


@torch.library.custom_op(f"{LIB}::norm_bwd", mutates_args=())
def norm_bwd(dy: Tensor, dsum: Optional[Tensor], total: Tensor, weight: Tensor, rstd: Tensor,
             eps: float) -> tuple[Tensor, Tensor]:
    return _norm_bwd_impl(dy, dsum, total, weight, rstd, eps)


@norm_bwd.register_fake
def _(dy, dsum, total, weight, rstd, eps):
    return total.new_empty(total.shape), weight.new_empty(weight.shape)


class _Norm(torch.autograd.Function):
    """Autograd of the norm.  The kernels are called directly in eager mode;
    a tracing compiler sees the custom ops (whose dispatch costs the host more)."""

    @staticmethod
    def forward(ctx, x, residual, weight, eps):
        fwd = norm_fwd if torch.compiler.is_compiling() else _norm_fwd_impl
        y, total, rstd = fwd(x, residual, weight, eps, True)
        ctx.eps, ctx.added = eps, residual is not None
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(total if ctx.added else x, weight, rstd)
        return (y, total) if ctx.added else y

    @staticmethod
    def backward(ctx, dy, dsum=None):
        total, weight, rstd = ctx.saved_tensors
        if dy is None:
            return dsum, dsum if ctx.added else None, None, None
        bwd = norm_bwd if torch.compiler.is_compiling() else _norm_bwd_impl
        dx, dweight = bwd(dy, dsum, total, weight, rstd, ctx.eps)
        return dx, dx if ctx.added else None, dweight, None


def _norm(x, residual, weight, eps):
    _check(x, weight, eps, residual)
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad
                                    or (residual is not None and residual.requires_grad)):
        return _Norm.apply(x, residual, weight, float(eps))
    fwd = norm_fwd if torch.compiler.is_compiling() else _norm_fwd_impl
    y, total, _ = fwd(x, residual, weight, float(eps), False)
    return y if residual is None else (y, total)


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
    stored sum too where there is a residual.  For inference: no gradient."""
    _check(x, weight, eps, residual)
    if group not in (None, GROUP):
        raise ValueError(f"group must be None (one scale per row) or {GROUP}, got {group}")
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad
                                    or (residual is not None and residual.requires_grad)):
        raise RuntimeError("rms_norm_8bit has no gradient: call it under torch.no_grad()")
    with _lib.on_device(x):
        n_scales = -(-x.shape[-1] // GROUP) if group else 1
        codes = torch.empty(x.shape, dtype=torch.float8_e4m3fn, device=x.device)
        scales = torch.empty(*x.shape[:-1], n_scales, dtype=torch.float32, device=x.device)
        total = torch.empty(x.shape, dtype=x.dtype, device=x.device) if residual is not None else None
        if x.numel():
            x2, weight = _rows(x), weight.contiguous()
            a = _args(x2, weight, eps)
            a.y, a.scales, a.group = codes.data_ptr(), scales.data_ptr(), group or 0
            if residual is not None:
                r2 = _rows(residual)
                a.residual, a.residual_stride, a.sum = r2.data_ptr(), r2.stride(0), total.data_ptr()
            _lib.check(_lib.load().ts_b200_norm_fwd(ctypes.byref(a), _lib.stream()))
        return (codes, scales) if residual is None else (codes, scales, total)
