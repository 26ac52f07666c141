"""The gated feed-forward block ``y = (act(x Wg^T) * (x Wu^T)) Wd^T``.

* :func:`gated_ffn` -- the function, with its gradients;
* :class:`GatedFFN` -- the module, with ``torch.nn.Linear`` weight layouts.

The kernels (``csrc/ffn.cu``) form both projections, the activation and the
product in one launch and the down projection in a second.  For a backward
pass the block keeps its input and 8 bytes per hidden value: ``h`` in bf16 and
both projections in 24 bits.  bf16 operands with f32 accumulators and one
rounding for every stored value.  Any number of rows; widths that are
multiples of 8.
"""
from __future__ import annotations

import ctypes
from typing import Optional

import torch
import torch.nn as nn
from torch import Tensor

from . import _lib

LIB = "thetascan_b200"
ACTIVATIONS = {"silu": _lib.TS_FFN_SILU, "gelu": _lib.TS_FFN_GELU, "relu2": _lib.TS_FFN_RELU2}


def _check(x, w_gate, w_up, w_down, activation):
    for name, t in (("x", x), ("w_gate", w_gate), ("w_up", w_up), ("w_down", w_down)):
        if not t.is_cuda:
            raise RuntimeError("b200 backend requires CUDA tensors")
        if t.dtype != torch.bfloat16:
            raise ValueError(f"{name} must be bfloat16, got {t.dtype}")
        if t.device != x.device:
            raise ValueError(f"{name} is on {t.device}, x on {x.device}")
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation must be one of {sorted(ACTIVATIONS)}, got {activation!r}")
    if x.ndim < 1 or w_gate.ndim != 2 or w_gate.shape != w_up.shape or w_gate.shape[1] != x.shape[-1]:
        raise ValueError(f"w_gate {tuple(w_gate.shape)} and w_up {tuple(w_up.shape)} must be [hidden, {x.shape[-1]}]")
    if w_down.ndim != 2 or w_down.shape[1] != w_gate.shape[0]:
        raise ValueError(f"w_down {tuple(w_down.shape)} must be [width_out, {w_gate.shape[0]}]")
    if w_gate.shape[0] % 8 or w_gate.shape[1] % 8 or w_down.shape[0] % 8 or 0 in w_gate.shape or 0 in w_down.shape:
        raise NotImplementedError("gated_ffn: widths must be nonzero multiples of 8")


def _matrix(t):
    """``t [..., width]`` as rows with contiguous channels, a 16-byte aligned
    base and a row stride that is a multiple of 8: a view where ``t`` is one,
    else a copy."""
    t = t.reshape(-1, t.shape[-1])
    if t.shape[0] == 1:
        t = t.as_strided(t.shape, (t.shape[1], t.stride(1)))
    if t.stride(1) != 1 or t.stride(0) % 8 or t.stride(0) < t.shape[1] or t.data_ptr() % 16:
        t = t.clone(memory_format=torch.contiguous_format)
    return t


def _args(x2, w_gate, w_up, w_down, activation):
    a = _lib.FfnArgs()
    a.rows, a.width = x2.shape
    a.hidden, a.width_out, a.activation = w_gate.shape[0], w_down.shape[0], ACTIVATIONS[activation]
    a.x, a.w_gate, a.w_up, a.w_down = x2.data_ptr(), w_gate.data_ptr(), w_up.data_ptr(), w_down.data_ptr()
    a.x_stride, a.w_gate_stride, a.w_up_stride, a.w_down_stride = (x2.stride(0), w_gate.stride(0), w_up.stride(0),
                                                                   w_down.stride(0))
    return a


def _workspace(a, query, device):
    nbytes = query(ctypes.byref(a))
    if nbytes == 0:
        _lib.check(_lib.last_error()[0] or _lib.TS_ERR_VALUE)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=device)
    a.workspace, a.workspace_bytes = ws.data_ptr(), nbytes
    return ws


def _hidden(rows, hidden):
    """Bytes of the projections that a forward keeps (``ts_b200_ffn_kept_bytes``, from shapes alone)."""
    return -(-rows // 32) * -(-hidden // 32) * 6144


def _rows_of(x):
    return x.numel() // x.shape[-1]


def _ffn_fwd_impl(x, w_gate, w_up, w_down, activation, keep):
    """(y, h, kept); the last two are empty unless ``keep``."""
    with _lib.on_device(x):
        y = torch.empty(*x.shape[:-1], w_down.shape[0], dtype=x.dtype, device=x.device)
        rows, hidden = _rows_of(x), w_gate.shape[0]
        h = torch.empty((rows, hidden) if keep else 0, dtype=x.dtype, device=x.device)
        kept = torch.empty(_hidden(rows, hidden) if keep else 0, dtype=torch.uint8, device=x.device)
        if x.numel():
            lib = _lib.load()
            m = [_matrix(t) for t in (x, w_gate, w_up, w_down)]
            a = _args(*m, activation)
            a.y = y.data_ptr()
            if keep:
                a.h, a.kept = h.data_ptr(), kept.data_ptr()
            ws = _workspace(a, lib.ts_b200_ffn_fwd_workspace_bytes, x.device)
            _lib.check(lib.ts_b200_ffn_fwd(ctypes.byref(a), _lib.stream()))
            del ws
        return y, h, kept


def _ffn_bwd_impl(dy, x, w_gate, w_up, w_down, h, kept, activation, wanted):
    """Gradients of x and the three weights; an empty tensor where not wanted."""
    with _lib.on_device(x):
        inputs = (x, w_gate, w_up, w_down)
        out = [torch.empty(t.shape if need else 0, dtype=t.dtype, device=t.device) for t, need in zip(inputs, wanted)]
        if not x.numel():
            return tuple(t.zero_() for t in out)
        lib = _lib.load()
        m = [_matrix(t) for t in inputs]
        dy2 = _matrix(dy)
        a = _args(*m, activation)
        a.h, a.kept = h.data_ptr(), kept.data_ptr()
        ws = _workspace(a, lib.ts_b200_ffn_bwd_workspace_bytes, x.device)
        g = _lib.FfnGradArgs()
        g.dy, g.dy_stride = dy2.data_ptr(), dy2.stride(0)
        g.dx, g.dw_gate, g.dw_up, g.dw_down = (t.data_ptr() if need else None for t, need in zip(out, wanted))
        _lib.check(lib.ts_b200_ffn_bwd(ctypes.byref(a), ctypes.byref(g), _lib.stream()))
        del ws
        return tuple(out)


@torch.library.custom_op(f"{LIB}::gated_ffn_fwd", mutates_args=())
def gated_ffn_fwd(x: Tensor, w_gate: Tensor, w_up: Tensor, w_down: Tensor, activation: str,
                  keep: bool) -> tuple[Tensor, Tensor, Tensor]:
    """The block's output, and what its backward reads: h and the projections (empty unless ``keep``)."""
    return _ffn_fwd_impl(x, w_gate, w_up, w_down, activation, keep)


@gated_ffn_fwd.register_fake
def _(x, w_gate, w_up, w_down, activation, keep):
    rows, hidden = _rows_of(x), w_gate.shape[0]
    return (x.new_empty(*x.shape[:-1], w_down.shape[0]), x.new_empty((rows, hidden) if keep else (0,)),
            x.new_empty(_hidden(rows, hidden) if keep else 0, dtype=torch.uint8))


@torch.library.custom_op(f"{LIB}::gated_ffn_bwd", mutates_args=())
def gated_ffn_bwd(dy: Tensor, x: Tensor, w_gate: Tensor, w_up: Tensor, w_down: Tensor, h: Tensor, kept: Tensor,
                  activation: str, wanted: list[bool]) -> tuple[Tensor, Tensor, Tensor, Tensor]:
    """Gradients of x, w_gate, w_up, w_down (empty where not wanted)."""
    return _ffn_bwd_impl(dy, x, w_gate, w_up, w_down, h, kept, activation, wanted)


@gated_ffn_bwd.register_fake
def _(dy, x, w_gate, w_up, w_down, h, kept, activation, wanted):
    return tuple(t.new_empty(t.shape if need else (0,)) for t, need in zip((x, w_gate, w_up, w_down), wanted))


class _GatedFFN(torch.autograd.Function):
    """Autograd of the block.  The kernels are called directly in eager mode;
    a tracing compiler sees the custom ops (whose dispatch costs the host more)."""

    @staticmethod
    def forward(ctx, x, w_gate, w_up, w_down, activation):
        fwd = gated_ffn_fwd if torch.compiler.is_compiling() else _ffn_fwd_impl
        y, h, kept = fwd(x, w_gate, w_up, w_down, activation, True)
        ctx.activation = activation
        ctx.save_for_backward(x, w_gate, w_up, w_down, h, kept)
        return y

    @staticmethod
    def backward(ctx, dy):
        wanted = list(ctx.needs_input_grad[:4])
        bwd = gated_ffn_bwd if torch.compiler.is_compiling() else _ffn_bwd_impl
        grads = bwd(dy, *ctx.saved_tensors, ctx.activation, wanted)
        return (*(t if need else None for t, need in zip(grads, wanted)), None)


def gated_ffn(x: Tensor, w_gate: Tensor, w_up: Tensor, w_down: Tensor, activation: str = "silu") -> Tensor:
    """``(act(x w_gate^T) * (x w_up^T)) w_down^T`` over the last dimension of
    ``x [..., width]``; ``w_gate`` and ``w_up`` are ``[hidden, width]``,
    ``w_down`` is ``[width_out, hidden]``, all bf16.  ``activation`` is
    ``"silu"``, ``"gelu"`` (exact) or ``"relu2"`` (``max(g, 0)^2``)."""
    _check(x, w_gate, w_up, w_down, activation)
    if torch.is_grad_enabled() and any(t.requires_grad for t in (x, w_gate, w_up, w_down)):
        return _GatedFFN.apply(x, w_gate, w_up, w_down, activation)
    fwd = gated_ffn_fwd if torch.compiler.is_compiling() else _ffn_fwd_impl
    return fwd(x, w_gate, w_up, w_down, activation, False)[0]


class GatedFFN(nn.Module):
    """Gated feed-forward block with weights ``gate`` and ``up`` ``[hidden,
    d_model]`` and ``down`` ``[d_model, hidden]`` (no biases).  Operands are
    rounded to bf16 where they are kept wider; the output has the type of the
    input."""

    def __init__(self, d_model: int, hidden: int, activation: str = "silu", *, device=None,
                 dtype: Optional[torch.dtype] = None):
        super().__init__()
        if activation not in ACTIVATIONS:
            raise ValueError(f"activation must be one of {sorted(ACTIVATIONS)}, got {activation!r}")
        if d_model < 8 or hidden < 8 or d_model % 8 or hidden % 8:
            raise NotImplementedError("gated_ffn: widths must be nonzero multiples of 8")
        kw = dict(bias=False, device=device, dtype=dtype)
        self.gate, self.up = nn.Linear(d_model, hidden, **kw), nn.Linear(d_model, hidden, **kw)
        self.down = nn.Linear(hidden, d_model, **kw)
        self.activation = activation

    def forward(self, x):
        bf = torch.bfloat16
        y = gated_ffn(x.to(bf), self.gate.weight.to(bf), self.up.weight.to(bf), self.down.weight.to(bf),
                      self.activation)
        return y.to(x.dtype)
