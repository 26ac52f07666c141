"""AdamW over many tensors in one launch, with states in 32 or in 8 bits.

* :func:`adamw_step` -- one step on lists of tensors, in place;
* :class:`AdamW` -- the ``torch.optim.Optimizer`` that keeps the states.

One kernel launch updates up to 400 tensors of one kind (``csrc/adamw.cu``);
their addresses travel with the launch, so nothing is kept between calls.

8-bit states hold e4m3 codes of the first moment and of the square root of
the second, and an f32 scale for each 256 elements of a tensor (its largest
magnitude / 448).  The step uses f32 values; the codes are rounded
stochastically, because a moving average moves by less than half a code per
step and rounding to nearest would hold it in place.  The random words are a
hash of ``(seed, step, place of the tensor, element)``: a step is a function of
its arguments.  A NaN stays in its element; an infinite value makes its block
of 256 non-finite.  Finite gradients up to 1e37 do neither.
"""
from __future__ import annotations

import torch

from . import _lib

BLOCK = 256
_DTYPES = (torch.float32, torch.bfloat16)


def state_scales(n: int) -> int:
    """Scales of an 8-bit state of ``n`` elements."""
    return -(-n // BLOCK)


def _require(ok, message):
    if not ok:
        raise ValueError(f"adamw: {message}")


def _require_options(lr, betas, eps, weight_decay):
    b1, b2 = betas
    if not (0 <= b1 < 1 and 0 <= b2 < 1):
        raise ValueError(f"adamw: betas must lie in [0, 1), got {betas}")
    _require(lr >= 0 and eps >= 0 and weight_decay >= 0, "lr, eps and weight_decay must be >= 0")


def adamw_step(params, grads, exp_avgs, exp_avg_sqs, *, step: int, lr: float, betas=(0.9, 0.999), eps: float = 1e-8,
               weight_decay: float = 1e-2, masters=None, exp_avg_scales=None, exp_avg_sq_scales=None,
               seed: int = 0, ordinals=None) -> None:
    """One AdamW step, in place, on lists of CUDA tensors of one device.

    ``params`` are f32 or bf16 and contiguous, ``grads`` f32 or bf16 of the
    same shapes (or flat, as the other lists).  ``masters`` (f32) belong to
    bf16 parameters and carry their values.  States are f32 tensors, or ``float8_e4m3fn`` codes (of the first
    moment, and of the root of the second) with f32 scales of
    ``state_scales(numel)`` entries.  ``step`` counts from 1; ``ordinals`` are
    the tensors' places in the whole step (default 0, 1, ...), which key the
    stochastic rounding of 8-bit states with ``seed``."""
    if not (isinstance(step, int) and step >= 1):
        raise ValueError(f"adamw: step must be an integer >= 1, got {step!r}")
    _require_options(lr, betas, eps, weight_decay)
    b1, b2 = betas
    _lib.host().adamw(params, grads, exp_avgs, exp_avg_sqs, masters, exp_avg_scales, exp_avg_sq_scales, ordinals, step, lr,
                      b1, b2, eps, weight_decay, seed)


class AdamW(torch.optim.Optimizer):
    """AdamW with decoupled weight decay over :func:`adamw_step`.

    ``state_bits=8`` keeps the moments in 8 bits; ``master_weights=True`` keeps
    an f32 value behind every bf16 parameter, which carries it from its first
    step on: a parameter that is written otherwise afterwards (weights loaded
    into the model) needs its ``state["master"]`` written too, or the optimizer
    made anew.  Parameters are contiguous CUDA tensors in f32 or bf16; gradients
    may be either type.  ``seed`` keys the rounding of 8-bit states.  A step
    that is refused with an error does not count."""

    def __init__(self, params, lr: float = 1e-3, betas=(0.9, 0.999), eps: float = 1e-8, weight_decay: float = 1e-2, *,
                 state_bits: int = 32, master_weights: bool = False, seed: int = 0):
        super().__init__(params, dict(lr=lr, betas=tuple(betas), eps=eps, weight_decay=weight_decay,
                                      state_bits=state_bits, master_weights=master_weights, seed=seed))

    def add_param_group(self, param_group):
        super().add_param_group(param_group)
        group = self.param_groups[-1]
        try:
            _require(group["state_bits"] in (8, 32), f"state_bits must be 8 or 32, got {group['state_bits']}")
            _require_options(group["lr"], group["betas"], group["eps"], group["weight_decay"])
            for p in group["params"]:
                _require(p.dtype in _DTYPES, f"parameters must be float32 or bfloat16, got {p.dtype}")
                _require(p.is_contiguous(), "parameters must be contiguous")
        except ValueError:
            self.param_groups.pop()
            raise

    def _new_state(self, p, group):
        state = {"step": 0}
        if group["state_bits"] == 8:
            for name in ("exp_avg", "exp_avg_sq"):
                state[name] = torch.zeros(p.shape, dtype=torch.float8_e4m3fn, device=p.device)
                state[name + "_scale"] = torch.zeros(state_scales(p.numel()), device=p.device)
        else:
            for name in ("exp_avg", "exp_avg_sq"):
                state[name] = torch.zeros(p.shape, dtype=torch.float32, device=p.device)
        if group["master_weights"] and p.dtype == torch.bfloat16:
            state["master"] = p.detach().float()
        return state

    def load_state_dict(self, state_dict):
        """States keep the types that they were saved in (the base class would
        give them the parameters')."""
        super().load_state_dict(state_dict)
        saved = state_dict["state"]
        ids = [i for g in state_dict["param_groups"] for i in g["params"]]
        for i, p in zip(ids, (p for g in self.param_groups for p in g["params"]), strict=True):
            if i in saved:
                self.state[p] = {k: v.detach().to(p.device, copy=True) if torch.is_tensor(v) else v
                                 for k, v in saved[i].items()}

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        calls, ordinal = [], 0
        for group in self.param_groups:
            together = {}
            for p in group["params"]:
                ordinal += 1
                if p.grad is None:
                    continue
                if p.grad.is_sparse:
                    raise RuntimeError("adamw: sparse gradients are not supported")
                state = self.state[p]
                if not state:
                    state.update(self._new_state(p, group))
                # tensors of one step count and device go together, those with a master apart
                master = "master" in state
                key = (state["step"] + 1, p.device, master, (p.dtype, p.grad.dtype) if master else None)
                together.setdefault(key, []).append((ordinal - 1, p, state))
            calls += [(group, count, master, *zip(*entries)) for (count, _, master, _), entries in together.items()]
        for group, count, master, ordinals, params, states in calls:
            eight = group["state_bits"] == 8
            adamw_step(params, [p.grad for p in params], [s["exp_avg"] for s in states], [s["exp_avg_sq"] for s in states],
                       step=count, lr=float(group["lr"]), betas=group["betas"], eps=group["eps"],
                       weight_decay=group["weight_decay"], masters=[s["master"] for s in states] if master else None,
                       exp_avg_scales=[s["exp_avg_scale"] for s in states] if eight else None,
                       exp_avg_sq_scales=[s["exp_avg_sq_scale"] for s in states] if eight else None,
                       seed=group["seed"], ordinals=ordinals)
            for state in states:   # a refused step does not count
                state["step"] = count
        return loss
