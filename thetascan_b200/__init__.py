"""thetascan_b200 -- B200-native (sm_100a) backend for the ThetaScan mixer hot path.

Public surface (mirrors the reference package ``thetascan``):

* ``ThetaScan`` / ``ThetaScanConfig`` (+ sub-configs): the mixer module and
  its configuration, state-dict compatible with the reference;
* ``scan``: the scan-backend contract (``linattn_views`` / ``linattn``);
* ``kernel.kernel_core``: the fused kernel-family hot path;
* ``rms_norm`` / ``add_rms_norm`` / ``rms_norm_8bit``: the norms around it;
* ``gated_ffn`` / ``GatedFFN``: the gated feed-forward block;
* ``AdamW`` / ``adamw_step``: the optimizer step over many tensors;
* ``integration.install()``: register ``backend="b200"`` in an installed
  reference package.

All compute goes through the C ABI of ``include/thetascan_b200.h``.
"""
from __future__ import annotations

from .config import (GNConfig, KernelConfig, RegularizationConfig, RoPEConfig, RuntimeConfig,
                     TemporalConfig, ThetaScanConfig)
from .ffn import GatedFFN, gated_ffn
from .mixer import ThetaScan
from .norm import add_rms_norm, rms_norm, rms_norm_8bit
from .optim import AdamW, adamw_step

__version__ = "0.1.0"
BACKEND_NAME = "b200"

__all__ = ["GNConfig", "KernelConfig", "RegularizationConfig", "RoPEConfig", "RuntimeConfig",
           "TemporalConfig", "ThetaScan", "ThetaScanConfig", "BACKEND_NAME",
           "AdamW", "GatedFFN", "adamw_step", "add_rms_norm", "gated_ffn", "rms_norm", "rms_norm_8bit"]
