"""MI355X-native kernels for the decaying-fast-weight recurrence (drop-in for T2FW's
``LFWFunction`` / ``DFWFunction`` autograd functions)."""
from .functional_lfw import (LFWFunction, LFWGatedFunction, LFWHeadsFunction, sigmoid_gates, lfw_step,  # noqa: F401
                             lfw_apply_16bit, lfw_apply_padded, DEFAULT_CKPT_INTERVAL)
from .functional_dfw import DFWFunction  # noqa: F401
from .functional_scan import gated_scan, gated_scan_step  # noqa: F401
from .functional_norm import residual_rms_norm, residual_rms_norm_fp8  # noqa: F401
from .functional_loss import policy_loss  # noqa: F401
from .grad_clip import clip_grad_norm, grad_norm  # noqa: F401
from .state_cache import FastWeightState  # noqa: F401

__all__ = ["LFWFunction", "LFWGatedFunction", "LFWHeadsFunction", "DFWFunction", "FastWeightState", "sigmoid_gates", "lfw_step", "lfw_apply_16bit", "lfw_apply_padded",
           "gated_scan", "gated_scan_step", "residual_rms_norm", "residual_rms_norm_fp8", "policy_loss", "clip_grad_norm", "grad_norm",
           "DEFAULT_CKPT_INTERVAL"]
