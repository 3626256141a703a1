"""Device collectives and the operators that models are trained with: thin Python layers over
the sm_100a kernels."""
from .device import (ALGO_NVLS, ALGO_NVLS_ONESHOT, ALGO_ONESHOT, ALGO_TWOSHOT, DeviceSession,
                     dtype_code, op_code)
from .train import check, distill_loss, gated_linear, group_norm

__all__ = ["DeviceSession", "dtype_code", "op_code", "ALGO_ONESHOT", "ALGO_TWOSHOT", "ALGO_NVLS",
           "ALGO_NVLS_ONESHOT", "check", "distill_loss", "gated_linear", "group_norm"]
