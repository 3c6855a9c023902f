"""B200-native MLX affine group-quantized linear (the quantized DiT linear of
image-forger / vincenthz/qwen-imager), behind the reference's operator API.

Public API:
  Linear, linear, Affine   -- src/quant.rs `quant::Linear` mirror (quant.py)
  VarBuilder               -- weight supply (weights.py)
  QmmError                 -- non-OK status of the C ABI (include/qmm.h)
  mx_quantize, MxTensor, MxLinear -- MXFP4 quantisation and product (mxfp4.py)
  RotaryAxes, qk_norm_rotary      -- q/k norm and multi-axis rotary positions (rotary.py)
  gated_residual_norm             -- norms before and after a block, gate, residual (gated_norm.py)
"""
from ._lib import QmmError
from .gated_norm import gated_residual_norm
from .mxfp4 import MxLinear, MxTensor, mx_quantize
from .quant import Affine, Linear, device_error, linear
from .rotary import RotaryAxes, qk_norm_rotary
from .weights import VarBuilder, WeightError

__all__ = ["Affine", "Linear", "MxLinear", "MxTensor", "QmmError", "RotaryAxes", "VarBuilder", "WeightError", "device_error",
           "gated_residual_norm", "linear", "mx_quantize", "qk_norm_rotary"]
