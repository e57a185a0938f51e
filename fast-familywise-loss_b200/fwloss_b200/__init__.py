"""fwloss_b200: Familywise loss forward+backward on NVIDIA B200 (sm_100a).

Python API (drop-in for the reference's Python-facing entry points):
  familywise_loss(logits, target, reduction)  like fwcpp.familywise_loss
  FWLoss(num_classes, reduction, device)      like reference_impl.FWLoss
  fw_radix_cuda (sibling module)              like the reference's extension
The two ends of a language model around the loss:
  embed_tokens                                embedding rows and the table's gradient
  rms_norm, rms_norm_int8                     norm of a residual stream, float or 8-bit output
  lm_head_cross_entropy                       softmax cross entropy of an output layer, no logits kept
  int8_linear, quantize_rows_int8             output layer in 8-bit integers (serving)
C ABI: libfwloss_b200.so, declared in include/fwloss_b200.h; `capi` binds it
with ctypes.
"""
from .functional import familywise_loss, fw_rows, mean_of_rows  # noqa: F401
from .modules import FWLoss  # noqa: F401
from .cross_entropy import lm_head_cross_entropy  # noqa: F401
from .embedding import embed_tokens  # noqa: F401
from .int8 import int8_linear, quantize_rows_int8  # noqa: F401
from .norm import rms_norm, rms_norm_int8  # noqa: F401
from . import capi  # noqa: F401

__all__ = ["familywise_loss", "fw_rows", "mean_of_rows", "FWLoss", "embed_tokens", "rms_norm", "rms_norm_int8",
           "lm_head_cross_entropy", "int8_linear", "quantize_rows_int8", "capi"]
__version__ = "0.1.0"
