"""Operators on rows of any kind: the sites of a scale, points, tokens.  They need no Metadata object and take float32,
bfloat16 or float16 matrices on a GPU; results go to the current stream of the tensors' device.

``layers.py`` has the module forms (RMSNormalization, AddRMSNormalization, ...).  None of these is in the reference; they
stand beside its BatchNormalization and NetworkInNetwork."""
import torch

from . import SCN

_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_E4M3 = 3


def _type_code(dtype, name):
    if dtype is None:
        return -1
    if dtype not in _TYPES:
        raise ValueError("%s must be torch.float32, torch.bfloat16 or torch.float16" % name)
    return _TYPES[dtype]


def _row_weight(weight):
    return weight if weight is None or weight.dtype == torch.float32 else weight.float()


def rms_norm(x, weight=None, residual=None, eps=1e-6, out_dtype=None):
    """Root-mean-square norm of every row of ``x`` [.., planes]: x / sqrt(mean(x^2) + eps) * weight.

    With ``residual`` (same shape and type) the norm is that of s = x + residual, rounded to the type of x, and the result
    is the pair (norm, s): s is what the next residual connection adds to.  ``weight``: [planes], None for ones.
    ``out_dtype``: type of the norm, None for the type of x.  Differentiable (once) in x, residual and weight; x and
    residual receive the same gradient.  Sums are float32."""
    return SCN._binding.rms_norm(x, _row_weight(weight), residual, eps, _type_code(out_dtype, "out_dtype"))


def rms_norm_quantized(x, weight=None, residual=None, eps=1e-6):
    """``rms_norm`` with the norm in 8 bits: (q, scale) or, with ``residual``, (q, scale, s).  q is a torch.float8_e4m3fn
    tensor of the shape of x, scale float32 of its leading sizes: q * scale is the norm, and the largest value of a row is
    448 in q (a row of zeros is zeros).  No gradient."""
    return SCN._binding.rms_norm(x, _row_weight(weight), residual, eps, _E4M3)
