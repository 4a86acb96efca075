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


def grouped_product(x, weight, offsets, bias=None, out_dtype=None):
    """Every group of rows times its own weights: for offsets[g] <= r < offsets[g + 1]

        out[r] = x[r] @ weight[g] (+ bias[g])

    x: [n, nIn], rows in group order; weight: [groups, nIn, nOut]; bias: [groups, nOut]; all of one type.  offsets: int64 or
    int32 CUDA tensor [groups + 1], not decreasing (1 to 1024 groups, empty ones among them); the host never waits for
    them.  Rows of no group (before the first, behind the last) are zeros and have no gradient.
    bfloat16 and float16 are multiplied as they are; float32 by ``set_precision``: 'fp32' with all bits, 'tf32x3' and 'tf32'
    to 2^-17 of a product, 'bf16' rounded to bfloat16 (the input's gradient by ``set_backward_precision``, the weights'
    with all bits).  In 'fp32' values below 2^-110 (8e-34) are held to within 2^-134.  Sums are float32, results ``out_dtype``
    (None: the type of x); the gradient of float32 results of 16-bit operands is rounded to the operands' type first.  A float32 row with an infinity may
    give NaN.  Differentiable (once) in x, weight and bias."""
    return SCN._binding.grouped_product(x, weight, offsets, bias, _type_code(out_dtype, "out_dtype"), SCN._precision,
                                        SCN._backward_precision)


def quantize_group_weights(weight):
    """Weights [groups, nIn, nOut] as ``grouped_product_quantized`` reads them: (float8_e4m3fn [groups, nOut, nIn], float32
    scales [groups, nOut]), the largest value of a column at 448.  Done once for a network that serves."""
    w = weight.detach().float().transpose(1, 2)
    scale = w.abs().amax(2).clamp_min(1e-30) / 448
    return (w / scale[:, :, None]).contiguous().to(torch.float8_e4m3fn), scale


def grouped_product_quantized(q, scale, weight, weight_scale, offsets, bias=None, out_dtype=torch.bfloat16):
    """``grouped_product`` on 8-bit rows, as ``rms_norm_quantized`` makes them, and 8-bit weights
    (``quantize_group_weights``):

        out[r, o] = scale[r] * weight_scale[g, o] * sum_i q[r, i] weight[g, o, i] (+ bias[g, o])

    The products are exact and summed in float32; no gradient."""
    if out_dtype not in _TYPES:
        raise ValueError("out_dtype must be torch.float32, torch.bfloat16 or torch.float16")
    return SCN._binding.grouped_product_quantized(q, scale, weight, weight_scale, offsets, bias, _TYPES[out_dtype])


def poll_errors():
    """Waits for the current stream and raises if a wait inside a grouped product of the current device ran out (its results are
    incomplete then).  A later grouped product raises this without waiting; what is behind the last one, or in a replayed graph,
    shows here.  The counterpart of ``Metadata.poll_errors``."""
    SCN.check(SCN.lib.scn_rows_poll_errors(SCN._stream()))
