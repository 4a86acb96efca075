"""Calls on rows that are refused instead of answered wrongly."""
import pytest
import torch
import torch.autograd.forward_ad as forward_ad

import sparseconvnet_b200 as scn

pytestmark = pytest.mark.gpu


def test_forward_mode_of_products_in_8_bits(cuda):
    """A tangent of any operand would be lost."""
    o = torch.tensor([0, 3, 8], device="cuda")
    q, scale = scn.rms_norm_quantized(torch.randn(8, 32, device="cuda"))
    w, ws = scn.quantize_group_weights(torch.randn(2, 32, 16, device="cuda"))
    bias = torch.randn(2, 16, device="cuda")
    with forward_ad.dual_level():
        for name in ("scale", "ws", "bias"):
            given = dict(scale=scale, ws=ws, bias=bias)
            given[name] = forward_ad.make_dual(given[name], torch.ones_like(given[name]))
            with pytest.raises(NotImplementedError, match="forward-mode"):
                scn.grouped_product_quantized(q, given["scale"], w, given["ws"], o, given["bias"])
        y = scn.grouped_product_quantized(q, scale, w, ws, o, bias)
        assert forward_ad.unpack_dual(y).tangent is None
