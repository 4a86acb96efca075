"""Gradients of norms around the widths at which a block needs more shared memory than kernels have by themselves."""
import pytest
import torch

import sparseconvnet_b200 as scn

pytestmark = pytest.mark.gpu
E = 2.0 ** -24


@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dy_type", [None, torch.float32])
@pytest.mark.parametrize("planes", [8192, 8193, 12223, 12224, 12225, 12226, 12272, 12280, 12288, 12289, 16383, 16384])
def test_widths(cuda, planes, t, dy_type):
    g = torch.Generator(device="cuda").manual_seed(planes)
    x, w = torch.randn(3, planes, generator=g, device="cuda").to(t).requires_grad_(), torch.randn(planes, generator=g, device="cuda").requires_grad_()
    y = scn.rms_norm(x, w, out_dtype=dy_type)
    dy = torch.randn(3, planes, generator=g, device="cuda").to(y.dtype)
    dx, dw = torch.autograd.grad(y, [x, w], dy)
    s = x.detach().double()
    k = (s.square().mean(1, keepdim=True) + 1e-6).rsqrt()
    h, d = s * k, dy.double()
    along = (d * w.detach().double() * h).mean(1, keepdim=True)
    want, size = k * (d * w.detach().double() - h * along), k * ((d * w.detach().double()).abs() + h.abs() * (d * w.detach().double() * h).abs().mean(1, keepdim=True))
    # fp32 sums of 16384 values by 512 threads: 32 additions a thread and ten more, halved by the root, a handful of products: 100 E with room
    assert bool(((dx.double() - want).abs() <= torch.finfo(t).eps / 2 * want.abs() * (1 + 1e-6) + 100 * E * size + torch.finfo(t).smallest_normal).all())
    assert bool(((dw.double() - (d * h).sum(0)).abs() <= 60 * E * (d * h).abs().sum(0)).all())
