"""float32 operands of grouped products near the lower end of the range.

A value is the sum of three bf16 numbers, each rounded to nearest of what those before it leave: all 24 bits from 2^-110 on, whose last bit is
2^-133, bf16's smallest number; below that, half of it, 2^-134, may be lost of each value.  Products and sums as elsewhere: 2^-25 of
a product left out and (2 * 16 + n / 256 + 4) 2^-23 of the sum of the products' sizes."""
import pytest
import torch

import sparseconvnet_b200 as scn

pytestmark = pytest.mark.gpu
E = 2.0 ** -23


def values(*shape, low, high, seed):
    """Of sizes 2^low to 2^high, spread over the powers of two, with all bits of the mantissa"""
    g = torch.Generator(device="cuda").manual_seed(seed)
    u = torch.rand(2, *shape, generator=g, device="cuda", dtype=torch.float64)
    v = (1 + u[0]) * 2.0 ** (low + (high - low) * u[1]).floor()
    return (v * (torch.randint(0, 2, shape, generator=g, device="cuda") * 2 - 1)).float()


@pytest.mark.parametrize("k", [96, 300])  # split in the kernel, and in memory
@pytest.mark.parametrize("low,high", [(-110, -109), (-110, -60), (-118, -110), (-126, -110)])
def test_small_values(cuda, k, low, high):
    o = torch.tensor([0, 70, 200], device="cuda")
    x, w = values(200, k, low=low, high=high, seed=1).requires_grad_(), values(2, k, 72, low=60, high=80, seed=2).requires_grad_()
    dy = values(200, 72, low=60, high=80, seed=3)
    y = scn.grouped_product(x, w, o)
    (dw,) = torch.autograd.grad(y, [w], dy)
    lost = 0.0 if low >= -110 else 2.0 ** -134
    rel = lambda n: 2.0 ** -25 + (2 * 16 + n / 256 + 4) * E  # noqa: E731
    for g, r in enumerate((slice(0, 70), slice(70, 200))):
        a, b, d = x[r].detach().double(), w[g].detach().double(), dy[r].double()
        for got, want, size, other, n in ((y[r], a @ b, a.abs() @ b.abs(), b.abs().sum(0), k), (dw[g], a.T @ d, a.abs().T @ d.abs(), d.abs().sum(0), len(d))):
            off = (got.detach().double() - want).abs()
            assert bool((off <= 2.0 ** -24 * want.abs() * (1 + 1e-6) + rel(n) * size + lost * other).all()), float((off / size).max())
