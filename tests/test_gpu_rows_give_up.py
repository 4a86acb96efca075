"""A wait inside a grouped product that runs out does not stay silent."""
import pytest
import torch

import sparseconvnet_b200 as scn
from sparseconvnet_b200._lib import lib

pytestmark = pytest.mark.gpu


# one block to a tile, two, fp32 rows that the kernel splits, and long sums of one block and of two
SHAPES = [(256, 4096, 256, torch.bfloat16), (20000, 4096, 512, torch.bfloat16), (200000, 256, 64, torch.float32), (130, 16384, 200, torch.float16),
          (2600, 16384, 2304, torch.bfloat16)]


@pytest.mark.parametrize("rows,k,n,t,then", [(*s, "forward") for s in SHAPES] + [(*SHAPES[0], then) for then in ("backward", "quantized")])
def test_the_next_call_says_so(cuda, rows, k, n, t, then):
    """One arrival is left out: the call gives up in bounded time, and the next one on the device raises, once."""
    o = torch.tensor([0, rows], device="cuda")
    x, w = torch.randn(rows, k, device="cuda").to(t), torch.randn(1, k, n, device="cuda").to(t).requires_grad_()
    y = scn.grouped_product(x, w, o)
    dy = torch.randn(rows, n, device="cuda").to(t)
    (want,) = torch.autograd.grad(y, [w], dy, retain_graph=True)
    q, scale = scn.rms_norm_quantized(x[:8].float())
    wq, ws = scn.quantize_group_weights(w)
    few = torch.tensor([0, 8], device="cuda")
    calls = dict(forward=lambda: scn.grouped_product(x, w.detach(), o), backward=lambda: torch.autograd.grad(y, [w], dy, retain_graph=True)[0],
                 quantized=lambda: scn.grouped_product_quantized(q, scale, wq, ws, few))
    right = calls["quantized"]()
    scn.poll_errors()
    lib.scn_test_drop_barrier_arrival()
    scn.grouped_product(x, w.detach(), o)
    torch.cuda.synchronize()
    with pytest.raises(Exception, match="ran out"):
        calls[then]()
    scn.poll_errors()  # it has been said
    assert torch.equal(calls["forward"](), y) and torch.equal(calls["backward"](), want) and torch.equal(calls["quantized"](), right)
    scn.poll_errors()
