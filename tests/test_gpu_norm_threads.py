"""Norms of wide rows from two host threads at once."""
import threading

import pytest
import torch

import sparseconvnet_b200 as scn
from sparseconvnet_b200._lib import lib

pytestmark = pytest.mark.gpu


def test_gradients_of_two_widths_at_once(cuda):
    """Rows of more than 12 288 planes need more shared memory than a kernel has by itself, each width an amount of its own."""
    failed = []

    def calls(planes, seed):
        with torch.cuda.stream(torch.cuda.Stream()):
            g = torch.Generator(device="cuda").manual_seed(seed)
            s, dy = (torch.randn(2, planes, generator=g, device="cuda") for _ in range(2))
            k, dx, dw = torch.ones(2, device="cuda"), torch.empty_like(s), torch.empty(planes, device="cuda")
            for _ in range(4000):
                status = lib.scn_rms_norm_backward(s.data_ptr(), planes, 0, None, k.data_ptr(), dy.data_ptr(), 0, None, 2, planes, dx.data_ptr(),
                                                   dw.data_ptr(), torch.cuda.current_stream().cuda_stream)
                if status:
                    failed.append((planes, status))
                    return
            torch.cuda.current_stream().synchronize()
            off = dw.double() - (s.double() * dy.double()).sum(0)
            if not float(off.abs().max()) <= 4 * 2.0 ** -24 * float((s * dy).abs().sum(0).max()):
                failed.append((planes, "values"))

    threads = [threading.Thread(target=calls, args=a) for a in ((16384, 1), (12800, 2), (14336, 3))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed
    x = torch.randn(3, 16000, device="cuda", requires_grad=True)
    (dx,) = torch.autograd.grad(scn.rms_norm(x).sum(), [x])
    assert bool(dx.isfinite().all())
