"""Every allocation of a grouped product that can fail, in both directions: an error that says so, nothing lost, and the next call right."""
import ctypes as C

import pytest
import torch

import sparseconvnet_b200 as scn
from sparseconvnet_b200._lib import lib

pytestmark = pytest.mark.gpu


def used():
    a, b = C.c_uint64(), C.c_uint64()
    assert lib.scn_memory_usage(C.byref(a), C.byref(b)) == 0
    return b.value


# fp32 rows that the kernel splits: the weights' parts; backward those and the partial sums (with the bias's).  Wider ones: parts of rows and
# weights; backward of dy, weights and x, partial sums of weights and of bias.  bf16 rows of odd width: a copy of x, and the same sums.
@pytest.mark.parametrize("t,k,n,forward,backward", [(torch.float32, 64, 96, 1, 2), (torch.float32, 300, 300, 2, 5), (torch.bfloat16, 63, 96, 1, 3)])
def test_each_allocation_in_turn(cuda, t, k, n, forward, backward):
    o = torch.tensor([0, 150, 800], device="cuda")
    x, w, b, dy = (torch.randn(*s, device="cuda").to(t) for s in ((800, k), (2, k, n), (2, n), (800, n)))
    type_, stream = {torch.float32: 0, torch.bfloat16: 1}[t], torch.cuda.current_stream().cuda_stream
    sizes = (o.data_ptr(), 1, 800, 2, k, n, 0)

    def product():
        y = torch.empty(800, n, device="cuda", dtype=t)
        return lib.scn_grouped_product_forward(x.data_ptr(), k, type_, w.data_ptr(), b.data_ptr(), type_, *sizes, y.data_ptr(), type_, stream), (y,)

    def gradients():
        made = [torch.empty_like(v) for v in (x, w, b)]
        return lib.scn_grouped_product_backward(x.data_ptr(), k, type_, w.data_ptr(), dy.data_ptr(), n, *sizes, *(v.data_ptr() for v in made), stream), made

    for call, allocations in ((product, forward), (gradients, backward)):
        status, want = call()
        assert status == 0
        torch.cuda.synchronize()
        before = used()
        for which in range(1, allocations + 2):
            lib.scn_test_fail_allocation(which)
            try:
                status, _ = call()
            finally:
                lib.scn_test_fail_allocation(0)
            if which <= allocations:
                assert status != 0 and b"out of memory" in lib.scn_last_error(), which
            else:
                assert status == 0, which  # there is no further one
            assert used() == before
            status, got = call()
            assert status == 0 and all(torch.equal(p, q) for p, q in zip(got, want))
    scn.poll_errors()
