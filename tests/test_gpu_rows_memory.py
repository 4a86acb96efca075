"""Memory that the operators on rows take for themselves."""
import ctypes as C
import itertools

import pytest
import torch

import sparseconvnet_b200 as scn
from sparseconvnet_b200._lib import lib

pytestmark = pytest.mark.gpu


def reserved():
    a, b = C.c_uint64(), C.c_uint64()
    assert lib.scn_memory_usage(C.byref(a), C.byref(b)) == 0
    return a.value


@pytest.mark.parametrize("rows,groups,k,n,t,most", [
    # partial sums of units of 256 rows: 128 * 256 * 4 bytes for each, one unit more than that for a group
    (1000001, 1, 128, 256, torch.float32, (1000001 / 256 + 1) * 128 * 256 * 4),
    (1000001, 16, 64, 96, torch.float32, (1000001 / 256 + 16) * 65 * 96 * 4 + 16 * 64 * 96 * 6),
    # units of 1/4 of the rows: 64 tiles of 256 x 256 results, two units wanted for each SM
    (60000, 1, 2048, 2048, torch.bfloat16, 5 * 2048 * 2048 * 4)])
def test_a_weights_gradient(cuda, rows, groups, k, n, t, most):
    o = torch.linspace(0, rows, groups + 1, device="cuda").long()
    x, dy = torch.randn(rows, k, device="cuda").to(t), torch.randn(rows, n, device="cuda").to(t)
    w = torch.randn(groups, k, n, device="cuda").to(t).requires_grad_()
    y = scn.grouped_product(x, w, o)
    torch.cuda.synchronize()
    assert lib.scn_trim_memory(0) == 0
    before = reserved()
    torch.autograd.grad(y, [w], dy)
    torch.cuda.synchronize()
    # sizes are rounded up by a quarter at most, and the pool takes 32 MB at a time
    assert reserved() - before <= 1.25 * most + (64 << 20), (reserved() - before) / most


@pytest.mark.parametrize("sizes", [[257] * 40, [256] * 40, [257] * 20 + [10280] + [0] * 5, [513] * 8 + [1] * 100, list(range(0, 1200, 37))])
def test_partial_sums_have_room(cuda, sizes):
    """Groups just above a unit's rows are the most units for their rows: what lies behind the sums stays as it was."""
    o = torch.tensor([0] + list(itertools.accumulate(sizes)), device="cuda")
    rows = int(o[-1])
    x, dy = (torch.randint(-4, 5, (rows, c), device="cuda").float() for c in (40, 24))  # exact sums
    w, b = torch.zeros(len(sizes), 40, 24, device="cuda", requires_grad=True), torch.zeros(len(sizes), 24, device="cuda", requires_grad=True)
    for _ in range(3):
        dw, db = torch.autograd.grad(scn.grouped_product(x, w, o, b), [w, b], dy)
        for g in range(len(sizes)):
            r = slice(int(o[g]), int(o[g + 1]))
            assert torch.equal(dw[g].double(), x[r].double().T @ dy[r].double()) and torch.equal(db[g].double(), dy[r].double().sum(0))
