"""Grouped products of 16- and 8-bit values whose sums are long: the error must not grow with their length.

The tensor core cuts its running sum off at every instruction, 16 products of 16-bit values or 32 of 8-bit ones.  A sum is
handed over to fp32 registers after 256 instructions, so that with products of one sign it loses at most 2 * 257 * 2^-23 of itself
(each instruction may cut the products' alignment and the addition off, 2^-23 of the part's sum each), and the parts' sums are
added with rounding to nearest, half a unit of 2^-23 for each of them.  Rounding to a result's type keeps the order of numbers,
so a result lies between the roundings of the two ends of that range: a loss of a part of a rounding step shows as well."""
import pytest
import torch

import sparseconvnet_b200 as scn

pytestmark = pytest.mark.gpu
E = 2.0 ** -23
HALF = [torch.float16, torch.bfloat16]


def positive(*shape, t, seed, most=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.rand(*shape, generator=g, device="cuda", dtype=torch.float32).mul_(most).to(t)


def check(got, want, parts, t, others=0.0):
    """`parts`: hand-overs; `others`: what the addition of partial sums and the scales bring, relative"""
    room = 2 * 257 * E + parts * E / 2 + others + E  # (E: the ends are rounded to float32 on their way)
    low, high = (want * (1 - room)).to(t), (want * (1 + room)).to(t)
    assert bool(((low <= got) & (got <= high)).all()), float(((got.double() - want) / want).mean())


# rows, nIn, nOut: tiles of one block (few planes on one side, so that a group is one unit all the same) and of two
@pytest.mark.parametrize("t", HALF)
@pytest.mark.parametrize("rows,nin,nout", [(200003, 2304, 2304), (120007, 64, 19000), (150001, 130, 19000)])
def test_weights_gradient_of_a_long_group(cuda, rows, nin, nout, t):
    """Most rows in one group, which is a single unit of work: there are tiles of the result enough for all SMs."""
    sizes = [70, rows - 170, 100]
    o = torch.tensor([0, 70, rows - 100, rows], device="cuda")
    x, dy = positive(rows, nin, t=t, seed=1), positive(rows, nout, t=t, seed=2, most=0.25)
    w = torch.zeros(3, nin, nout, device="cuda", dtype=t, requires_grad=True)
    (dw,) = torch.autograd.grad(scn.grouped_product(x, w, o), [w], dy)
    for g, first in enumerate((0, 70, rows - 100)):
        r = slice(first, first + sizes[g])
        for c in (slice(0, 64), slice(nout - 40, nout)):
            check(dw[g][:, c], x[r].double().T @ dy[r, c].double(), sizes[g] / 4096 + 1, t)


@pytest.mark.parametrize("t", HALF)
@pytest.mark.parametrize("rows,nout", [(130, 200), (2600, 2304)])
def test_many_planes(cuda, rows, nout, t):
    """A forward sum, and the input's gradient, over 131 072 planes"""
    k = 131072
    o = torch.tensor([0, rows - 30, rows], device="cuda")
    x, w = positive(rows, k, t=t, seed=1), positive(2, k, nout, t=t, seed=2, most=0.25)
    y = scn.grouped_product(x, w, o)
    for g, r in enumerate((slice(0, rows - 30), slice(rows - 30, rows))):
        check(y[r, :64], x[r].double() @ w[g, :, :64].double(), k / 4096 + 1, t)
    del y
    v = w.transpose(1, 2).contiguous()  # [2, nout, k]: its gradient's sums run over k
    z = torch.zeros(rows, nout, device="cuda", dtype=t, requires_grad=True)
    (dz,) = torch.autograd.grad(scn.grouped_product(z, v, o), [z], x)
    for g, r in enumerate((slice(0, rows - 30), slice(rows - 30, rows))):
        check(dz[r, :64], x[r].double() @ w[g, :, :64].double(), k / 4096 + 1, t)


@pytest.mark.parametrize("rows,nout", [(130, 200), (2600, 2304)])
def test_many_planes_in_eight_bits(cuda, rows, nout):
    k, t = 262144, torch.float16
    o = torch.tensor([0, rows - 30, rows], device="cuda")
    q, w = positive(rows, k, t=torch.float8_e4m3fn, seed=1, most=400.0), positive(2, nout, k, t=torch.float8_e4m3fn, seed=2, most=400.0)
    scale, ws = positive(rows, t=torch.float32, seed=3) * 1e-5 + 1e-5, positive(2, nout, t=torch.float32, seed=4) * 1e-2 + 1e-2
    y = scn.grouped_product_quantized(q, scale, w, ws, o, out_dtype=t)
    for g, r in enumerate((slice(0, rows - 30), slice(rows - 30, rows))):
        want = q[r].double() @ w[g, :64].double().T * scale[r].double()[:, None] * ws[g, :64].double()
        check(y[r, :64], want, k / 8192 + 1, t, others=2 * E)


@pytest.mark.parametrize("t", HALF)
def test_lengths_around_a_hand_over(cuda, t):
    """Groups that end before, at and behind a hand-over, and in the step after it, beside short ones"""
    sizes = [4096, 4095, 4097, 8192, 8193, 8191, 1, 0, 12288, 64, 12289, 30001, 4160]
    rows = sum(sizes)
    o = torch.tensor([sum(sizes[:i]) for i in range(len(sizes) + 1)], device="cuda")
    for nin, nout in ((600, 10000), (40, 19000)):
        x, dy = (torch.randn(rows, c, device="cuda", generator=torch.Generator(device="cuda").manual_seed(c)).to(t) for c in (nin, nout))
        w = torch.zeros(len(sizes), nin, nout, device="cuda", dtype=t, requires_grad=True)
        dw, = torch.autograd.grad(scn.grouped_product(x, w, o), [w], dy)
        for g, n in enumerate(sizes):
            a, d = x[o[g]:o[g + 1]].double(), dy[o[g]:o[g + 1], -70:].double()
            want, size = a.T @ d, a.abs().T @ d.abs()
            room = (2 * (min(n, 4096) / 16 + 1) + n / 4096 + 1) * E
            tiny = torch.finfo(t).smallest_normal * torch.finfo(t).eps
            assert bool(((dw[g][:, -70:].double() - want).abs() <= torch.finfo(t).eps / 2 * want.abs() * (1 + 1e-6) + room * size + tiny).all()), g
        again, = torch.autograd.grad(scn.grouped_product(x, w, o), [w], dy)
        assert torch.equal(dw, again)
        scn.poll_errors()


@pytest.mark.parametrize("t", [torch.float32, *HALF])
@pytest.mark.parametrize("rows,nout", [(130, 203), (2600, 2303), (2600, 2320), (19000, 264)])
def test_every_way_out(cuda, rows, nout, t):
    """Results of all types, in rows of any alignment, with a bias: 16-bit operands (but for float32 results, whose sums are short), and 8-bit
    ones"""
    k = 20000
    o = torch.tensor([3, 80, rows - 1], device="cuda")
    parts = ((slice(3, 80), 0), (slice(80, rows - 1), 1))
    half = t if t != torch.float32 else torch.float16
    x, w, b = positive(rows, k, t=half, seed=1), positive(2, k, nout, t=half, seed=2, most=0.25), positive(2, nout, t=half, seed=3, most=900.0)
    y = scn.grouped_product(x, w, o, b, out_dtype=t)
    q, v = positive(rows, k, t=torch.float8_e4m3fn, seed=4, most=400.0), positive(2, nout, k, t=torch.float8_e4m3fn, seed=5, most=400.0)
    scale, ws = positive(rows, t=torch.float32, seed=6) * 1e-5 + 1e-5, positive(2, nout, t=torch.float32, seed=7) * 1e-2 + 1e-2
    z = scn.grouped_product_quantized(q, scale, v, ws, o, b, out_dtype=t)
    for r, g in parts:
        for c in (slice(0, 70), slice(nout - 70, nout)):
            check(y[r, c], x[r].double() @ w[g, :, c].double() + b[g, c].double(), k / 4096 + 1, t, others=2 * E)
            check(z[r, c], q[r].double() @ v[g, c].double().T * scale[r].double()[:, None] * ws[g, c].double() + b[g, c].double(), k / 8192 + 1, t, others=4 * E)
    outside = torch.tensor([0, 1, 2, rows - 1], device="cuda")
    assert bool((y[outside] == 0).all()) and bool((z[outside] == 0).all())
    scn.poll_errors()


@pytest.mark.parametrize("t", HALF)
def test_many_groups_of_many_planes(cuda, t):
    """Tiles of one block and 256 columns: groups too small for two blocks to a tile, 300 and 100 columns for narrower ones"""
    k, groups = 9000, 90
    o = torch.arange(groups + 1, device="cuda") * 31
    rows = int(o[-1])
    x = positive(rows, k, t=t, seed=1)
    for nout in (1000, 300, 100):
        w = positive(groups, k, nout, t=t, seed=2, most=0.25)
        y = scn.grouped_product(x, w, o)
        v, z = w.transpose(1, 2).contiguous(), torch.zeros(rows, nout, device="cuda", dtype=t, requires_grad=True)
        (dz,) = torch.autograd.grad(scn.grouped_product(z, v, o), [z], x)
        for g in (0, 1, 44, 89):
            r = slice(31 * g, 31 * g + 31)
            want = x[r].double() @ w[g].double()
            check(y[r], want, k / 4096 + 1, t)
            check(dz[r], want, k / 4096 + 1, t)
    q, v = positive(rows, 2 * k, t=torch.float8_e4m3fn, seed=4, most=400.0), positive(groups, 1000, 2 * k, t=torch.float8_e4m3fn, seed=5, most=400.0)
    scale, ws = positive(rows, t=torch.float32, seed=6) * 1e-5 + 1e-5, positive(groups, 1000, t=torch.float32, seed=7) * 1e-2 + 1e-2
    y = scn.grouped_product_quantized(q, scale, v, ws, o, out_dtype=t)
    for g in (0, 44, 89):
        r = slice(31 * g, 31 * g + 31)
        check(y[r], q[r].double() @ v[g].double().T * scale[r].double()[:, None] * ws[g].double(), 2 * k / 8192 + 1, t, others=4 * E)


@pytest.mark.parametrize("nin,nout", [(64, 64), (100, 128), (128, 72)])
def test_millions_of_rows(cuda, nin, nout):
    """A result of a tile or two: units of a 300th of the rows, each of them long"""
    rows, t = 3000017, torch.bfloat16
    o = torch.tensor([0, 9001, rows - 11, rows], device="cuda")
    x, dy = positive(rows, nin, t=t, seed=1), positive(rows, nout, t=t, seed=2, most=0.25)
    w, b = torch.zeros(3, nin, nout, device="cuda", dtype=t, requires_grad=True), torch.zeros(3, nout, device="cuda", dtype=t, requires_grad=True)
    dw, db = torch.autograd.grad(scn.grouped_product(x, w, o, b), [w, b], dy)
    for g in range(3):
        r = slice(int(o[g]), int(o[g + 1]))
        want, sums = torch.zeros(nin, nout, device="cuda", dtype=torch.float64), torch.zeros(nout, device="cuda", dtype=torch.float64)
        for s in range(r.start, r.stop, 500000):
            e = min(r.stop, s + 500000)
            want += x[s:e].double().T @ dy[s:e].double()
            sums += dy[s:e].double().sum(0)
        check(dw[g], want, 3, t, others=300 * E)  # (the partial sums of 300 units, one after the other)
        check(db[g], sums, 0, t, others=(10200 / 64 + 300 + 20) * E)
