"""Grouped products on the GPU against the formulas in 64 bits.

Tolerances, relative to S, the sum of the sizes of a result's products.  The tensor core cuts its running sum off at every
instruction of 16 products: at most 2^-23 of the sum, once for the products' alignment and once for the addition, so
2 (n / 16 + 1) 2^-23 S for n products.  fp32 in three parts: hand-overs after 16 instructions of the largest products, their sums
in fp32: (2 * 16 + n / 256 + 4) 2^-23 S, the products left out are 2^-25 S; two parts leave out 3 * 2^-18 S; one part rounds
both operands, 2 * 2^-9 S.  A result of type t is rounded once: eps(t) / 2 of it."""
import pytest
import torch

import sparseconvnet_b200 as scn

pytestmark = pytest.mark.gpu
E = 2.0 ** -23
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def room(n, t, precision="fp32"):
    if t != torch.float32:
        return 2 * (n / 16 + 1) * E
    return {"fp32": 2.0 ** -25, "tf32x3": 3 * 2.0 ** -18, "tf32": 3 * 2.0 ** -18, "bf16": 2.0 ** -8}[precision] + (2 * 16 + n / 256 + 4) * E


def near(got, want, size, e, t):
    d = (got.double() - want).abs()
    most = torch.finfo(t).eps / 2 * want.abs() * (1 + 1e-6) + e * size + torch.finfo(t).smallest_normal * torch.finfo(t).eps
    assert bool((d <= most).all()), (float((d / most.clamp_min(1e-300)).max()), int(d.argmax()))


def formula(x, w, offsets, b=None, dy=None):
    x, w, o = x.detach().double(), w.detach().double(), offsets.tolist()
    y, size = x.new_zeros(len(x), w.size(2)), x.new_zeros(len(x), w.size(2))
    made = dict(dx=torch.zeros_like(x), dxs=torch.zeros_like(x), dw=torch.zeros_like(w), dws=torch.zeros_like(w),
                db=w.new_zeros(w.size(0), w.size(2)), dbs=w.new_zeros(w.size(0), w.size(2)))
    for g in range(len(w)):
        r = slice(o[g], o[g + 1])
        y[r], size[r] = x[r] @ w[g], x[r].abs() @ w[g].abs()
        if b is not None:
            y[r] += b[g].detach().double()
            size[r] += b[g].detach().double().abs()
        if dy is not None:
            d = dy[r].double()
            made["dx"][r], made["dxs"][r] = d @ w[g].T, d.abs() @ w[g].abs().T
            made["dw"][g], made["dws"][g] = x[r].T @ d, x[r].abs().T @ d.abs()
            made["db"][g], made["dbs"][g] = d.sum(0), d.abs().sum(0)
    return dict(made, y=y, size=size)


def normal(*shape, t=torch.float32, seed=0):
    return torch.randn(*shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda").to(t)


def offsets_of(sizes, before=0, wide=True):
    o = [before]
    for s in sizes:
        o.append(o[-1] + s)
    return torch.tensor(o, device="cuda", dtype=torch.int64 if wide else torch.int32)


# (sizes of the groups, rows in front, rows behind, nIn, nOut)
SHAPES = [([1], 0, 0, 1, 1), ([1, 0, 2], 0, 0, 16, 16), ([5], 3, 2, 8, 24), ([128, 128], 0, 0, 64, 64), ([129, 0, 127, 1], 0, 5, 64, 96),
          ([33, 64, 0, 0, 200], 7, 0, 72, 136), ([300, 1, 17], 0, 0, 20, 3), ([40, 41], 0, 1, 3, 20), ([700, 90], 1, 1, 130, 257),
          ([64] * 9, 0, 0, 128, 320), ([1000, 2500, 37], 0, 0, 256, 128), ([20, 31], 0, 0, 1024, 512), ([0, 0], 4, 9, 32, 32),
          ([3] * 100, 0, 0, 48, 40), ([4000], 0, 0, 40, 64),
          # tiles of two blocks: groups that end in the first and in the second block's rows, inside and at the end of a stage
          ([3000, 0, 5000, 2900], 5, 3, 264, 300), ([2560, 2816, 4096, 1024], 0, 0, 512, 256), ([10001, 77, 1, 640], 0, 0, 136, 1000),
          ([9000, 130], 1, 1, 1000, 264),
          # fp32 rows split in the kernel: up to 256 planes, weights' gradients of up to 128 x 256, with and without room for the bias
          ([700, 0, 257, 256, 1], 3, 2, 128, 256), ([1, 15, 16, 17, 255, 300], 2, 0, 127, 200), ([500, 40], 0, 1, 257, 100), ([600, 70], 0, 0, 100, 260)]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("sizes,front,behind,nin,nout", SHAPES)
def test_forward_and_gradients(cuda, sizes, front, behind, nin, nout, t):
    o = offsets_of(sizes, front, wide=nin % 3 != 0)
    n = int(o[-1]) + behind
    x, w = normal(n, nin, t=t, seed=1), normal(len(sizes), nin, nout, t=t, seed=2)
    b, dy = normal(len(sizes), nout, t=t, seed=3), normal(n, nout, t=t, seed=4)
    outside = torch.ones(n, dtype=torch.bool, device="cuda")
    outside[front:n - behind] = False
    want = formula(x, w, o, b, dy)
    x[outside], dy[outside] = float("nan"), float("nan")  # rows of no group: nothing of them reaches a result
    for p in (x, w, b):
        p.requires_grad_()
    y = scn.grouped_product(x, w, o, b)
    assert y.dtype == t
    near(y.detach(), want["y"], want["size"], room(nin, t), t)
    dx, dw, db = torch.autograd.grad(y, [x, w, b], dy)
    assert bool((y[outside] == 0).all()) and bool((dx[outside] == 0).all())
    near(dx, want["dx"], want["dxs"], room(nout, t), t)
    longest = max(sizes)
    near(dw, want["dw"], want["dws"], room(longest, t) + 8 * E, t)
    near(db, want["db"], want["dbs"], (longest / 256 + 16) * E, t)
    scn.poll_errors()


@pytest.mark.parametrize("precision", ["fp32", "tf32x3", "tf32", "bf16"])
def test_precisions_of_float32(cuda, precision):
    o = offsets_of([200, 0, 130, 5])
    x, w, dy = normal(335, 200, seed=1).requires_grad_(), normal(4, 200, 72, seed=2).requires_grad_(), normal(335, 72, seed=3)
    want = formula(x, w, o, None, dy)
    try:
        scn.set_precision(precision)
        scn.set_backward_precision(precision)
        y = scn.grouped_product(x, w, o)
        dx, dw = torch.autograd.grad(y, [x, w], dy)
    finally:
        scn.set_precision("fp32")
        scn.set_backward_precision("fp32")
    near(y.detach(), want["y"], want["size"], room(200, torch.float32, precision), torch.float32)
    near(dx, want["dx"], want["dxs"], room(72, torch.float32, precision), torch.float32)
    near(dw, want["dw"], want["dws"], room(200, torch.float32), torch.float32)


@pytest.mark.parametrize("t", [torch.bfloat16, torch.float16])
def test_float32_results_of_16_bits(cuda, t):
    o = offsets_of([100, 200])
    x, w, dy = normal(300, 1000, t=t, seed=1).requires_grad_(), normal(2, 1000, 136, t=t, seed=2).requires_grad_(), normal(300, 136, seed=3)
    y = scn.grouped_product(x, w, o, out_dtype=torch.float32)
    want = formula(x, w, o, None, dy.to(t))
    assert y.dtype == torch.float32
    near(y.detach(), want["y"], want["size"], (2 * 16 + 1000 / 256 + 4) * E, torch.float32)
    dx, dw = torch.autograd.grad(y, [x, w], dy)
    assert dx.dtype == dw.dtype == t
    near(dx, want["dx"], want["dxs"], room(136, t), t)
    near(dw, want["dw"], want["dws"], room(200, t), t)


@pytest.mark.parametrize("out", TYPES)
@pytest.mark.parametrize("sizes,front,behind,nin,nout", SHAPES)
def test_eight_bits(cuda, sizes, front, behind, nin, nout, out):
    o = offsets_of(sizes, front)
    n = int(o[-1]) + behind
    q, scale = scn.rms_norm_quantized(normal(n, nin, seed=1))
    w, ws = scn.quantize_group_weights(normal(len(sizes), nin, nout, seed=2))
    b = normal(len(sizes), nout, t=out, seed=3)
    y = scn.grouped_product_quantized(q, scale, w, ws, o, b, out_dtype=out)
    want = formula(q.double() * scale.double()[:, None], (w.double() * ws.double()[:, :, None]).transpose(1, 2), o, b)
    assert y.dtype == out and y.shape == (n, nout)
    near(y, want["y"], want["size"], 2 * (nin / 32 + 4) * E, out)
    assert bool((y[:front] == 0).all()) and bool((y[n - behind:] == 0).all())


def test_groups_do_not_reach_into_each_other(cuda):
    """A NaN or an infinity in one group's rows or weights stays there, in every gradient."""
    for t in (torch.float32, torch.bfloat16):
        o = offsets_of([70, 33, 90])
        x, w, dy = normal(193, 64, t=t, seed=1), normal(3, 64, 64, t=t, seed=2), normal(193, 64, t=t, seed=3)
        x[70:103] = float("nan")
        x[75, 3] = float("inf")
        dy[70:103] = float("inf")
        w[1] = float("nan")
        x.requires_grad_()
        w.requires_grad_()
        y = scn.grouped_product(x, w, o)
        dx, dw = torch.autograd.grad(y, [x, w], dy)
        for r in (y, dx):
            assert bool(r[:70].isfinite().all()) and bool(r[103:].isfinite().all()) and bool(r[70:103].isnan().all())
        assert bool(dw[0].isfinite().all()) and bool(dw[2].isfinite().all()) and bool(dw[1].isnan().all())


def test_large_and_small_values_of_float32(cuda):
    """Values near the ends of the range keep their bits: their bf16 parts have the same exponents."""
    o = offsets_of([40])
    for scale_x, scale_w in ((1e38, 1e-30), (1e-30, 1e20), (3e-20, 3e-10), (1e15, 1e15)):
        x, w = normal(40, 96, seed=1).clamp(-3, 3) * scale_x, normal(1, 96, 40, seed=2) * scale_w
        want = formula(x, w, o)
        near(scn.grouped_product(x, w, o), want["y"], want["size"], room(96, torch.float32), torch.float32)
    x = torch.full((40, 96), torch.finfo(torch.float32).max, device="cuda")
    assert bool(scn.grouped_product(x, torch.full((1, 96, 8), 2.0 ** -10, device="cuda"), o).isfinite().all())


def test_strides_and_alignment(cuda):
    o = offsets_of([30, 34])
    w = normal(2, 64, 48, t=torch.bfloat16, seed=2)
    base = normal(70, 200, t=torch.bfloat16, seed=1)
    shifted = torch.empty(2 * 64 * 48 + 1, dtype=torch.bfloat16, device="cuda")[1:].view(2, 64, 48).copy_(w)
    for x in (base[:64, 8:72], base[:64, 3:67], base[1:65, 64:128], base.t()[:64].t()[:64], base[5:6, 8:72].expand(64, 64), base[::1, 100:164][6:]):
        want = formula(x, w, o)
        for weight in (w, shifted, w.transpose(1, 2).contiguous().transpose(1, 2)):
            near(scn.grouped_product(x, weight, o), want["y"], want["size"], room(64, torch.bfloat16), torch.bfloat16)


def test_broadcast_rows_and_weights(cuda):
    """Gradients of operands that were broadcast are summed over the copies."""
    o = offsets_of([4, 5, 6])
    x, w = normal(1, 32, seed=1).requires_grad_(), normal(1, 32, 24, seed=2).requires_grad_()
    dy = normal(15, 24, seed=3)
    y = scn.grouped_product(x.expand(15, 32), w.expand(3, 32, 24), o)
    dx, dw = torch.autograd.grad(y, [x, w], dy)
    d, a, b = dy.double(), x.detach().double(), w.detach().double()[0]
    near(dx, (d @ b.T).sum(0, keepdim=True), (d.abs() @ b.abs().T).sum(0, keepdim=True), room(24, torch.float32) + 16 * E, torch.float32)
    near(dw[0], a.expand(15, 32).T @ d, a.abs().expand(15, 32).T @ d.abs(), room(15, torch.float32) + 4 * E, torch.float32)


def test_offsets_that_make_no_sense_stay_inside(cuda):
    """Offsets outside the rows or in falling order: every group begins at the largest offset so far, within the rows."""
    x, w, dy = normal(300, 64, t=torch.bfloat16, seed=1).requires_grad_(), normal(4, 64, 32, t=torch.bfloat16, seed=2).requires_grad_(), normal(300, 32, t=torch.bfloat16, seed=3)
    for bad, good in (([-5, 100, 50, 400, 7], [0, 100, 100, 300, 300]), ([300, 0, 300, 0, 300], [300] * 5), ([10, 10 ** 12, -10 ** 12, 5, 6], [10, 300, 300, 300, 300])):
        one, two = (torch.tensor(v, device="cuda") for v in (bad, good))
        a, b = (scn.grouped_product(x, w, v) for v in (one, two))
        assert torch.equal(a, b)
        for p, q in zip(torch.autograd.grad(a, [x, w], dy), torch.autograd.grad(b, [x, w], dy)):
            assert torch.equal(p, q)


def test_one_large_group_among_many(cuda):
    """A group that has nearly all rows is split over the SMs; the sum of its parts does not depend on timing."""
    sizes = [3] * 60 + [60001] + [0, 5]
    o = offsets_of(sizes)
    n = int(o[-1])
    for t in (torch.float32, torch.bfloat16):
        x, w, dy = normal(n, 48, t=t, seed=1).requires_grad_(), normal(63, 48, 64, t=t, seed=2).requires_grad_(), normal(n, 64, t=t, seed=3)
        b = normal(63, 64, t=t, seed=4).requires_grad_()
        want = formula(x, w, o, b, dy)
        y = scn.grouped_product(x, w, o, b)
        first = torch.autograd.grad(y, [x, w, b], dy, retain_graph=True)
        near(first[1], want["dw"], want["dws"], room(1024, t) + 128 * E, t)
        near(first[2], want["db"], want["dbs"], 300 * E, t)
        again = torch.autograd.grad(y, [x, w, b], dy)
        assert all(torch.equal(p, q) for p, q in zip(first, again))


def test_most_groups(cuda):
    g = 1024
    sizes = [(7 * i) % 5 for i in range(g)]
    o = offsets_of(sizes, wide=False)
    x, w, dy = normal(int(o[-1]), 16, seed=1).requires_grad_(), normal(g, 16, 16, seed=2).requires_grad_(), normal(int(o[-1]), 16, seed=3)
    y = scn.grouped_product(x, w, o)
    want = formula(x, w, o, None, dy)
    near(y.detach(), want["y"], want["size"], room(16, torch.float32), torch.float32)
    dx, dw = torch.autograd.grad(y, [x, w], dy)
    near(dx, want["dx"], want["dxs"], room(16, torch.float32), torch.float32)
    near(dw, want["dw"], want["dws"], room(16, torch.float32), torch.float32)
    with pytest.raises(Exception, match="groups"):
        scn.grouped_product(x, torch.zeros(1025, 16, 16, device="cuda"), torch.zeros(1026, dtype=torch.int64, device="cuda"))


def test_no_rows(cuda):
    x, w, b = (torch.zeros(s, device="cuda", requires_grad=True) for s in ((0, 8), (2, 8, 16), (2, 16)))
    y = scn.grouped_product(x, w, torch.zeros(3, dtype=torch.int64, device="cuda"), b)
    dx, dw, db = torch.autograd.grad(y, [x, w, b], torch.zeros(0, 16, device="cuda"))
    assert y.shape == (0, 16) and dx.shape == (0, 8) and bool((dw == 0).all()) and bool((db == 0).all())


def test_gradients_against_differences(cuda):
    o = offsets_of([3, 4])
    x, w, b = normal(7, 6, seed=1).requires_grad_(), normal(2, 6, 5, seed=2).requires_grad_(), normal(2, 5, seed=3).requires_grad_()
    dy = normal(7, 5, seed=4)
    grads = torch.autograd.grad(scn.grouped_product(x, w, o, b), [x, w, b], dy)
    at = lambda *p: float((formula(p[0], p[1], o, p[2])["y"] * dy.double()).sum())  # noqa: E731
    for i, g in enumerate(grads):  # the products are linear in each operand: a difference in 64 bits is the gradient itself
        for j in range(g.numel()):
            p = [t.detach().double().clone() for t in (x, w, b)]
            q = [t.clone() for t in p]
            p[i].view(-1)[j] += 0.5
            q[i].view(-1)[j] -= 0.5
            assert abs(at(*p) - at(*q) - float(g.view(-1)[j])) < 1e-4


def test_streams_graphs_and_one_gradient_only(cuda):
    o = offsets_of([60, 0, 140])
    x, w, dy = normal(200, 64, t=torch.bfloat16, seed=1).requires_grad_(), normal(3, 64, 96, t=torch.bfloat16, seed=2).requires_grad_(), normal(200, 96, t=torch.bfloat16, seed=3)

    def step():
        y = scn.grouped_product(x, w, o)
        return (y.detach(),) + torch.autograd.grad(y, [x, w], dy)

    want = [t.clone() for t in step()]
    (dw,) = torch.autograd.grad(scn.grouped_product(x.detach(), w, o), [w], dy)
    (dx,) = torch.autograd.grad(scn.grouped_product(x, w.detach(), o), [x], dy)
    assert torch.equal(dx, want[1]) and torch.equal(dw, want[2])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    o.copy_(offsets_of([0, 200, 0]))  # other groups in the same graph
    graph.replay()
    other = [t.clone() for t in got]
    ref = step()
    assert all(torch.equal(a, b) for a, b in zip(other, ref)) and not torch.equal(other[0], want[0])


def test_two_streams_at_once(cuda):
    sets = [(offsets_of([500, 700]), normal(1200, 256, seed=i), normal(2, 256, 192, seed=10 + i)) for i in range(2)]
    want = [scn.grouped_product(x, w, o) for o, x, w in sets]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in sets], [[], []]
    for _ in range(10):
        for k, (o, x, w) in enumerate(sets):
            with torch.cuda.stream(streams[k]):
                got[k].append(scn.grouped_product(x, w, o))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want[k]) for k in range(2) for g in got[k])


def test_a_thread_of_its_own(cuda):
    """The call may be the first that a thread makes of the GPU, as in autograd's threads."""
    import threading
    o = offsets_of([30, 34])
    x, w, dy = normal(64, 64, t=torch.bfloat16, seed=1).requires_grad_(), normal(2, 64, 64, t=torch.bfloat16, seed=2).requires_grad_(), normal(64, 64, t=torch.bfloat16, seed=3)
    want = scn.grouped_product(x, w, o)
    grads = torch.autograd.grad(want, [x, w], dy)
    torch.cuda.synchronize()
    got = []

    def work():
        with torch.no_grad():
            got.append(scn.grouped_product(x, w, o))

    threads = [threading.Thread(target=work) for _ in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert len(got) == 3 and all(torch.equal(g, want) for g in got) and grads[0].shape == x.shape


def test_refusals(cuda):
    x, w, o = normal(4, 8), normal(2, 8, 16), offsets_of([1, 3])
    for args, said in (((x, w[:1], o), "groups"), ((x, w, o[:1]), "offsets"), ((x, w.half(), o), "type"), ((x, w, o.float()), "int64 or int32"), ((x, w, o.cpu()), "CUDA"),
                       ((x[:, :7], w, o), "nIn"), ((x.double(), w.double(), o), "float32, bfloat16 or float16"), ((x, w, o, normal(2, 15)), "bias"), ((x[0], w, o), "matrix")):
        with pytest.raises(RuntimeError, match=said):
            scn.grouped_product(*args)
    leaf = x.clone().requires_grad_()
    with pytest.raises(RuntimeError, match="again"):
        torch.autograd.grad(scn.grouped_product(leaf, w, o).sum(), [leaf], create_graph=True)
    q, s = scn.rms_norm_quantized(x)
    wq, ws = scn.quantize_group_weights(w)
    for args, said in (((x, s, wq, ws, o), "float8"), ((q, s[:3], wq, ws, o), "per row"), ((q, s, wq, ws[:, :3], o), "weight_scale"), ((q, s.half(), wq, ws, o), "float32"),
                       ((q, s.clone().requires_grad_(), wq, ws, o), "no gradient")):
        with pytest.raises(RuntimeError, match=said):
            scn.grouped_product_quantized(*args)


def test_a_wait_that_runs_out_is_reported(cuda):
    """Leaves out one arrival in one block: the call gives up in bounded time, poll_errors says so, the next call is right."""
    from sparseconvnet_b200._lib import lib
    # one block to a tile, two, and fp32 rows that the kernel splits
    for rows, k, n, t in ((256, 4096, 256, torch.bfloat16), (20000, 4096, 512, torch.bfloat16), (200000, 256, 64, torch.float32)):
        o = offsets_of([rows])
        x, w = normal(rows, k, t=t, seed=1), normal(1, k, n, t=t, seed=2)
        want = scn.grouped_product(x, w, o)
        scn.poll_errors()
        lib.scn_test_drop_barrier_arrival()
        scn.grouped_product(x, w, o)
        with pytest.raises(Exception, match="ran out"):
            scn.poll_errors()
        assert torch.equal(scn.grouped_product(x, w, o), want)
        scn.poll_errors()


def test_more_than_2_31_values(cuda):
    for t, n, k, m in ((torch.bfloat16, 270001, 8192, 64), (torch.float32, 9000001, 256, 16), (torch.bfloat16, 9000001, 16, 256)):
        o = offsets_of([n // 3, n - n // 3 - 4, 4])
        x, w = torch.empty(n, k, device="cuda", dtype=t).normal_(), normal(3, k, m, t=t, seed=1)
        x[-4:] = normal(4, k, t=t, seed=2)
        y = scn.grouped_product(x, w, o)
        near(y[-4:], x[-4:].double() @ w[2].double(), x[-4:].double().abs() @ w[2].double().abs(), room(k, t), t)
        near(y[:4], x[:4].double() @ w[0].double(), x[:4].double().abs() @ w[0].double().abs(), room(k, t), t)
        dy = torch.zeros(n, m, device="cuda", dtype=t)  # a gradient for the last rows only: exact sums of few terms
        dy[-4:] = normal(4, m, t=t, seed=3)
        x.requires_grad_()
        w.requires_grad_()
        dx, dw = torch.autograd.grad(scn.grouped_product(x, w, o), [x, w], dy)
        d = dy[-4:].double()
        near(dx[-4:], d @ w[2].detach().double().T, d.abs() @ w[2].detach().double().abs().T, room(m, t), t)
        near(dw[2], x[-4:].detach().double().T @ d, x[-4:].detach().double().abs().T @ d.abs(), room(4, t), t)
        assert bool((dw[:2] == 0).all()) and bool((dx[:8] == 0).all())
        del x, y, dy, dx


def test_memory_that_runs_out(cuda):
    """An allocation that fails ends the call with an error, and the next one is right."""
    from sparseconvnet_b200._lib import lib
    o = offsets_of([300, 500])
    for t, k, n in ((torch.float32, 64, 96), (torch.float32, 300, 300), (torch.bfloat16, 63, 96)):
        x, w, dy = normal(800, k, t=t, seed=1).requires_grad_(), normal(2, k, n, t=t, seed=2).requires_grad_(), normal(800, n, t=t, seed=3)
        y = scn.grouped_product(x, w, o)
        want = torch.autograd.grad(y, [x, w], dy, retain_graph=True)
        for which in (1, 2, 3):
            lib.scn_test_fail_allocation(which)
            try:
                with pytest.raises(Exception):
                    scn.grouped_product(x.detach(), w.detach(), o)
                    raise RuntimeError("fewer allocations than that")
            finally:
                lib.scn_test_fail_allocation(0)
            assert torch.equal(scn.grouped_product(x, w, o), y)
        got = torch.autograd.grad(y, [x, w], dy)
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_a_block_in_training(cuda):
    """Norm, grouped product and optimiser together, as a residual block over sites uses them: gradients against the same block in
    64 bits, and the optimiser's step on them."""
    torch.manual_seed(0)
    o = offsets_of([150, 90, 260])
    norm, product = scn.AddRMSNormalization(48).to(cuda), scn.GroupedNetworkInNetwork(3, 48, 48, True).to(cuda)
    a, r = normal(500, 48, seed=1).requires_grad_(), normal(500, 48, seed=2)
    wrap = lambda f: scn.SparseConvNetTensor(f, None, None)  # noqa: E731
    normed, total = norm([wrap(a), wrap(r)])
    out = product([normed, o])
    loss = (out.features * total.features).sum()
    loss.backward()
    p = {k: v.detach().double().requires_grad_() for k, v in dict(a=a, n=norm.weight, w=product.weight, b=product.bias).items()}
    s = p["a"] + r.double()
    h = s * (s.square().mean(1, keepdim=True) + 1e-6).rsqrt() * p["n"]
    want = torch.cat([h[x:y] @ p["w"][g] + p["b"][g] for g, (x, y) in enumerate(zip(o.tolist(), o.tolist()[1:]))])
    (want * s).sum().backward()
    for got, k in ((a.grad, "a"), (norm.weight.grad, "n"), (product.weight.grad, "w"), (product.bias.grad, "b")):
        # sums of up to 500 x 48 products of fp32 values with errors of some 30 E each: 1e-5 of the largest with room
        assert float((got.double() - p[k].grad).abs().max()) < 1e-5 * float(p[k].grad.abs().max()) + 1e-5
    params = [norm.weight, product.weight, product.bias]
    before = [q.detach().clone() for q in params]
    scn.AdamW(params, lr=1e-2, weight_decay=0.0).step()
    for q, was in zip(params, before):  # the first step of Adam is lr times the gradient's sign
        big = q.grad.abs() > 1e-3
        assert float(((was - q.detach()) - 1e-2 * q.grad.sign())[big].abs().max()) < 1e-6 * 1e2


def test_a_block_in_8_bits(cuda):
    """Serving: the norm's 8-bit rows go straight into the product."""
    o = offsets_of([37, 0, 91])
    x, r, w = normal(128, 256, t=torch.bfloat16, seed=1), normal(128, 256, t=torch.bfloat16, seed=2), normal(3, 256, 320, seed=3) / 16
    wq, ws = scn.quantize_group_weights(w)
    q, scale, s = scn.rms_norm_quantized(x, residual=r)
    y = scn.grouped_product_quantized(q, scale, wq, ws, o)
    full = scn.grouped_product(scn.rms_norm(s.float()), w, o)
    # both operands rounded to half a step of e4m3, independent errors of uniform distribution: 2 / sqrt(12) 2^-4 relative of the
    # norm of the products at most, and bf16's rounding: 4% of the 2-norm
    assert float((y.float() - full).norm()) < 0.045 * float(full.norm())
