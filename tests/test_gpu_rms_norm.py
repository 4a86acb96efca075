"""Row norms on the GPU against the formulas in 64 bits.

Tolerances.  Results of type t are rounded once: u = eps(t) / 2 of the value.  What precedes that rounding is fp32, e = 2^-24: the
sum of squares of n values is n / threads additions to a thread and some ten more (relative error below (32 + 10) e for
all shapes here but the longest rows, 2 x that for them), which the root halves; the root, the division and two products
add 4 e: 32 e with room.  A sum of rows is compared relative to the sum of its terms' sizes."""
import pytest
import torch

import sparseconvnet_b200 as scn

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]
E = 2.0 ** -24


def unit(t):
    return torch.finfo(t).eps / 2


def near(got, want, size, e, t):
    """|got - want| <= u |want| + e size, and a type's smallest step"""
    d = (got.double() - want).abs()
    most = unit(t) * want.abs() * (1 + 1e-6) + e * size + torch.finfo(t).smallest_normal * torch.finfo(t).eps
    assert bool((d <= most).all()), (float((d / most).max()), d.argmax())


def formula(x, w, r, eps):
    s = x.double() if r is None else (x.float() + r.float()).to(x.dtype).double()
    k = (s.square().mean(-1, keepdim=True) + eps).rsqrt()
    return s, k, s * k * (1 if w is None else w.double())


def rows(n, c, t, seed=0, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(n, c, generator=g, device="cuda") * scale).to(t)


SHAPES = [(1, 1), (1, 16), (5, 3), (33, 17), (2, 30), (1000, 96), (257, 224), (64, 1001), (3, 2048), (19, 4096), (7, 5000), (2, 16384), (3, 16391),
          (2, 40000)]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("n,c", SHAPES)
def test_forward_and_gradients(cuda, n, c, t):
    x, r, w = rows(n, c, t, 1).requires_grad_(), rows(n, c, t, 2, 3.0).requires_grad_(), (1 + 0.2 * rows(1, c, torch.float32, 3)[0]).requires_grad_()
    dy, ds = rows(n, c, t, 4), rows(n, c, t, 5)
    y, s = scn.rms_norm(x, w, residual=r, eps=1e-5)
    gx, gr, gw = torch.autograd.grad([y, s], [x, r, w], [dy, ds])
    s_, k, y_ = formula(x.detach(), w.detach(), r.detach(), 1e-5)
    assert y.dtype == s.dtype == t and torch.equal(s.double(), s_)
    long = 2 if c > 16384 else 1
    near(y.detach(), y_, y_.abs(), 32 * E * long, t)
    d, w_ = dy.double() * w.detach().double(), w.detach().double()
    along = (d * s_ * k).mean(-1, keepdim=True)
    size = k * (d.abs() + (s_ * k).abs() * (d * s_ * k).abs().mean(-1, keepdim=True)) + ds.double().abs()
    near(gx, k * (d - s_ * k * along) + ds.double(), size, 64 * E * long, t)
    assert torch.equal(gx, gr)
    terms = dy.double() * s_ * k
    near(gw, terms.sum(0), terms.abs().sum(0), 64 * E, torch.float32)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("out", TYPES)
def test_types_of_the_result(cuda, t, out):
    x, w = rows(37, 80, t, 1).requires_grad_(), rows(1, 80, torch.float32, 2)[0]
    y = scn.rms_norm(x, w, out_dtype=out)
    y_ = formula(x.detach(), w, None, 1e-6)[2]
    assert y.dtype == out
    near(y.detach(), y_, y_.abs(), 32 * E, out)
    dy = rows(37, 80, out, 3)
    (gx,) = torch.autograd.grad(y, [x], dy)
    s, k, _ = formula(x.detach(), w, None, 1e-6)
    d = dy.double() * w.double()
    near(gx, k * (d - s * k * (d * s * k).mean(-1, keepdim=True)), k * (d.abs() + (s * k).abs() * (d * s * k).abs().mean(-1, keepdim=True)), 64 * E, t)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("n,c", [(1, 1), (5, 3), (33, 18), (300, 96), (9, 4096), (3, 5003), (2, 16400)])
def test_eight_bits(cuda, n, c, t, residual):
    x, w, r = rows(n, c, t, 1), 1 + 0.2 * rows(1, c, torch.float32, 2)[0], rows(n, c, t, 3) if residual else None
    made = scn.rms_norm_quantized(x, w, residual=r)
    s_, _, y_ = formula(x, w, r, 1e-6)
    q, scale = made[:2]
    assert q.dtype == torch.float8_e4m3fn and q.shape == x.shape and scale.shape == (n,) and scale.dtype == torch.float32
    if residual:
        assert torch.equal(made[2].double(), s_)
    most = y_.abs().amax(1)
    assert bool(((scale.double() * 448 - most).abs() <= 64 * E * most).all())
    assert bool((q.float().abs().amax(1) == 448).all())
    got = q.double() * scale.double()[:, None]
    # e4m3: half a step is 2^-4 of a normal value, 2^-10 below 2^-6; the value itself is 70 E off at most
    assert bool(((got - y_).abs() <= y_.abs() * (2.0 ** -4 + 70 * E) + 2.0 ** -10 * scale.double()[:, None]).all())


def test_rows_that_are_zero_huge_or_not_numbers(cuda):
    x = rows(6, 64, torch.float32, 1)
    x[0] = 0
    x[1, 5] = float("nan")
    x[2, 7] = float("inf")
    x[3] *= 1e-30
    x[4] *= 1e15
    y, q, scale = scn.rms_norm(x), *scn.rms_norm_quantized(x)
    assert bool((y[0] == 0).all()) and bool((q[0].float() == 0).all()) and 0 < float(scale[0]) < 1e-30
    assert bool(y[1].isnan().all()) and bool(q[1].float().isnan().all()) and bool(scale[1].isnan())
    plain = x[2] * torch.rsqrt((x[2] * x[2]).mean() + 1e-6)
    assert torch.equal(y[2].isnan(), plain.isnan()) and bool(scale[2].isnan())
    s, k, y_ = formula(x, None, None, 1e-6)
    near(y[3:], y_[3:], y_[3:].abs(), 32 * E, torch.float32)
    assert bool(y[5].isfinite().all())   # neighbours of such rows are as ever


@pytest.mark.parametrize("t", TYPES)
def test_strides_shapes_and_alignment(cuda, t):
    base = rows(40, 100, t, 1)
    w = rows(1, 64, torch.float32, 2)[0]
    for x in (base[:, 4:68], base[:, 3:67], base[::2, 8:72], base[:1, 8:72].expand(7, 64), base[:, :64].reshape(4, 10, 64), base.t()[:64, :].t(), base[:, 8:72].reshape(2, 20, 64)[:, 1:7], base[3, :64]):
        y = scn.rms_norm(x, w)
        y_ = formula(x, w, None, 1e-6)[2]
        assert y.shape == x.shape and y.is_contiguous()
        near(y, y_, y_.abs(), 32 * E, t)
    out, s = scn.rms_norm(base[:, 3:67], w, residual=base[:, 30:94])
    s_, _, y_ = formula(base[:, 3:67], w, base[:, 30:94], 1e-6)
    assert torch.equal(s.double(), s_)
    near(out, y_, y_.abs(), 32 * E, t)


def test_broadcast_rows_and_shared_inputs(cuda):
    """The gradient of a row that was broadcast is the sum over its copies; a tensor that is both operands gets both parts."""
    x = rows(1, 48, torch.float32, 1).requires_grad_()
    y = scn.rms_norm(x.expand(9, 48))
    dy = rows(9, 48, torch.float32, 2)
    (gx,) = torch.autograd.grad(y, [x], dy)
    s, k, _ = formula(x.detach(), None, None, 1e-6)
    d = dy.double()
    each = k * (d - s * k * (d * s * k).mean(-1, keepdim=True))
    near(gx, each.sum(0, keepdim=True), (k * (d.abs() + (s * k).abs() * (d * s * k).abs().mean(-1, keepdim=True))).sum(0, keepdim=True), 64 * E, torch.float32)
    y, total = scn.rms_norm(x, residual=x)
    (both,) = torch.autograd.grad([total], [x], [torch.ones_like(x)])
    assert torch.equal(both, torch.full_like(x, 2))
    leaf = x.detach().clone().requires_grad_()
    other = rows(1, 48, torch.float32, 5).requires_grad_()
    y, total = scn.rms_norm(leaf, residual=other)
    (y.sum() + total.sum()).backward()
    assert leaf.grad.data_ptr() != other.grad.data_ptr() and torch.equal(leaf.grad, other.grad)


def test_empty_rows(cuda):
    x, w = torch.zeros(0, 24, device=cuda, requires_grad=True), torch.ones(24, device=cuda, requires_grad=True)
    y = scn.rms_norm(x, w)
    gx, gw = torch.autograd.grad(y, [x, w], torch.zeros(0, 24, device=cuda))
    assert y.shape == gx.shape == (0, 24) and bool((gw == 0).all())
    q, scale = scn.rms_norm_quantized(x.detach(), w.detach())
    assert q.shape == (0, 24) and scale.shape == (0,)


def test_gradients_against_differences(cuda):
    x, w = rows(4, 11, torch.float32, 1).requires_grad_(), rows(1, 11, torch.float32, 2)[0].requires_grad_()
    dy = rows(4, 11, torch.float32, 3)
    gx, gw = torch.autograd.grad(scn.rms_norm(x, w, eps=0.1), [x, w], dy)
    at = lambda a, b: float((formula(a, b, None, 0.1)[2] * dy.double()).sum())  # noqa: E731
    h = 1e-4  # central differences in 64 bits: h^2 of third derivatives of some tens, 1e-7
    for i in range(4):
        for j in (0, 5, 10):
            up, down = x.detach().double().clone(), x.detach().double().clone()
            up[i, j] += h
            down[i, j] -= h
            assert abs((at(up, w.detach()) - at(down, w.detach())) / (2 * h) - float(gx[i, j])) < 2e-5
    for j in range(11):
        up, down = w.detach().double().clone(), w.detach().double().clone()
        up[j] += h
        down[j] -= h
        assert abs((at(x.detach(), up) - at(x.detach(), down)) / (2 * h) - float(gw[j])) < 2e-5


def test_one_gradient_only(cuda):
    """Either of the two results, or either operand, may be the only one with a gradient."""
    x, r, w = rows(5, 32, torch.float32, 1), rows(5, 32, torch.float32, 2), rows(1, 32, torch.float32, 3)[0]
    d = rows(5, 32, torch.float32, 4)
    full = torch.autograd.grad(scn.rms_norm(x.requires_grad_(), w.requires_grad_(), residual=r)[0], [x, w], d)
    x.requires_grad_(False)
    (gw,) = torch.autograd.grad(scn.rms_norm(x, w, residual=r)[0], [w], d)
    assert torch.equal(gw, full[1])
    w.requires_grad_(False)
    r.requires_grad_()
    y, s = scn.rms_norm(x, w, residual=r)
    assert torch.equal(torch.autograd.grad(y, [r], d, retain_graph=True)[0], full[0])
    assert torch.equal(torch.autograd.grad(s, [r], d)[0], d)


def test_streams_and_graphs(cuda):
    x, w = rows(300, 96, torch.bfloat16, 1).requires_grad_(), rows(1, 96, torch.float32, 2)[0].requires_grad_()
    dy = rows(300, 96, torch.bfloat16, 3)

    def step():
        y = scn.rms_norm(x, w)
        return (y.detach(),) + torch.autograd.grad(y, [x, w], dy)  # (torch captures no backward pass beside a living graph of its leaves)

    want = [t.clone() for t in step()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            got = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    with torch.no_grad():
        x.copy_(x.flip(0))
        dy.copy_(dy.flip(0))
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got[0], want[0].flip(0)) and torch.equal(got[1], want[1].flip(0))


def test_refusals(cuda):
    x = rows(4, 16, torch.float32, 1)
    for bad, said in ((dict(weight=torch.ones(15, device=cuda)), "entries"), (dict(weight=torch.ones(16)), "CUDA"),
                      (dict(residual=x[:3]), "residual"), (dict(residual=x.half()), "residual"), (dict(eps=-1.0), "eps")):
        with pytest.raises(RuntimeError, match=said):
            scn.rms_norm(x, **bad)
    with pytest.raises(RuntimeError, match="float32, bfloat16 or float16"):
        scn.rms_norm(x.double())
    with pytest.raises(RuntimeError, match="plane"):
        scn.rms_norm(torch.zeros(4, 0, device=cuda))
    with pytest.raises(RuntimeError, match="no gradient"):
        scn.rms_norm_quantized(x.clone().requires_grad_())
    y = scn.rms_norm(x.clone().requires_grad_()).sum()
    leaf = x.clone().requires_grad_()
    with pytest.raises(RuntimeError, match="again"):
        torch.autograd.grad(scn.rms_norm(leaf).sum(), [leaf], create_graph=True)
    del y


def test_more_than_2_31_values(cuda):
    """Rows are independent, so those at the end have the bits that they have alone."""
    n, c = 530001, 4096
    x, r = torch.empty(n, c, device=cuda, dtype=torch.bfloat16).normal_(), rows(3, c, torch.bfloat16, 1)
    x[-3:] = rows(3, c, torch.bfloat16, 2)
    y, s = scn.rms_norm(x, residual=x)
    want, sums = scn.rms_norm(x[-3:].clone(), residual=x[-3:].clone())
    assert torch.equal(y[-3:], want) and torch.equal(s[-3:], sums)
    del y, s
    q, scale = scn.rms_norm_quantized(x)
    want, scales = scn.rms_norm_quantized(x[-3:].clone())
    assert torch.equal(q[-3:].float(), want.float()) and torch.equal(scale[-3:], scales)
    del q
    x.requires_grad_()
    y = scn.rms_norm(x)
    (gx,) = torch.autograd.grad(y, [x], y.detach())
    part = x.detach()[-3:].clone().requires_grad_()
    out = scn.rms_norm(part)
    (want,) = torch.autograd.grad(out, [part], out.detach())
    assert torch.equal(gx[-3:], want) and r.shape == want.shape


def test_modules_over_sites(cuda):
    import numpy as np
    rng = np.random.default_rng(0)
    coords = torch.from_numpy(np.unique(rng.integers(0, 20, (500, 3)), axis=0))
    feats = torch.randn(len(coords), 24, device=cuda, requires_grad=True)
    inp = scn.InputLayer(3, 20)([coords, feats])
    block = scn.Sequential().add(scn.ConcatTable().add(scn.SubmanifoldConvolution(3, 24, 24, 3, False)).add(scn.Identity())).add(
        scn.AddRMSNormalization(24)).to(cuda)
    norm, total = block(inp)
    branch = block[0][0](inp).features + inp.features
    assert torch.equal(total.features, branch)
    near(norm.features.detach(), formula(branch.detach(), None, None, 1e-6)[2], formula(branch.detach(), None, None, 1e-6)[2].abs(), 32 * E, torch.float32)
    scn.RMSNormalization(24).to(cuda)(norm).features.sum().backward()
    assert feats.grad is not None and block[1].weight.grad is not None
