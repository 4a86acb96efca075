"""The AdamW step on the GPU against its formula in 64 bits.

Tolerances, e = 2^-24.  m and v are two products and a sum: 3 e of the sum of the terms' sizes.  The update is m / (sqrt(v) c + eps)
times a rate: root 2 e, c 4 e (expm1 and a root in fp32), quotient 4 e, rate 6 e, and what m and v bring (3 e of the terms,
1.5 e): 24 e of the update with room, 3 e of the parameter.  8-bit moments are a neighbour of the exact value among those of
e4m3: a step of the block's scale at that value, 2^-3 of it or 2^-9 below 2^-6, and a few e."""
import math

import pytest
import torch

import sparseconvnet_b200 as scn

pytestmark = pytest.mark.gpu
E = 2.0 ** -24
SIZES = [1, 0, 3, 255, 256, 257, 4096, 1000, 70001, 2048]
HYPER = dict(lr=3e-3, betas=(0.9, 0.99), eps=1e-6, weight_decay=0.1)


def normal(n, seed, t=torch.float32, scale=1.0):
    return (torch.randn(n, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda") * scale).to(t)


def formula(p, g, m, v, t, lr, betas, eps, weight_decay):
    """In 64 bits: (p, m, v), and the sizes that the tolerances go by"""
    b1, b2 = betas
    p, g = p.double(), g.double()
    m, size = b1 * m + (1 - b1) * g, b1 * m.abs() + (1 - b1) * g.abs()
    v = b2 * v + (1 - b2) * g * g
    low = (v / (1 - b2 ** t)).sqrt() + eps
    return p * (1 - lr * weight_decay) - lr / (1 - b1 ** t) * m / low, m, v, size, lr / (1 - b1 ** t) * size / low


def make(sizes, bits, param=torch.float32, grad=torch.float32, seed=0):
    st = {"params": [normal(n, seed + 7 * i, param) for i, n in enumerate(sizes)],
          "grads": [normal(n, seed + 7 * i + 1, grad, 0.1) for i, n in enumerate(sizes)]}
    m = [normal(n, seed + 7 * i + 2, scale=0.05) for i, n in enumerate(sizes)]
    r = [normal(n, seed + 7 * i + 3, scale=0.1).abs() for i, n in enumerate(sizes)]
    if bits == 32:
        st.update(exp_avgs=m, exp_avg_sqs=[x * x for x in r])
    else:
        for k, xs in (("exp_avg", m), ("exp_avg_sq", r)):
            scales = [torch.stack([b.abs().amax() / 448 for b in x.split(256)]) if len(x) else x.clone() for x in xs]
            st[k + "s"] = [(x / s.repeat_interleave(256)[:len(x)]).to(torch.float8_e4m3fn) for x, s in zip(xs, scales)]
            st[k + "_scales"] = scales
    return st


def wide(st, k, i):
    x = st[k + "s"][i].double()
    return x * st[k + "_scales"][i].double().repeat_interleave(256)[:len(x)] if k + "_scales" in st else x


def copy_of(st):
    return {k: [x.clone() for x in v] for k, v in st.items()}


def steps(n):
    return torch.tensor([n], device="cuda")


def half(t):
    return torch.finfo(t).eps / 2


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("param,grad", [(torch.float32, torch.float32), (torch.float32, torch.bfloat16), (torch.bfloat16, torch.bfloat16),
                                        (torch.float16, torch.float32), (torch.bfloat16, torch.float16)])
@pytest.mark.parametrize("copies", [None, torch.bfloat16, torch.float16])
def test_one_step(cuda, bits, param, grad, copies):
    st = make(SIZES, bits, param, grad)
    was, step = copy_of(st), steps(6)
    made = None if copies is None else [torch.zeros_like(p, dtype=copies) for p in st["params"]]
    scn.adamw_step(step=step, copies=made, **st, **HYPER)
    assert int(step) == 7
    for i, n in enumerate(SIZES):
        r0 = wide(was, "exp_avg_sq", i)
        p, m, v, size, update = formula(was["params"][i], was["grads"][i], wide(was, "exp_avg", i), r0 if bits == 32 else r0 * r0, 7, **HYPER)
        room = 24 * E * update + 3 * E * p.abs()
        off = (st["params"][i].double() - p).abs()
        # (a type's smallest step counts where fp16 is below its normal values)
        assert bool((off <= half(param) * p.abs() * (1 + 1e-6) + room + 2.0 ** -25 * (param == torch.float16)).all()), float((off - room).max())
        if made:
            assert torch.equal(made[i], st["params"][i].to(copies)) or param != torch.float32
            off = (made[i].double() - p).abs()
            assert bool((off <= half(copies) * p.abs() * (1 + 1e-6) + room + 2.0 ** -25 * (copies == torch.float16)).all())
        if bits == 32:
            assert bool(((st["exp_avgs"][i].double() - m).abs() <= 3 * E * size).all())
            assert bool(((st["exp_avg_sqs"][i].double() - v).abs() <= 4 * E * v).all())
        else:
            for k, want in (("exp_avg", m), ("exp_avg_sq", v.sqrt())):
                for block, scale, q in zip(want.split(256), st[k + "_scales"][i], st[k + "s"][i].float().split(256)):
                    most = block.abs().amax()
                    assert abs(float(scale) * 448 - float(most)) <= 8 * E * float(size.abs().amax() if k == "exp_avg" else most)
                    exact = block / scale.double()
                    gap = torch.maximum(2.0 ** (exact.abs().log2().floor() - 3), torch.tensor(2.0 ** -9, device="cuda", dtype=torch.float64))
                    assert bool(((q.double() - exact).abs() <= gap * (1 + 1e-3)).all())
                    if k == "exp_avg_sq":
                        assert bool((q > 0).all())


@pytest.mark.parametrize("bits", [32, 8])
def test_rounding_by_chance_keeps_the_mean(cuda, bits):
    """With a gradient of zero m shrinks by b1 a step, below half a step of 8 bits for b1 = 0.99: rounded to nearest it would stay.
    The mean over n values of one size has a standard deviation of at most half a step / sqrt(n)."""
    n, h = 65536, dict(HYPER, betas=(0.99, 0.999))
    st = make([n], bits)
    st["grads"][0].zero_()
    first = torch.full((n,), 0.7, device="cuda")
    first[::256] = 1.0  # the largest of each block, which is exact
    if bits == 8:
        st["exp_avg_scales"][0].fill_(1 / 448)
        st["exp_avgs"][0].copy_((first * 448).to(torch.float8_e4m3fn))
    else:
        st["exp_avgs"][0].copy_(first)
    step = steps(0)
    start = wide(st, "exp_avg", 0).clone()
    for k in range(1, 11):
        scn.adamw_step(step=step, seed=5, **st, **h)
        got, want = wide(st, "exp_avg", 0), start * 0.99 ** k
        # steps of 2^-3 relative, ten roundings: 6 standard deviations of sqrt(10) / 2 * 2^-3 / sqrt(n) = 4.7e-3, and 20 E
        assert abs(float((got / want).mean()) - 1) < 5e-3


def test_the_same_call_gives_the_same_bits(cuda):
    st = make(SIZES, 8)
    other = copy_of(st)
    for s in (st, other):
        step = steps(41)
        for _ in range(3):
            scn.adamw_step(step=step, seed=9, **s, **HYPER)
    bits = lambda t: t.view(torch.uint8)  # noqa: E731
    assert all(torch.equal(bits(a), bits(b)) for k in st for a, b in zip(st[k], other[k]))
    third = make(SIZES, 8)
    scn.adamw_step(step=steps(41), seed=10, **third, **HYPER)
    fourth = make(SIZES, 8)
    scn.adamw_step(step=steps(41), seed=9, **fourth, **HYPER)
    assert not torch.equal(bits(third["exp_avgs"][8]), bits(fourth["exp_avgs"][8])) and torch.equal(third["params"][8], fourth["params"][8])


@pytest.mark.parametrize("bits", [32, 8])
def test_many_tensors_and_odd_addresses(cuda, bits):
    """More tensors than fit one launch; values at addresses that no vector load takes.  The result of a value depends on its block
    alone, so the same tensors at aligned addresses give the same bits."""
    sizes = [1 + (i * 37) % 700 for i in range(1000)]
    st = make(sizes, bits)
    shifted = {}
    for k, xs in st.items():
        shifted[k] = [torch.empty(len(x) + 1, dtype=x.dtype, device="cuda")[1:] for x in xs]
        for a, b in zip(shifted[k], xs):
            a.copy_(b)
    was, step, other = copy_of(st), steps(0), steps(0)
    scn.adamw_step(step=step, **st, **HYPER)
    scn.adamw_step(step=other, **shifted, **HYPER)
    assert int(step) == int(other) == 1
    for k in st:
        assert all(torch.equal(a.float(), b.float()) for a, b in zip(st[k], shifted[k])), k
    for i in (0, 439, 440, 441, 999):
        r0 = wide(was, "exp_avg_sq", i)
        p, _, _, _, update = formula(was["params"][i], was["grads"][i], wide(was, "exp_avg", i), r0 if bits == 32 else r0 * r0, 1, **HYPER)
        assert bool(((st["params"][i].double() - p).abs() <= 24 * E * update + 3 * E * p.abs()).all())


def test_nothing_behind_a_tensor_is_written(cuda):
    buf = {k: torch.full((1024,), 3.0, device="cuda") for k in ("params", "exp_avgs", "exp_avg_sqs")}
    st = {k: [b[4:304]] for k, b in buf.items()}
    scn.adamw_step(grads=[torch.ones(300, device="cuda")], step=steps(0), **st, **HYPER)
    for b in buf.values():
        assert bool((b[:4] == 3).all()) and bool((b[304:] == 3).all()) and bool((b[4:304] != 3).all())


def test_first_steps_of_a_network(cuda):
    """Moments of zero, both kinds of states, and the smallest betas"""
    for bits in (32, 8):
        for betas in ((0.9, 0.999), (0.0, 0.0), (0.0, 0.9)):
            p = torch.nn.Parameter(normal(3000, 1))
            q = torch.nn.Parameter(p.detach().double())
            h = dict(lr=1e-2, betas=betas, eps=1e-5, weight_decay=0.1)
            opt, ref = scn.AdamW([p], state_bits=bits, **h), torch.optim.AdamW([q], **h)
            for k in range(4):
                p.grad = normal(3000, 50 + k)
                q.grad = p.grad.double()
                opt.step()
                ref.step()
                if bits == 32 or k == 0:
                    off = (p.detach().double() - q.detach()).abs()  # an update is at most lr / sqrt(1 - b2) here
                    assert float(off.max()) < 1e-2 * 32 * 64 * E + 8 * E * float(p.detach().abs().max())
            assert bool(p.isfinite().all()) and int(opt.state[p]["step"]) == 4


def test_gradients_that_are_no_numbers(cuda):
    for bits in (32, 8):
        st = make([1024], bits)
        st["grads"][0][300] = float("nan")
        scn.adamw_step(step=steps(3), **st, **HYPER)
        bad = st["params"][0].isnan().nonzero().view(-1).tolist()
        assert bad == [300]
        m = st["exp_avgs"][0].float().isnan().nonzero().view(-1).tolist()
        assert m == ([300] if bits == 32 else list(range(256, 512)))


def test_rate_on_the_device_and_a_captured_step(cuda):
    for bits in (32, 8):
        st = make([5000, 77], bits)
        eager = copy_of(st)
        lr, step = torch.tensor([1e-3], device="cuda"), steps(0)
        h = {k: v for k, v in HYPER.items() if k != "lr"}
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            scn.adamw_step(step=step, lr=lr, **st, **h)
        assert int(step) == 0
        for rate in (1e-3, 5e-3, 0.0):
            lr.fill_(rate)
            graph.replay()
        other = steps(0)
        for rate in (1e-3, 5e-3, 0.0):
            scn.adamw_step(step=other, lr=rate, **eager, **h)
        assert int(step) == 3
        for k in st:
            assert all(torch.equal(a.float(), b.float()) for a, b in zip(st[k], eager[k])), (bits, k)


def test_two_lists_at_once_on_two_streams(cuda):
    sets = [make(SIZES, 8, seed=1000 * i) for i in range(2)]
    alone = [copy_of(s) for s in sets]
    counts = [steps(0), steps(10)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(5):
        for s, c, q in zip(sets, counts, streams):
            with torch.cuda.stream(q):
                scn.adamw_step(step=c, **s, **HYPER)
    torch.cuda.synchronize()
    for s, first in zip(alone, (0, 10)):
        step = steps(first)
        for _ in range(5):
            scn.adamw_step(step=step, **s, **HYPER)
    assert [int(c) for c in counts] == [5, 15]
    for s, o in zip(sets, alone):
        assert all(torch.equal(a.float(), b.float()) for k in s for a, b in zip(s[k], o[k]))


@pytest.mark.parametrize("bits", [32, 8])
def test_optimizer_against_torch(cuda, bits):
    torch.manual_seed(0)
    mine = [torch.nn.Parameter(normal(n, i)) for i, n in enumerate((300, 17, 5000))]
    theirs = [torch.nn.Parameter(p.detach().clone()) for p in mine]
    h = dict(lr=1e-2, betas=(0.9, 0.99), eps=1e-6, weight_decay=0.05)
    opt = scn.AdamW([{"params": mine[:2]}, {"params": mine[2:], "lr": 2e-2}], state_bits=bits, **h)
    ref = torch.optim.AdamW([{"params": theirs[:2]}, {"params": theirs[2:], "lr": 2e-2}], **h)
    for k in range(6):
        for j, (p, q) in enumerate(zip(mine, theirs)):
            p.grad = None if (k, j) == (2, 1) else normal(p.numel(), 100 + 10 * k + j)
            q.grad = None if p.grad is None else p.grad.clone()
        opt.step()
        ref.step()
        if k == 3:  # through a checkpoint
            saved = opt.state_dict()
            opt = scn.AdamW([{"params": mine[:2]}, {"params": mine[2:], "lr": 2e-2}], state_bits=bits, **h)
            opt.load_state_dict(saved)
            assert opt.state[mine[0]]["exp_avg"].dtype == (torch.float32 if bits == 32 else torch.float8_e4m3fn)
    assert [int(opt.state[p]["step"]) for p in mine] == [6, 5, 6]
    for p, q in zip(mine, theirs):
        # an update is at most lr (1 - b1) / sqrt(1 - b2) / ... = some 2 lr; in 8 bits each may be 2^-2 of itself off
        assert float((p - q).detach().abs().max()) < (6 * 2e-2 * 2 * (100 * E if bits == 32 else 0.5))


def test_no_tensors(cuda):
    """A list of nothing, or of tensors without values, is a step all the same."""
    step = steps(4)
    scn.adamw_step([], [], [], [], step)
    empty = [torch.zeros(0, device="cuda")] * 2
    scn.adamw_step(empty, empty, empty, empty, step)
    assert int(step) == 6


def test_a_checkpoint_in_a_file(cuda, tmp_path):
    """States go through a file with their types, and the run goes on as it would have."""
    runs = []
    for through_file in (False, True):
        p = torch.nn.Parameter(normal(3000, 1, torch.bfloat16))
        opt = scn.AdamW([p], lr=1e-2, state_bits=8, master_weights=True, seed=3)
        for k in range(4):
            p.grad = normal(3000, 10 + k, torch.bfloat16)
            opt.step()
            if through_file and k == 1:
                torch.save(opt.state_dict(), tmp_path / "state")
                opt = scn.AdamW([p], lr=1e-2, state_bits=8, master_weights=True, seed=3)
                opt.load_state_dict(torch.load(tmp_path / "state"))
        runs.append((p.detach(), opt.state[p]))
    assert torch.equal(runs[0][0], runs[1][0])
    for k, v in runs[0][1].items():
        assert v.dtype == runs[1][1][k].dtype and torch.equal(v.float(), runs[1][1][k].float()), k


def test_master_weights(cuda):
    """Updates below half a step of bfloat16 add up in the fp32 weights."""
    p = torch.nn.Parameter(torch.ones(512, device="cuda", dtype=torch.bfloat16))
    opt = scn.AdamW([p], lr=1e-4, weight_decay=0.0, master_weights=True)
    for _ in range(60):
        p.grad = torch.ones_like(p)
        opt.step()
    master = opt.state[p]["master"]
    # the update of a constant gradient is lr * (1 + small): 60 of them; eps / (sqrt(v) + eps) is 1e-8
    assert float((master - (1 - 60e-4)).abs().max()) < 60 * (1e-4 * 24 * E + 2 * E)
    assert torch.equal(p.detach(), master.to(torch.bfloat16)) and float(p.detach()[0]) < 1


def test_writes_are_seen_by_version(cuda):
    p = torch.nn.Parameter(normal(100, 1))
    p.grad = normal(100, 2)
    before = p._version
    scn.AdamW([p]).step()
    assert p._version > before
    y = (p * p).sum()
    p.grad = normal(100, 2)
    scn.AdamW([p]).step()
    with pytest.raises(RuntimeError, match="modified"):
        y.backward()


def test_more_than_2_31_values(cuda):
    n = 2 ** 31 + 1000
    st = {"params": [torch.zeros(n, device="cuda", dtype=torch.bfloat16)], "grads": [torch.zeros(n, device="cuda", dtype=torch.bfloat16)],
          "exp_avgs": [torch.zeros(n, device="cuda", dtype=torch.uint8).view(torch.float8_e4m3fn)],
          "exp_avg_sqs": [torch.zeros(n, device="cuda", dtype=torch.uint8).view(torch.float8_e4m3fn)],
          "exp_avg_scales": [torch.zeros(-(-n // 256), device="cuda")], "exp_avg_sq_scales": [torch.zeros(-(-n // 256), device="cuda")]}
    p, g = normal(1000, 1, torch.bfloat16), normal(1000, 2, torch.bfloat16)
    st["params"][0][-1000:], st["grads"][0][-1000:] = p, g
    zero = torch.zeros(1000, device="cuda")
    scn.adamw_step(step=steps(0), **st, **HYPER)
    want, _, _, _, update = formula(p, g, zero, zero, 1, **HYPER)
    off = (st["params"][0][-1000:].double() - want).abs()
    assert bool((off <= half(torch.bfloat16) * want.abs() * (1 + 1e-6) + 24 * E * update + 3 * E * want.abs()).all())
    assert bool((st["params"][0][:1000] == 0).all()) and bool((st["exp_avgs"][0][-1000:].float() != 0).any())


def test_refusals(cuda):
    def call(**k):
        st = make([64, 64], 32)
        st.update(step=steps(0))
        st.update(k)
        scn.adamw_step(**st)

    f = lambda n=64, t=torch.float32: torch.zeros(n, device="cuda").to(t)  # noqa: E731
    same = f()
    for k, said in ((dict(params=[same, same]), "twice"), (dict(grads=[f()]), "tensors"), (dict(grads=[f(), f(63)]), "shapes"), (dict(step=steps(0).int()), "step"),
                    (dict(step=torch.zeros(2, dtype=torch.int64, device="cuda")), "step"), (dict(exp_avgs=[f(t=torch.bfloat16)] * 2), "exp_avgs"),
                    (dict(exp_avg_scales=[f(1)] * 2), "both"), (dict(params=[f(), f(t=torch.float16)]), "params"), (dict(params=[f(128)[::2], f()]), "contiguous"),
                    (dict(copies=[f(), f()]), "copies"), (dict(lr=torch.zeros(2, device="cuda")), "lr"), (dict(lr=torch.zeros(1)), "CUDA"),
                    (dict(grads=[f(t=torch.float64)] * 2), "grads")):
        with pytest.raises(RuntimeError, match=said):
            call(**k)
    for k in (dict(betas=(1.0, 0.9)), dict(lr=-1.0), dict(eps=-1.0)):
        with pytest.raises(Exception, match="adamw_step"):
            call(**k)
