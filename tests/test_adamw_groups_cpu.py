"""The optimiser around the step: what it refuses and how it keeps count, without a GPU."""
import pytest
import torch

import sparseconvnet_b200 as scn


def parameters(n):
    return [torch.nn.Parameter(torch.ones(3)) for _ in range(n)]


@pytest.mark.parametrize("bad", [dict(state_bits=16), dict(state_bits=7), dict(lr=-1.0), dict(betas=(1.0, 0.9)), dict(betas=(0.9, -0.1)), dict(eps=-1e-8),
                                 dict(weight_decay=-0.1), dict(lr=float("nan"))])
def test_a_groups_own_values_are_checked(bad):
    p, q = parameters(2)
    with pytest.raises(ValueError, match=next(iter(bad))):
        scn.AdamW([{"params": [p]}, dict(bad, params=[q])])
    opt = scn.AdamW([p])
    with pytest.raises(ValueError, match=next(iter(bad))):
        opt.add_param_group(dict(bad, params=[q]))
    assert len(opt.param_groups) == 1  # nothing of the refused group stays
    opt.add_param_group(dict(params=[q], state_bits=8, lr=torch.tensor([1e-3])))
    assert opt.param_groups[1]["state_bits"] == 8 and opt.param_groups[1]["betas"] == (0.9, 0.999)


def with_states(opt):
    for group in opt.param_groups:
        step = torch.tensor([4])
        for p in group["params"]:
            opt.state[p] = dict(opt._start(p, group), step=step)
    return opt


def test_another_optimizers_checkpoint_is_refused():
    p, q = parameters(2)
    theirs = torch.optim.AdamW([p], lr=1e-2)
    p.grad = torch.ones(3)
    theirs.step()
    opt = with_states(scn.AdamW([q], lr=5e-3, state_bits=8))
    before = opt.state_dict()
    for bad in (theirs.state_dict(), torch.optim.SGD([p], lr=1.0).state_dict()):
        with pytest.raises(ValueError, match="another optimizer"):
            opt.load_state_dict(bad)
    after = opt.state_dict()
    assert after["param_groups"] == before["param_groups"] and all(torch.equal(v.float(), after["state"][0][k].float()) for k, v in before["state"][0].items())


@pytest.mark.parametrize("bits", [8, 32])
def test_a_checkpoint_that_does_not_fit_is_refused(bits):
    make = lambda n, t: torch.nn.Parameter(torch.ones(n, dtype=t))  # noqa: E731
    opt = with_states(scn.AdamW([make(300, torch.bfloat16)], state_bits=bits, master_weights=True))
    fresh = lambda n=300, t=torch.bfloat16: scn.AdamW([make(n, t)], state_bits=bits)  # noqa: E731
    good = fresh()
    good.load_state_dict(opt.state_dict())
    (state,) = good.state.values()
    assert {k: v.dtype for k, v in state.items()} == {k: v.dtype for k, v in opt.state_dict()["state"][0].items()} and int(state["step"]) == 4
    for other in (fresh(299), fresh(t=torch.float32)):  # other sizes; no master copy wanted
        with pytest.raises(ValueError, match="does not fit"):
            other.load_state_dict(opt.state_dict())
        assert not other.state
    for k, v in dict(step=torch.tensor(4.0), exp_avg=torch.ones(300, dtype=torch.float64), exp_avg_sq=None, master=torch.ones(300, dtype=torch.bfloat16)).items():
        saved = opt.state_dict()
        saved["state"] = {0: {**saved["state"][0], k: v}}
        with pytest.raises(ValueError, match="does not fit"):
            fresh().load_state_dict(saved)
    saved = opt.state_dict()
    saved["param_groups"] = [dict(saved["param_groups"][0], state_bits=40 - bits)]
    with pytest.raises(ValueError, match="does not fit"):
        fresh().load_state_dict(saved)
    with pytest.raises(ValueError, match="parameter group"):
        scn.AdamW(parameters(2)).load_state_dict(opt.state_dict())
    empty = scn.AdamW([make(300, torch.bfloat16)])
    empty.load_state_dict(fresh().state_dict())  # one that has not stepped yet
    assert empty.param_groups[0]["state_bits"] == bits


@pytest.fixture
def steps_taken(monkeypatch):
    """The step on the device, replaced by what it does to the count; the lists that were stepped"""
    taken = []

    def step(params, grads, exp_avgs, exp_avg_sqs, step, *args):
        step.add_(1)
        taken.append((len(params), int(step)))
    monkeypatch.setattr(scn.optim, "adamw_step", step)
    return taken


def test_parameters_of_one_count_step_together_again(steps_taken):
    """64 parameters, each without a gradient one time in ten: as many launches as there are different counts."""
    random = torch.Generator().manual_seed(0)
    ps = parameters(64)
    opt = scn.AdamW(ps)
    counts = [0] * 64
    for k in range(60):
        steps_taken.clear()
        now = [bool(torch.rand(1, generator=random) >= 0.1) for _ in ps]
        for i, p in enumerate(ps):
            p.grad = torch.ones(3) if now[i] else None
        opt.step()
        assert len(steps_taken) == len({c for c, n in zip(counts, now) if n})
        counts = [c + n for c, n in zip(counts, now)]
        assert sum(n for n, _ in steps_taken) == sum(now)
        assert [int(opt.state[p]["step"]) if opt.state[p] else 0 for p in ps] == counts
        if k == 30:  # through a checkpoint
            saved = opt.state_dict()
            opt = scn.AdamW(ps)
            opt.load_state_dict(saved)
    assert len(opt._known) <= 3 * len(ps)


def test_types_and_groups_keep_counts_of_their_own(steps_taken):
    half = [torch.nn.Parameter(torch.ones(3, dtype=torch.bfloat16)) for _ in range(4)]
    full = parameters(4)
    opt = scn.AdamW([{"params": half + full}, {"params": parameters(2)}])
    every = [p for g in opt.param_groups for p in g["params"]]
    for k in range(6):
        steps_taken.clear()
        for p in every:
            p.grad = torch.ones_like(p)
        if k == 2:
            half[0].grad = full[0].grad = None
        opt.step()
        assert sorted(n for n, _ in steps_taken) == ([2, 4, 4] if k < 2 else [2, 3, 3] if k == 2 else [1, 1, 2, 3, 3])
    assert [int(opt.state[p]["step"]) for p in every] == [5, 6, 6, 6, 5, 6, 6, 6, 6, 6]
    half[0].grad = full[0].grad = None
    for p in every:
        if p is not half[0] and p is not full[0]:
            p.grad = None
    half[0].grad, full[0].grad = torch.ones_like(half[0]), torch.ones_like(full[0])
    opt.step()  # these two catch up
    for p in every:
        p.grad = torch.ones_like(p)
    steps_taken.clear()
    opt.step()
    assert sorted(n for n, _ in steps_taken) == [2, 4, 4] and [int(opt.state[p]["step"]) for p in every] == [7] * 10


def test_a_count_that_someone_else_has_changed(steps_taken):
    """What the host believes of a counter holds only as long as nobody else has written to it."""
    a, b = parameters(2)
    opt = scn.AdamW([a, b])
    for p, n in ((a, 2), (b, 1)):
        for q in (a, b):
            q.grad = torch.ones(3) if q is p else None
        for _ in range(n):
            opt.step()
    opt.state[a]["step"].fill_(1)  # both 1 now, but for all the host knows 2 and 1
    a.grad = b.grad = torch.ones(3)
    opt.step()
    assert int(opt.state[a]["step"]) == int(opt.state[b]["step"]) == 2
    opt.state[b]["step"].fill_(9)
    opt.step()
    assert int(opt.state[a]["step"]) == 3 and int(opt.state[b]["step"]) == 10


def test_a_copy_of_an_optimizer_counts_on(steps_taken):
    import copy
    import pickle
    ps = parameters(3)
    opt = scn.AdamW(ps)
    for p in ps:
        p.grad = torch.ones(3)
    opt.step()
    for other in (copy.deepcopy(opt), pickle.loads(pickle.dumps(opt))):
        (group,) = other.param_groups
        for p in group["params"]:
            p.grad = torch.ones(3)
        steps_taken.clear()
        other.step()
        assert steps_taken == [(3, 2)] and [int(opt.state[p]["step"]) for p in ps] == [1, 1, 1]


def test_parameters_without_a_gradient_have_no_state(steps_taken):
    a, b = parameters(2)
    opt = scn.AdamW([a, b])
    a.grad = torch.ones(3)
    opt.step()
    opt.step()
    saved = opt.state_dict()
    assert list(saved["state"]) == [0]
    saved["state"][1] = {}  # as torch writes it for a parameter that was only looked at
    other = scn.AdamW([a, b])
    other.load_state_dict(saved)
    b.grad = torch.ones(3)
    other.step()
    assert int(other.state[a]["step"]) == 3 and int(other.state[b]["step"]) == 1
