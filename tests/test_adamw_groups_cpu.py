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
