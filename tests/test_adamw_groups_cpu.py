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
