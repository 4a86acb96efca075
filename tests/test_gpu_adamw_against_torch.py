"""The optimizer with moments in 8 bits against torch's in float32, over several steps with rates by group, absent gradients and a
reload: how far parameters have moved, not how far they may be."""
import pytest
import torch

import sparseconvnet_b200 as scn

pytestmark = pytest.mark.gpu


def distances(rate=1.0, forget=False):
    """Relative 2-norm of the difference from torch's displacement, per parameter group.  `rate`: what the rates are multiplied by;
    `forget`: the moments are lost at the reload."""
    g = torch.Generator(device="cuda").manual_seed(0)
    first = [torch.randn(n, generator=g, device="cuda") for n in (3000, 170, 50000)]
    mine, theirs = ([torch.nn.Parameter(p.clone()) for p in first] for _ in range(2))
    h = dict(betas=(0.9, 0.99), eps=1e-6, weight_decay=0.05)
    groups = lambda ps, r: [{"params": ps[:2], "lr": 1e-2 * r}, {"params": ps[2:], "lr": 2e-2 * r}]  # noqa: E731
    opt, ref = scn.AdamW(groups(mine, rate), state_bits=8, **h), torch.optim.AdamW(groups(theirs, 1.0), **h)
    for k in range(6):
        for j, (p, q) in enumerate(zip(mine, theirs)):
            grad = torch.randn(p.shape, generator=g, device="cuda")
            p.grad, q.grad = (None, None) if (k, j) == (2, 1) else (grad, grad.clone())
        opt.step()
        ref.step()
        if k == 3:
            saved = opt.state_dict()
            opt = scn.AdamW(groups(mine, rate), state_bits=8, **h)
            if not forget:
                opt.load_state_dict(saved)
    norm = lambda ts: torch.cat(ts).double().norm()  # noqa: E731
    return [float(norm([p.detach() - q.detach() for p, q in zip(mine[s], theirs[s])]) / norm([q.detach() - f for q, f in zip(theirs[s], first[s])]))
            for s in (slice(0, 2), slice(2, 3))]


def test_displacement_in_8_bits(cuda):
    # A step is m / sqrt(v), both from moments that have been rounded to a neighbour in e4m3, 2^-3 apart at most: by chance in proportion to the
    # distance, so at most 2^-4 of the value in standard deviation, in each moment at each step.  m of one step keeps 0.9, 0.81 .. of the
    # roundings before it: less than 2^-4 sqrt(0.81 / (1 - 0.81)) = 0.13 in the long run, sqrt(v) less than half of that times 0.99's share in the
    # same direction.  A value's displacement is the sum of six such updates, whose roundings are partly independent; values near zero in their
    # blocks are off by more than their own size, but move little.  10% of the displacement's 2-norm, and nothing half as good passes.
    right = distances()
    assert max(right) < 0.10, right
    assert min(distances(rate=0.5)) > 0.4 and min(distances(forget=True)) > 0.15
