"""The optimiser's step in a captured graph: it goes on as the eager one would, or is refused."""
import pytest
import torch

import sparseconvnet_b200 as scn

pytestmark = pytest.mark.gpu


def network(seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    ps = [torch.nn.Parameter(torch.randn(n, generator=g, device="cuda").to(t)) for n, t in ((700, torch.float32), (5, torch.float32), (300, torch.bfloat16))]
    for p in ps:
        p.grad = torch.randn(p.shape, generator=g, device="cuda").to(p.dtype)
    return ps


@pytest.mark.parametrize("bits", [32, 8])
def test_a_captured_step_goes_on(cuda, bits):
    eager, captured = network(1), network(1)
    one, two = (scn.AdamW(ps, lr=1e-2, state_bits=bits, master_weights=True, seed=7) for ps in (eager, captured))
    for _ in range(2):
        one.step()
        two.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        two.step()
    for _ in range(3):
        one.step()
        graph.replay()
    one.step()
    two.step()  # outside again
    for p, q in zip(eager, captured):
        assert torch.equal(p, q) and int(one.state[p]["step"]) == int(two.state[q]["step"]) == 6
        assert all(torch.equal(v.float(), two.state[q][k].float()) for k, v in one.state[p].items())


@pytest.mark.parametrize("bits", [32, 8])
def test_what_a_graph_cannot_hold_is_refused(cuda, bits):
    """A first step would set its moments to zero with every replay; a count that is split from another's would never go on."""
    ps = network(2)
    opt = scn.AdamW(ps, state_bits=bits)
    was = [p.detach().clone() for p in ps]
    with pytest.raises(RuntimeError, match="first step"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            opt.step()
    assert all(torch.equal(p, q) for p, q in zip(ps, was)) and not any(opt.state[p] for p in ps)
    opt.step()
    opt.step()
    grad, ps[1].grad = ps[1].grad, None
    with pytest.raises(RuntimeError, match="together"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            opt.step()
    opt.step()
    ps[1].grad = grad
    opt.step()
    assert [int(opt.state[p]["step"]) for p in ps] == [4, 3, 4]
