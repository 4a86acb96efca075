"""What the optimiser refuses, and its host side, without a GPU."""
import ctypes

import pytest
import torch

import sparseconvnet_b200 as scn


def test_cpu_tensors_are_refused():
    t = [torch.zeros(4)]
    with pytest.raises(RuntimeError, match="no CPU path"):
        scn.adamw_step(t, t, t, t, torch.zeros(1, dtype=torch.int64))
    p = torch.nn.Parameter(torch.zeros(4))
    p.grad = torch.zeros(4)
    with pytest.raises(RuntimeError, match="no CPU path"):
        scn.AdamW([p]).step()


@pytest.mark.parametrize("bad", [dict(lr=-1.0), dict(betas=(1.0, 0.9)), dict(betas=(0.9, -0.1)), dict(eps=-1e-8), dict(weight_decay=-1.0),
                                 dict(state_bits=16)])
def test_bad_settings(bad):
    with pytest.raises(ValueError):
        scn.AdamW([torch.nn.Parameter(torch.zeros(4))], **bad)


def test_nothing_to_do():
    p = torch.nn.Parameter(torch.ones(4))
    opt = scn.AdamW([p])
    assert opt.step(lambda: 3.0) == 3.0 and torch.equal(p, torch.ones(4)) and not opt.state[p]


def test_library_refuses_what_it_cannot_do():
    from sparseconvnet_b200._lib import lib
    ok = dict(t=None, n=0, p=0, g=0, bits=32, copy=-1, step=8, lr=1e-3, dev=None, b1=0.9, b2=0.999, eps=1e-8, wd=0.01, seed=0, st=None)
    call = lambda **k: lib.scn_adamw_step(*{**ok, **k}.values())  # noqa: E731
    for bad in (dict(p=3), dict(g=-1), dict(bits=16), dict(copy=0), dict(b1=1.0), dict(b2=-0.5), dict(eps=-1.0), dict(wd=-1.0), dict(lr=-1.0),
                dict(n=-1), dict(n=1), dict(step=None), dict(b1=float("nan"))):
        assert call(**bad) == 1, bad

    class Entry(ctypes.Structure):
        _fields_ = [(k, ctypes.c_void_p) for k in ("param", "grad", "m", "v", "ms", "vs", "copy")] + [("n", ctypes.c_int64)]

    full = dict(param=16, grad=16, m=16, v=16, ms=None, vs=None, copy=None, n=4)
    for bad, more in ((dict(param=None), {}), (dict(grad=None), {}), (dict(v=None), {}), (dict(n=-4), {}), ({}, dict(bits=8)), (dict(copy=16), {}),
                      ({}, dict(copy=1))):
        e = Entry(**{**full, **bad})
        assert call(t=ctypes.addressof(e), n=1, **more) == 1, (bad, more)
