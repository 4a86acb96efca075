"""What the grouped products refuse, without a GPU."""
import pytest
import torch

import sparseconvnet_b200 as scn


def test_cpu_tensors_are_refused():
    x, w, o = torch.ones(4, 8), torch.ones(2, 8, 8), torch.tensor([0, 2, 4])
    with pytest.raises(RuntimeError, match="no CPU path"):
        scn.grouped_product(x, w, o)
    q, ws = scn.quantize_group_weights(w)
    assert q.dtype == torch.float8_e4m3fn and q.shape == (2, 8, 8) and ws.shape == (2, 8) and bool((q.float() == 448).all())
    with pytest.raises(RuntimeError, match="no CPU path"):
        scn.grouped_product_quantized(x.to(torch.float8_e4m3fn), torch.ones(4), q, ws, o)
    for bad in (torch.float64, None):
        with pytest.raises(ValueError, match="out_dtype"):
            scn.grouped_product_quantized(q[0], ws[0], q, ws, o, out_dtype=bad)


def test_weights_in_eight_bits():
    w = torch.randn(3, 17, 5)
    w[1, :, 2] = 0
    q, scale = scn.quantize_group_weights(w)
    back = (q.double() * scale.double()[:, :, None]).transpose(1, 2)
    # half a step of e4m3: 2^-4 of a value, 2^-10 of the scale below 2^-6
    assert bool(((back - w.double()).abs() <= w.double().abs() * 2.0 ** -4 * (1 + 1e-6) + 2.0 ** -10 * scale.double()[:, None, :]).all())
    assert bool((back[1, :, 2] == 0).all())


def test_module():
    m = scn.GroupedNetworkInNetwork(3, 4, 5, True)
    assert {k: tuple(v.shape) for k, v in m.state_dict().items()} == {"weight": (3, 4, 5), "bias": (3, 5)}
    assert repr(m) == "GroupedNetworkInNetwork3x4->5" and list(scn.GroupedNetworkInNetwork(3, 4, 5, False).state_dict()) == ["weight"]


def test_library_refuses_what_it_cannot_do():
    from sparseconvnet_b200._lib import lib
    ok = dict(x=16, xs=8, type=0, w=16, b=None, bt=0, o=16, o64=1, n=4, g=2, i=8, k=8, p=0, out=16, ot=0, st=None)
    call = lambda **k: lib.scn_grouped_product_forward(*{**ok, **k}.values())  # noqa: E731  (every refusal comes before a launch)
    assert call(n=0, o=None) == 0
    for bad in (dict(type=3), dict(ot=3), dict(b=16, bt=9), dict(p=4), dict(n=-1), dict(i=0), dict(k=0), dict(o=None), dict(x=None), dict(w=None), dict(out=None)):
        assert call(**bad) == 1, bad
    for bad in (dict(g=0), dict(g=1025), dict(n=1 << 31), dict(i=(1 << 20) + 1)):
        assert call(**bad) == 7, bad
    back = dict(x=16, xs=8, type=0, w=16, d=16, ds=8, o=16, o64=1, n=4, g=2, i=8, k=8, p=0, dx=16, dw=None, db=None, st=None)
    call = lambda **k: lib.scn_grouped_product_backward(*{**back, **k}.values())  # noqa: E731
    for bad in (dict(type=3), dict(d=None), dict(w=None), dict(x=None, dw=16), dict(p=-1)):
        assert call(**bad) == 1, bad
    quantized = dict(q=16, qs=16, s=16, w=16, ws=16, b=None, bt=0, o=16, o64=1, n=4, g=2, i=16, k=8, out=16, ot=1, st=None)
    call = lambda **k: lib.scn_grouped_product_quantized(*{**quantized, **k}.values())  # noqa: E731
    for bad in (dict(ot=3), dict(s=None), dict(ws=None), dict(q=None)):
        assert call(**bad) == 1, bad
