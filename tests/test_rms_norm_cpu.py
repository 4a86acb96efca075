"""What the row norms refuse, in this process and without a GPU."""
import pytest
import torch

import sparseconvnet_b200 as scn


def test_cpu_tensors_are_refused():
    for call in (scn.rms_norm, scn.rms_norm_quantized):
        with pytest.raises(RuntimeError, match="no CPU path"):
            call(torch.ones(2, 8), torch.ones(8))
    with pytest.raises(RuntimeError, match="must be a tensor"):
        scn.rms_norm([1.0, 2.0])


def test_result_type():
    with pytest.raises(ValueError, match="out_dtype"):
        scn.rms_norm(torch.ones(2, 8), out_dtype=torch.float64)


def test_modules():
    m = scn.RMSNormalization(6)
    assert list(m.state_dict()) == ["weight"] and torch.equal(m.weight, torch.ones(6)) and m.eps == 1e-6
    assert not scn.RMSNormalization(6, affine=False).state_dict()
    assert repr(scn.AddRMSNormalization(6, 1e-5)) == "AddRMSNormalization(6,eps=1e-05,affine=True)"
    assert m.input_spatial_size(torch.LongTensor([5])).tolist() == [5]
    with pytest.raises(AssertionError):
        m(scn.SparseConvNetTensor(torch.ones(2, 4), None, None))


def test_library_refuses_what_it_cannot_do():
    from sparseconvnet_b200._lib import lib
    ok = dict(x=16, xs=8, r=None, rs=8, type=0, w=None, n=4, c=8, eps=1e-6, s=None, out=32, ot=0, scale=None, inv=None, st=None)
    call = lambda **k: lib.scn_rms_norm_forward(*{**ok, **k}.values())  # noqa: E731  (every refusal comes before a launch)
    assert call(n=0) == 0
    for bad in (dict(type=3), dict(type=7), dict(ot=4), dict(n=-1), dict(c=0), dict(eps=-1.0), dict(eps=float("nan")), dict(x=None),
                dict(out=None), dict(r=48), dict(s=48), dict(ot=3), dict(scale=64)):
        assert call(**bad) == 1, bad
        assert lib.scn_last_error()
    assert lib.scn_rms_norm_backward(16, 8, 3, None, 16, 16, 0, None, 4, 8, 16, None, None) == 1
    assert lib.scn_rms_norm_backward(16, 8, 0, None, None, 16, 0, None, 4, 8, 16, None, None) == 1
