"""`format` beside `out`, in the calls that end in a microscaled format."""
from types import SimpleNamespace

import pytest
import torch

import tb_b200 as T


def given(fmt, rows=3, cols=200):
    return SimpleNamespace(rows=rows, cols=cols, format=fmt, device=0, c=object())


@pytest.mark.parametrize("fmt", ["e4m3", "e2m1"])
def test_out_has_its_own_format(fmt):
    out, other = given(fmt), {"e4m3": "e2m1", "e2m1": "e4m3"}[fmt]
    assert T._mx_out(None, 0, out, None, 3, 200, None) is out
    assert T._mx_out(None, 0, out, None, 3, 200, fmt) is out
    for wrong in (other, "e5m2"):
        with pytest.raises((TypeError, ValueError)):
            T._mx_out(None, 0, out, None, 3, 200, wrong)
    with pytest.raises(ValueError):
        T._mx_out(None, 0, out, None, 3, 201, fmt)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt,other", [("e4m3", "e2m1"), ("e2m1", "e4m3")])
def test_calls_refuse_another_format_than_outs(fmt, other, cuda):
    x = torch.randn(3, 200, device="cuda")
    out = T.MxTensor.empty(3, 200, fmt)
    out.codes.fill_(5)
    for call in (lambda **kw: T.mx_quantize(x, **kw), lambda **kw: T.swiglu_mx(x, x, **kw),
                 lambda **kw: T.residual_rms_norm_mx(x, x, None, 1e-5, **kw)):
        with pytest.raises(TypeError):
            call(format=other, out=out)
    assert (out.codes == 5).all()
    want = T.mx_quantize(x, fmt)
    for kw in (dict(), dict(format=fmt)):
        assert T.mx_quantize(x, out=out, **kw) is out
        assert torch.equal(out.codes, want.codes) and torch.equal(out.scales, want.scales)
    assert T.mx_quantize(x).format == "e4m3" and T.swiglu_mx(x, x).format == "e4m3"
    assert T.residual_rms_norm_mx(x, None, None, 1e-5)[1].format == "e4m3"
