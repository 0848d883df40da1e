"""Argument checks of the microscaled and sampling entry points, on the CPU: refused calls
return their TbError before any device work, empty ones TB_OK."""
import ctypes as C

import numpy as np
import pytest
import torch

import mx_ref as R
import tb_b200 as T

OK, ARG, SHAPE, DTYPE = 0, 8, 9, 10
FAKE = 0x10000  # an address that is checked but never read
E4M3, E2M1 = T.MX_FORMATS["e4m3"], T.MX_FORMATS["e2m1"]


def mx(**kw):
    f = dict(format=E4M3, rows=4, cols=256, codes=FAKE, scales=FAKE)
    f.update(kw)
    return T.Mx(**f)


BAD_TENSORS = [
    (dict(format=0), DTYPE), (dict(format=T.INT8), DTYPE), (dict(rows=-1), SHAPE),
    (dict(rows=2 ** 31 - 1), SHAPE), (dict(cols=0), SHAPE), (dict(cols=-5), SHAPE),
    (dict(cols=2 ** 24 + 1), SHAPE), (dict(codes=None), ARG), (dict(scales=None), ARG),
    (dict(codes=FAKE + 16), ARG), (dict(scales=FAKE + 8), ARG)]


@pytest.mark.parametrize("change,want", BAD_TENSORS)
def test_bad_tensors(change, want):
    L, t, good = T.lib(), mx(**change), mx()
    assert L.tb_b200_mx_quantize(T.F32, FAKE, 256, C.byref(t), None) == want
    assert L.tb_b200_mx_dequantize(C.byref(t), T.F32, FAKE, 256, None) == want
    assert L.tb_b200_residual_rms_norm_mx(T.F32, FAKE, None, None, None, C.byref(t), 1e-5,
                                          None) == want
    assert L.tb_b200_swiglu_mx(T.F32, FAKE, 256, FAKE, 256, C.byref(t), None) == want
    assert L.tb_b200_mx_linear(C.byref(t), C.byref(good), None, T.F32, FAKE, 256, None) == want
    assert L.tb_b200_mx_linear(C.byref(good), C.byref(t), None, T.F32, FAKE, 2 ** 31,
                               None) == want


@pytest.mark.parametrize("dtype", [T.F16, T.I32, T.INT8, -1])
def test_bad_dtypes(dtype):
    L, t = T.lib(), mx()
    assert L.tb_b200_mx_quantize(dtype, FAKE, 256, C.byref(t), None) == DTYPE
    assert L.tb_b200_mx_dequantize(C.byref(t), dtype, FAKE, 256, None) == DTYPE
    assert L.tb_b200_residual_rms_norm_mx(dtype, FAKE, None, None, None, C.byref(t), 1e-5,
                                          None) == DTYPE
    assert L.tb_b200_swiglu_mx(dtype, FAKE, 256, FAKE, 256, C.byref(t), None) == DTYPE
    assert L.tb_b200_mx_linear(C.byref(t), C.byref(t), None, dtype, FAKE, 256, None) == DTYPE


def test_bad_pointers_and_strides():
    L, t = T.lib(), mx()
    assert L.tb_b200_mx_quantize(T.F32, None, 256, C.byref(t), None) == ARG
    assert L.tb_b200_mx_quantize(T.F32, FAKE, 255, C.byref(t), None) == SHAPE
    assert L.tb_b200_mx_quantize(T.F32, FAKE, 256, None, None) == ARG
    assert L.tb_b200_mx_dequantize(C.byref(t), T.F32, None, 256, None) == ARG
    assert L.tb_b200_mx_dequantize(C.byref(t), T.F32, FAKE, 255, None) == SHAPE
    assert L.tb_b200_mx_dequantize(None, T.F32, FAKE, 256, None) == ARG
    assert L.tb_b200_residual_rms_norm_mx(T.F32, None, FAKE, None, None, C.byref(t), 1e-5,
                                          None) == ARG
    assert L.tb_b200_residual_rms_norm_mx(T.F32, FAKE, FAKE, None, None, None, 1e-5, None) == ARG
    assert L.tb_b200_swiglu_mx(T.F32, None, 256, FAKE, 256, C.byref(t), None) == ARG
    assert L.tb_b200_swiglu_mx(T.F32, FAKE, 256, None, 256, C.byref(t), None) == ARG
    assert L.tb_b200_swiglu_mx(T.F32, FAKE, 255, FAKE, 256, C.byref(t), None) == SHAPE
    assert L.tb_b200_swiglu_mx(T.F32, FAKE, 256, FAKE, 255, C.byref(t), None) == SHAPE
    w = mx(rows=9)
    assert L.tb_b200_mx_linear(C.byref(t), C.byref(w), None, T.F32, None, 9, None) == ARG
    assert L.tb_b200_mx_linear(C.byref(t), C.byref(w), None, T.F32, FAKE, 8, None) == SHAPE
    assert L.tb_b200_mx_linear(C.byref(t), C.byref(mx(cols=128)), None, T.F32, FAKE, 9,
                               None) == SHAPE
    assert L.tb_b200_mx_linear(None, C.byref(w), None, T.F32, FAKE, 9, None) == ARG
    assert L.tb_b200_mx_linear(C.byref(t), None, None, T.F32, FAKE, 9, None) == ARG


def test_empty_calls_do_nothing():
    L, t = T.lib(), mx(rows=0, codes=None, scales=None)
    assert L.tb_b200_mx_quantize(T.F32, None, 0, C.byref(t), None) == OK
    assert L.tb_b200_mx_dequantize(C.byref(t), T.F32, None, 0, None) == OK
    assert L.tb_b200_residual_rms_norm_mx(T.F32, None, None, None, None, C.byref(t), 1e-5,
                                          None) == OK
    assert L.tb_b200_swiglu_mx(T.F32, None, 0, None, 0, C.byref(t), None) == OK
    assert L.tb_b200_mx_linear(C.byref(t), C.byref(mx()), None, T.F32, None, 4, None) == OK
    assert L.tb_b200_mx_linear(C.byref(mx()), C.byref(t), None, T.F32, None, 0, None) == OK


@pytest.mark.parametrize("fmt,each", [("e4m3", 1), ("e2m1", 2)])
@pytest.mark.parametrize("rows,cols", [(0, 5), (1, 1), (128, 128), (129, 129), (1000, 11008)])
def test_bytes(rows, cols, fmt, each):
    codes, scales = C.c_size_t(), C.c_size_t()
    assert T.lib().tb_b200_mx_bytes(T.MX_FORMATS[fmt], rows, cols, C.byref(codes),
                                    C.byref(scales)) == OK
    assert codes.value == rows * R.up(cols, 128) // each
    assert scales.value == R.up(rows, 128) * R.up(cols, 128) // 32
    assert T.lib().tb_b200_mx_bytes(T.MX_FORMATS[fmt], rows, cols, None, C.byref(scales)) == ARG
    assert T.lib().tb_b200_mx_bytes(0, rows, cols, C.byref(codes), C.byref(scales)) == DTYPE


def test_scale_places_fill_their_tiles():
    for rows, cols in [(1, 32), (128, 128), (300, 1000)]:
        p = R.scale_places(rows, cols)
        assert len(np.unique(p)) == p.size
        assert p.max() < R.up(rows, 128) * R.up(cols, 128) // 32
    assert np.array_equal(np.sort(R.scale_places(256, 256).ravel()), np.arange(2048))


def sample(**kw):
    f = dict(dtype=T.F32, rows=2, vocab=100, logits=FAKE, stride=100, uniforms=FAKE, out=FAKE)
    f.update(kw)
    return T.Sample(**f)


@pytest.mark.parametrize("change,want", [
    (dict(dtype=T.F16), DTYPE), (dict(rows=-1), SHAPE), (dict(rows=2 ** 31), SHAPE),
    (dict(vocab=0), SHAPE), (dict(vocab=2 ** 22 + 1, stride=2 ** 23), SHAPE),
    (dict(stride=99), SHAPE), (dict(logits=None), ARG), (dict(uniforms=None), ARG),
    (dict(out=None), ARG), (dict(rows=0, logits=None, uniforms=None, out=None), OK)])
def test_sample_refusals(change, want):
    t = sample(**change)
    assert T.lib().tb_b200_sample(C.byref(t), None) == want
    assert T.lib().tb_b200_sample(None, None) == ARG


def test_python_refuses_tensors_of_the_host():
    x = torch.zeros(2, 64)
    for call in (lambda: T.mx_quantize(x), lambda: T.swiglu_mx(x, x),
                 lambda: T.residual_rms_norm_mx(x, x, None, 1e-5),
                 lambda: T.MxTensor(torch.zeros(2, 128, dtype=torch.uint8),
                                    torch.zeros(512, dtype=torch.uint8), 64, "e4m3"),
                 lambda: T.sample(x, torch.zeros(2, dtype=torch.float64))):
        with pytest.raises(ValueError):
            call()


def test_definition_of_sampling():
    """The definition that the GPU is held to, on cases worked out by hand."""
    x = np.log([0.1, 0.4, 0.2, 0.3])
    assert R.draw(x, 0.0) == 0 and R.draw(x, 0.0999) == 0 and R.draw(x, 0.1001) == 1
    assert R.draw(x, 0.9999) == 3
    assert R.draw(x, 0.0, top_k=2) == 1 and R.draw(x, 0.58, top_k=2) == 3
    assert R.draw(x, 0.56, top_k=2) == 1
    assert R.draw(x, 0.0, top_p=0.39) == 1 and R.draw(x, 0.99, top_p=0.41) == 3
    assert R.draw(x, 0.99, top_p=0.69) == 3 and R.draw(x, 0.5, top_p=0.71) == 2
    assert R.draw(x, 0.0, min_p=0.3) == 1 and R.draw(x, 0.99, min_p=0.8) == 1
    assert R.draw(x, 0.7, temperature=0.0) == 1
    assert R.draw([2.0, 2.0, 1.0], 0.9, top_k=1) == 0
    assert R.draw([-np.inf, np.nan], 0.5) == 0
