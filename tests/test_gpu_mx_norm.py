"""residual_rms_norm_mx on the GPU to the accuracy that it is written for.

h is the f32 sum of x and the residual.  Its squares are exact in double (24 bits times 24), their
sum and the factor 1 / sqrt((eps + sum) / cols) are off by less than 2^-45, the factor's two f32
parts hold it to 2^-48, and h times both times the weight carries what each product's rounding
leaves out: so a row's f32 value is off by its one rounding, finfo(float32).eps / 2 = 2^-24, and
less than 2^-40 more, or by half of f32's least number.  A code is then the nearest one of some
value within that of the exact one, and rounding is monotone."""
import numpy as np
import pytest
import torch

import mx_ref as R
import tb_b200 as T
from test_gpu_mx import DTYPES, FORMATS, f64, held, normal

pytestmark = pytest.mark.gpu

ONCE = 2.0 ** -24 * (1 + 2.0 ** -10)


def check_rounded(t, y, rel=ONCE):
    """t holds rows y (float64), known to rel |y| and half of f32's least number."""
    got, scales = held(t)
    rows, cols = y.shape
    least, most = (np.maximum(np.abs(y) * (1 + s * rel) + s * 2.0 ** -150, 0) for s in (-1, 1))

    def exponents(a):
        full = np.zeros((rows, R.up(cols, 32)))
        full[:, :cols] = a
        return R.scale_exponents(full.reshape(rows, -1, 32).max(-1), t.format) + 127
    assert ((exponents(least) <= scales) & (scales <= exponents(most))).all()
    s = np.repeat(np.ldexp(1.0, scales.astype(np.int64) - 127), 32, 1)[:, :cols]
    a = np.abs(got) / s
    off = (a < R.nearest(least / s, t.format)) | (a > R.nearest(most / s, t.format))
    assert not off.any(), (int(off.sum()), np.argwhere(off)[:5].tolist())
    assert (got * np.sign(y) >= 0).all()


def norm_of(h, w, eps):
    """The norm of rows h, scaled by a power of two so that squares stay within float64."""
    by = 2.0 ** -np.floor(np.log2(np.abs(h).max(-1, keepdims=True)))
    s = h * by
    y = s / np.sqrt((eps * by * by + (s * s).sum(-1, keepdims=True)) / h.shape[1])
    return y if w is None else y * w


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("cols", [1, 40, 1000, 4100, 70000])
@pytest.mark.parametrize("dtype,size", [(d, s) for d in DTYPES for s in
                                        (1e25, 3e37, 1e15, 1e-15, 1e-25, 1e-39)] + [("f32", 1e-43)])
def test_rows_of_all_sizes(dtype, size, cols, fmt):
    """Rows whose squares, or whose factor, are no numbers of f32."""
    x = (normal(1, 3, cols).abs() + 0.5) * torch.sign(normal(2, 3, cols))
    x = (x * 0.5 * size).to(DTYPES[dtype])
    assert (x != 0).all()
    w = 1 + normal(3, cols, dtype=dtype, std=0.1)
    _, y = T.residual_rms_norm_mx(x, None, w, 0.0, format=fmt)
    check_rounded(y, norm_of(f64(x), f64(w), 0.0))
    res = x.flip(1).clone()
    h = x.float() + res.float()
    h_out, y = T.residual_rms_norm_mx(x, res, w, 0.0, format=fmt)
    assert torch.equal(h_out, h.to(x.dtype))
    keep = (h != 0).any(1).cpu().numpy()  # (a row of zeros with no eps is 0 / 0)
    if keep.all():
        check_rounded(y, norm_of(f64(h), f64(w), 0.0))


@pytest.mark.parametrize("fmt", FORMATS)
def test_row_with_elements_of_all_sizes(fmt):
    x = normal(4, 6, 640) * torch.exp2(torch.linspace(-120, 100, 640, device="cuda"))
    x[3:] = x[3:].flip(1)
    check_rounded(T.residual_rms_norm_mx(x, None, None, 1e-5, format=fmt)[1],
                  norm_of(f64(x), None, 1e-5))


def next_to_borders(h, fmt, eps, seed):
    """f32 weights that bring a row's values within three units of f32 of ties between codes."""
    mids = R.CODES[fmt][:127 if fmt == "e4m3" else 8]
    mids = (mids[1:] + mids[:-1])[1:] / 2
    r, cols = np.random.default_rng(seed), h.shape[1]
    goal = r.choice(mids, cols)
    # which holds the block's scale at 2^0
    goal[::32] = r.choice(mids[mids > 0.55 * R.LARGEST[fmt]], len(goal[::32]))
    w = (goal / norm_of(h, None, eps)[0]).astype(np.float32)
    return (w.view(np.int32) + r.integers(-3, 4, cols).astype(np.int32)).view(np.float32)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("cols,calls", [(1, 60), (2, 40), (7, 40), (32, 40), (200, 20), (4096, 4),
                                        (70000, 2)])
def test_values_next_to_rounding_borders(cols, calls, fmt):
    """A value rounded twice, or a factor that is off by its own rounding, comes out on the other
    side of some."""
    for seed in range(calls):
        x = normal(seed + 10, 1, cols)
        h = f64(x)
        w = next_to_borders(h, fmt, 1e-5, 1000 * seed + cols)
        y = T.residual_rms_norm_mx(x, None, torch.from_numpy(w).cuda(), 1e-5, format=fmt)[1]
        check_rounded(y, norm_of(h, w.astype(np.float64), 1e-5))


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", [(130, 1024), (1000, 24), (77, 4100), (9, 16384), (3, 70000)])
def test_rows_are_rounded_once(rows, cols, dtype, fmt):
    x, res = normal(5, rows, cols, dtype=dtype), normal(6, rows, cols, dtype=dtype, std=2.0)
    w = 1 + normal(7, cols, dtype=dtype, std=0.1)
    _, y = T.residual_rms_norm_mx(x, res, w, 1e-5, format=fmt)
    check_rounded(y, norm_of(f64(x.float() + res.float()), f64(w), 1e-5))


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", DTYPES)
def test_swiglu_rows(dtype, fmt):
    """expf (2 units, 2^-22), the sum, the quotient and the product (2^-24 each): 7 * 2^-24, and
    less than 2^-24 of what these give together."""
    g, u = normal(8, 500, 4096, dtype=dtype, std=3.0), normal(9, 500, 4096, dtype=dtype)
    a, b = f64(g), f64(u)
    check_rounded(T.swiglu_mx(g, u, fmt), a / (1 + np.exp(-a)) * b, 8 * 2.0 ** -24)
