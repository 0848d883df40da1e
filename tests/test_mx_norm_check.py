"""What the check of the norm's codes notices, on the CPU: the kernel's steps restated, right and with
mistakes."""
from types import SimpleNamespace

import numpy as np
import pytest
import torch

import mx_ref as R
from test_gpu_mx_norm import check_rounded, next_to_borders, norm_of

F, W = np.float32, np.longdouble  # 64 bits of mantissa: an fma's sum, before it is rounded


def fma(a, b, c):
    return (a.astype(W) * b.astype(W) + c.astype(W)).astype(F)


def values(h, w, eps, mistake):
    """A row's f32 values as the kernel has them."""
    a = h.astype(np.float64)
    sum_ = (a * a).sum() if mistake != "sums in f32" else np.float64((h * h).astype(F).sum(dtype=F))
    s = np.sqrt(h.shape[1]) / np.sqrt(eps + sum_)
    hi = F(s)
    lo = F(s - np.float64(hi)) if mistake != "factor of one part" else F(0)
    hi, lo = np.full_like(h, hi), np.full_like(h, lo)
    t = (h * hi).astype(F)
    left = fma(h, lo, fma(h, hi, -t))
    y = (t * w).astype(F)
    rest = fma(left, w, fma(t, w, -y))
    if mistake == "rounded twice":
        return y
    return fma(t, w, rest) if mistake == "residual counted twice" else (y + rest).astype(F)


def held_as(y, fmt):
    """Rows of 32 columns at most, as a tensor of the format."""
    v, scales = R.quantised(y.astype(np.float64), fmt)
    rows, cols = y.shape
    codes = np.searchsorted(R.CODES[fmt][:127 if fmt == "e4m3" else 8],
                            np.abs(np.ldexp(v, 127 - scales.astype(np.int64)))).astype(np.uint8)
    codes |= (np.signbit(v) * (128 if fmt == "e4m3" else 8)).astype(np.uint8)
    wide = np.zeros((rows, 128), np.uint8)
    wide[:, :cols] = codes
    if fmt == "e2m1":
        wide = wide[:, ::2] | wide[:, 1::2] << 4
    tiled = np.zeros(512, np.uint8)
    tiled[R.scale_places(rows, cols)] = scales
    return SimpleNamespace(codes=torch.from_numpy(wide), scales=torch.from_numpy(tiled), rows=rows,
                           cols=cols, format=fmt)


@pytest.mark.parametrize("fmt", ["e4m3", "e2m1"])
@pytest.mark.parametrize("mistake", [None, "sums in f32", "factor of one part", "rounded twice",
                                     "residual counted twice"])
def test_mistakes_are_noticed(mistake, fmt):
    noticed = 0
    for seed in range(300):
        h = np.random.default_rng(seed).standard_normal((1, 32)).astype(F)
        w = next_to_borders(h.astype(np.float64), fmt, 1e-5, seed)
        y = values(h, w, 1e-5, mistake)
        try:
            check_rounded(held_as(y, fmt), norm_of(h.astype(np.float64), w.astype(np.float64), 1e-5))
        except AssertionError:
            noticed += 1
    assert (noticed == 0) if mistake is None else (noticed > 0), noticed
