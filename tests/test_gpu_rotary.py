"""Rotary positions and head norms (tb_b200_rotary, tb_b200_qk_norm_rotary,
tb_b200_rotary_freqs) against their formulas in 64 bits.

Tolerances, with u = 2^-24 (half a step of f32, relative):
- cos and sin are off by at most 1 ulp of sincospif (u, for values up to 1),
  2u of the first-order correction and u of the scaling; the two products and
  their sum add 2u of the larger sum: below 6u m (|x0| + |x1|) in all.
- a norm's sum of squares has at most 16 terms per lane, 5 shuffle steps and
  the products: 22u, 1 / d and the product and sum with it 2u, all halved by
  the root; rsqrtf's 2 ulp are 4u, two products 2u: 18u, below 20u.
- bf16 outputs are rounded once more, by at most 2^-8 of the value.
- the frequencies: pow in double within 2 ulp, 3 more operations: 2^-49.
"""
import math

import numpy as np
import pytest

import tb_b200 as T

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


@pytest.fixture(scope="module")
def dev(cuda):
    import torch
    torch.cuda.set_device(cuda)
    return cuda


def f64(t):
    return t.detach().double().cpu().numpy()


def want(x, w, eps, pos, freqs, layout, scale, norm):
    """(y, |terms|): the formula in 64 bits and what its errors are relative to."""
    x = f64(x)
    rel = 6 * U
    if norm:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * (1 if w is None else f64(w))
        rel += 20 * U
    r = 0 if freqs is None else 2 * len(freqs)
    y, mag = x.copy(), np.abs(x)
    if r:
        a = pos.astype(np.float64)[:, None, None] * freqs
        c, s = scale * np.cos(a), scale * np.sin(a)
        i = np.arange(r // 2)
        p, q = (i, i + r // 2) if layout == T.ROTARY_HALF else (2 * i, 2 * i + 1)
        y[..., p] = x[..., p] * c - x[..., q] * s
        y[..., q] = x[..., q] * c + x[..., p] * s
        mag[..., p] = mag[..., q] = scale * (np.abs(x[..., p]) + np.abs(x[..., q]))
    return y, rel * mag


def check(got, y, tol, bf16):
    got = f64(got)
    assert (np.abs(got - y) <= tol + (2.0 ** -8 * np.abs(y) if bf16 else 0) + 1e-37).all(), (
        np.abs(got - y) / np.maximum(tol, 1e-37)).max()


def inputs(dev, rows, hq, hkv, d, bf16, seed=0, pad=0, offset=0, tail=True):
    """q and k slices of one packed row of (hq + 2 hkv) d + pad elements."""
    import torch
    g = torch.Generator().manual_seed(seed + rows + d)
    width = (hq + 2 * hkv) * d + pad
    buf = torch.randn(rows * width + offset, generator=g)
    buf = buf.to(torch.bfloat16 if bf16 else torch.float32).to(dev)
    x = buf[offset:].view(rows, width)
    q = x[:, :hq * d].unflatten(1, (hq, d)) if hq else x[:, :0].reshape(rows, 0, d)
    k = x[:, hq * d:(hq + hkv) * d].unflatten(1, (hkv, d))
    pos = torch.randint(0, 1 << 20, (rows,), generator=g, dtype=torch.int32)
    w = [(1 + 0.2 * torch.randn(d, generator=g)).to(q.dtype).to(dev) for _ in range(2)]
    return q, k, pos, w


def freqs_of(r, theta=1e4):
    return theta ** (-2.0 * np.arange(r // 2) / r)


SHAPES = [  # rows, hq, hkv, d, r
    (1, 4, 4, 64, 64), (3, 1, 1, 128, 128), (65, 64, 8, 128, 128), (7, 32, 32, 80, 32),
    (5, 7, 1, 96, 48), (9, 3, 2, 256, 256), (4, 2, 1, 512, 512), (2, 5, 3, 40, 40),
    (6, 2, 2, 30, 6), (3, 2, 1, 1, 0), (2, 3, 1, 17, 16), (11, 2, 2, 64, 2), (300, 9, 1, 72, 24),
    (2, 1, 1, 511, 510), (1, 40, 8, 128, 64)]


@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("layout", [T.ROTARY_INTERLEAVED, T.ROTARY_HALF])
@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("rows,hq,hkv,d,r", SHAPES)
def test_rotary(dev, rows, hq, hkv, d, r, bf16, layout, norm):
    import torch
    q, k, pos, w = inputs(dev, rows, hq, hkv, d, bf16)
    fr = freqs_of(r) if r else None
    frd = torch.from_numpy(fr).to(dev) if r else None
    scale = 1.25 if d == 128 else 1.0
    if norm:
        got = T.qk_norm_rotary(q, k, w[0], w[1], 1e-6, pos.to(dev) if r else None, frd, layout,
                               scale)
    elif not r:
        return
    else:
        got = T.rotary(q, k, pos.to(dev), frd, layout, scale)
    for g, x, wx in zip(got, (q, k), w):
        check(g, *want(x, wx, 1e-6, pos.numpy(), fr, layout, scale, norm), bf16)


@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("pad,offset", [(1, 0), (0, 1), (4, 4), (8, 2), (3, 5)])
def test_strides_and_alignment(dev, bf16, norm, pad, offset):
    """Rows of every stride and start, outputs into padded buffers whose other
    elements stay as they were."""
    import torch
    rows, hq, hkv, d, r = 33, 5, 2, 64, 32
    q, k, pos, w = inputs(dev, rows, hq, hkv, d, bf16, pad=pad, offset=offset)
    fr = freqs_of(r)
    for layout in (T.ROTARY_INTERLEAVED, T.ROTARY_HALF):
        out = torch.full((rows, (hq + hkv) * d + 7), -3.0, dtype=q.dtype, device=dev)
        qo = out[:, :hq * d].unflatten(1, (hq, d))
        ko = out[:, hq * d + 7:].unflatten(1, (hkv, d))
        args = (pos.to(dev), torch.from_numpy(fr).to(dev), layout)
        if norm:
            T.qk_norm_rotary(q, k, w[0], None, 1e-5, *args, q_out=qo, k_out=ko)
        else:
            T.rotary(q, k, *args, q_out=qo, k_out=ko)
        for g, x, wx in zip((qo, ko), (q, k), (w[0], None)):
            check(g, *want(x, wx, 1e-5, pos.numpy(), fr, layout, 1.0, norm), bf16)
        assert bool((out[:, hq * d:hq * d + 7] == -3.0).all())


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("layout", [T.ROTARY_INTERLEAVED, T.ROTARY_HALF])
def test_in_place_equals_out_of_place(dev, bf16, layout):
    import torch
    q, k, pos, w = inputs(dev, 130, 8, 2, 128, bf16)
    q, k = q.clone(), k.clone()
    fr = torch.from_numpy(freqs_of(64)).to(dev)
    for norm in (False, True):
        a, b = q.clone(), k.clone()
        args = (pos.to(dev), fr, layout)
        if norm:
            want_ = T.qk_norm_rotary(q, k, w[0], w[1], 1e-6, *args)
            T.qk_norm_rotary(a, b, w[0], w[1], 1e-6, *args, q_out=a, k_out=b)
        else:
            want_ = T.rotary(q, k, *args)
            T.rotary(a, b, *args, q_out=a, k_out=b)
        assert torch.equal(a, want_[0]) and torch.equal(b, want_[1])


def test_far_negative_and_zero_positions(dev):
    import torch
    pos = np.array([0, -1, -(2 ** 31), 2 ** 31 - 1, 131071, 16777217], np.int32)
    q, k, _, _ = inputs(dev, len(pos), 2, 1, 128, False)
    fr = freqs_of(128, 5e5)
    got = T.rotary(q, k, torch.from_numpy(pos).to(dev), torch.from_numpy(fr).to(dev))
    for g, x in zip(got, (q, k)):
        y, tol = want(x, None, 0, pos, fr, T.ROTARY_HALF, 1.0, False)
        # at 2^31 the angle p f itself has an ulp of 2^-22 in 64 bits, on both sides
        far = (np.abs(pos.astype(np.float64)) > 2 ** 25)[:, None, None]
        check(g, y, tol * np.where(far, 16, 1), False)
    assert torch.equal(got[0][0], q[0])  # position 0 turns nothing


def test_norm_of_zeros_infinities_and_lone_heads(dev):
    import torch
    q = torch.zeros(3, 2, 64, device=dev)
    q[1, 0, 5] = float("inf")
    q[2, 1, 7] = float("nan")
    k = torch.ones(3, 0, 64, device=dev)
    qo, ko = T.qk_norm_rotary(q, k, None, None, 1e-6)
    assert ko.shape == (3, 0, 64)
    assert bool((qo[0] == 0).all()) and bool((qo[1, 1] == 0).all()) and bool((qo[2, 0] == 0).all())
    assert bool(torch.isnan(qo[1, 0, 5])) and bool(torch.isnan(qo[2, 1]).all())


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("layout", [T.ROTARY_INTERLEAVED, T.ROTARY_HALF])
def test_infinities_stay_in_their_pair(dev, bf16, layout):
    """What is past the rotated part is passed through, whatever stands beside it."""
    import torch
    for d, r in ((80, 32), (64, 16), (17, 6)):
        q, k, pos, _ = inputs(dev, 5, 3, 2, d, bf16)
        q, k = q.clone(), k.clone()
        q[:, :, r + 1::3] = float("inf")
        q[:, 1, r + 2::5] = float("nan")
        fr = freqs_of(r)
        got, _ = T.rotary(q, k, pos.to(dev), torch.from_numpy(fr).to(dev), layout)
        assert torch.equal(got[:, :, r:].nan_to_num(7.0, 8.0, 9.0),
                           q[:, :, r:].nan_to_num(7.0, 8.0, 9.0))
        clean = torch.where(torch.isfinite(q), q, torch.zeros_like(q))
        y, tol = want(clean, None, 0, pos.numpy(), fr, layout, 1.0, False)
        check(got[:, :, :r], y[..., :r], tol[..., :r], bf16)


SCALINGS = [("none", 1.0, 0, 0, 0), ("linear", 4.0, 0, 0, 0), ("ntk", 8.0, 0, 0, 0),
            ("bands", 8.0, 8192, 1.0, 4.0), ("yarn", 16.0, 4096, 1.0, 32.0)]


@pytest.mark.parametrize("kind,factor,trained,low,high", SCALINGS)
@pytest.mark.parametrize("r,theta", [(64, 1e4), (128, 5e5), (16, 1e6), (512, 1e4), (4, 1e4)])
def test_frequencies(dev, kind, factor, trained, low, high, r, theta):
    i = np.arange(r // 2)
    if kind == "ntk":
        theta_ = theta * factor ** (r / (r - 2))
    else:
        theta_ = theta
    f = theta_ ** (-2.0 * i / r)
    if kind == "linear":
        f = f / factor
    elif kind == "bands":  # by wavelength, as the method is usually stated
        out = []
        for x in f:
            wave = 2 * math.pi / x
            if wave < trained / high:
                out.append(x)
            elif wave > trained / low:
                out.append(x / factor)
            else:
                smooth = (trained / wave - low) / (high - low)
                out.append((1 - smooth) * x / factor + smooth * x)
        f = np.array(out)
    elif kind == "yarn":
        def at(t):
            return r * math.log(trained / (t * 2 * math.pi)) / (2 * math.log(theta))
        lo, hi = max(math.floor(at(high)), 0), min(math.ceil(at(low)), r - 1)
        ramp = np.clip((i - lo) / ((hi - lo) or 0.001), 0, 1)
        f = f / factor * ramp + f * (1 - ramp)
    got = f64(T.rotary_freqs(r, theta, kind, factor, trained, low, high))
    # the bands' test of a wavelength and the ramp cancel at most 6 bits
    assert (np.abs(got - f) <= 2.0 ** -43 * f).all()


def test_graph_stream_and_new_frequencies(dev):
    """A captured call replays with new rows, positions and frequencies, on a
    stream of its own."""
    import torch
    q, k, pos, w = inputs(dev, 17, 4, 2, 64, True)
    q, k, pos = q.clone(), k.clone(), pos.to(dev)
    fr = torch.empty(32, dtype=torch.float64, device=dev)
    qo, ko = torch.empty_like(q), torch.empty_like(k)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        T.rotary_freqs(64, 1e4, "linear", 2.0, out=fr)
        T.qk_norm_rotary(q, k, w[0], w[1], 1e-6, pos, fr, q_out=qo, k_out=ko)
    for step in range(3):
        q.copy_(torch.randn(q.shape, device=dev))
        pos.add_(1000 * step)
        graph.replay()
        torch.cuda.synchronize()
        f = freqs_of(64) / 2
        check(qo, *want(q, w[0], 1e-6, pos.cpu().numpy(), f, T.ROTARY_HALF, 1.0, True), True)
    s2 = torch.cuda.Stream()
    s2.wait_stream(torch.cuda.current_stream())
    a, _ = T.rotary(q, k, pos, fr, stream=s2.cuda_stream)
    s2.synchronize()
    assert torch.equal(a, T.rotary(q, k, pos, fr)[0])


def test_python_refusals(dev):
    import torch
    q, k, pos, w = inputs(dev, 4, 2, 1, 64, False)
    pos = pos.to(dev)
    fr = torch.from_numpy(freqs_of(64)).to(dev)
    with pytest.raises(TypeError):
        T.rotary(q, k, pos.long(), fr)
    with pytest.raises(TypeError):
        T.rotary(q, k, pos, fr.float())
    with pytest.raises(TypeError):
        T.rotary(q, k.bfloat16(), pos, fr)
    with pytest.raises(ValueError):
        T.rotary(q, k[:3], pos, fr)
    with pytest.raises(ValueError):
        T.rotary(q, k, pos[:3], fr)
    with pytest.raises(ValueError):
        T.rotary(q.transpose(0, 1), k, pos, fr)
    with pytest.raises(ValueError):
        T.qk_norm_rotary(q, k, w[0][:32], None, 1e-6, pos, fr)
    with pytest.raises(T.TbError):
        T.rotary(q, k, pos, torch.ones(33, dtype=torch.float64, device=dev))
    with pytest.raises(T.TbError):
        T.rotary(q, k, pos, fr, layout=3)
