"""Microscaled formats on the GPU against their definitions in 64 bits.

Quantising is exact by definition (a power-of-two scale, one rounding), so its values and
scales are equal.  Where a row op comes first, its f32 result y is off by at most REL |y|:
RMSNorm's squares are summed in f32 8 at a time, each with 8 roundings, then in double; half of
that of the root, and 4 more of h and its product with the factor and the weight: 8 * 2^-24;
residual_rms_norm, whose rows are compared with it, sums in f32: a chain of at most 128 terms a
thread and 10 levels of a tree, 138 * 2^-24 of the sum and half of that of its root, 6 more
roundings: 75 * 2^-24 < 2^-17.  SwiGLU has expf (2 ulp) and 4 roundings.
A code is then off by half a step of y + its error, with a scale that may be the next one
where the block's largest is within REL of a border.

The product sums cols / 32 partial sums of 32 terms in f32, each addition off by one unit of
the running sum at most (2^-23 of sum |x w|), 32 more for the terms of an instruction and 8
for the parts of a split; the bias and the output's rounding come last, each half a step:
finfo(bfloat16).eps / 2 = 2^-7 / 2 = 2^-8 of the value (8 significant bits: the tie 1 + 2^-8
lies between 1 and 1 + 2^-7), finfo(float32).eps / 2 = 2^-24.
"""
import numpy as np
import pytest
import torch

import mx_ref as R
import tb_b200 as T

pytestmark = pytest.mark.gpu

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
REL = 2.0 ** -17
FORMATS = ["e4m3", "e2m1"]


@pytest.fixture(autouse=True)
def _quiet(cuda):
    """No flag is raised by any call here."""
    T.check_status()
    yield
    assert T.check_status() == (0, 0)


def gen(seed):
    return torch.Generator("cuda").manual_seed(seed)


def normal(seed, *shape, dtype="f32", std=1.0):
    return (torch.randn(*shape, generator=gen(seed), device="cuda") * std).to(DTYPES[dtype])


def f64(t):
    return t.double().cpu().numpy()


def held(t):
    """(values, scale bytes [rows, blocks]) of an MxTensor; its fill is checked."""
    codes, scales = t.codes.cpu().numpy(), t.scales.cpu().numpy()
    rows, cols = t.rows, t.cols
    each = 1 if t.format == "e4m3" else 2
    wide = codes if each == 1 else np.stack([codes & 15, codes >> 4], -1).reshape(rows, -1)
    assert (wide[:, R.up(cols, 32):] == 0).all()  # (a last block that is NaN fills with NaN)
    places = R.scale_places(rows, cols)
    rest = np.delete(scales, places.ravel())
    assert (rest == 0).all()  # blocks and rows of the last tiles that are not there
    return R.values(codes, scales, cols, t.format), scales[places]


# ------------------------------------------------------------------ quantise
SHAPES = [(1, 1), (1, 32), (3, 31), (5, 128), (127, 129), (128, 256), (129, 100), (130, 333),
          (2, 4096), (1000, 96), (33, 2056)]


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_quantize(rows, cols, dtype, fmt):
    x = normal(1, rows, cols, dtype=dtype)
    x *= torch.exp2(torch.randint(-40, 40, (rows, cols), generator=gen(2), device="cuda") / 8.0)
    t = T.mx_quantize(x, fmt)
    got, scales = held(t)
    want, s = R.quantised(f64(x), fmt)
    assert np.array_equal(scales, s)
    assert np.array_equal(got, want)
    assert np.array_equal(f64(T.mx_dequantize(t)), want)
    assert torch.equal(T.mx_dequantize(t, torch.bfloat16), T.mx_dequantize(t).bfloat16())


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("off,stride", [(0, 400), (1, 401), (8, 408), (3, 336)])
def test_quantize_strided_rows(off, stride, dtype, fmt):
    big = normal(3, 70, stride, dtype=dtype)
    x = big[:, off:off + 333]
    got, scales = held(T.mx_quantize(x, fmt))
    want, s = R.quantised(f64(x), fmt)
    assert np.array_equal(scales, s) and np.array_equal(got, want)
    t = T.mx_quantize(x.contiguous(), fmt)
    y = torch.full((70, stride), 7.0, dtype=DTYPES[dtype], device="cuda")
    T.mx_dequantize(t, out=y[:, off:off + 333])
    assert np.array_equal(f64(y[:, off:off + 333]),
                          f64(torch.from_numpy(want).to(DTYPES[dtype])))
    y[:, off:off + 333] = 7.0
    assert (y == 7.0).all()  # nothing else was written


@pytest.mark.parametrize("fmt", FORMATS)
def test_quantize_borders(fmt):
    """Largest elements next to MAX 2^e, elements next to ties, both ends of f32."""
    most = R.LARGEST[fmt]
    rows = []
    for e in (-140, -127, -126, -20, -1, 0, 1, 60, 119):
        top = np.float32(np.ldexp(most, e))
        for v in (top, np.nextafter(top, np.float32(np.inf)), np.nextafter(top, np.float32(0))):
            row = np.zeros(32, np.float32)
            row[7] = -v
            row[8] = np.float32(v) / 3
            rows.append(row)
    mids = R.CODES[fmt][:127 if fmt == "e4m3" else 8]
    mids = ((mids[1:] + mids[:-1]) / 2).astype(np.float32)
    for m in mids:
        row = np.full(32, most, np.float32)
        row[:3] = m, np.nextafter(m, np.float32(0)), np.nextafter(m, np.float32(np.inf))
        row[3:6] = -row[:3]
        rows.append(row)
    rows.append(np.zeros(32, np.float32))
    rows.append(np.full(32, np.finfo(np.float32).max, np.float32))
    rows.append(np.full(32, 1e-45, np.float32))
    x = np.stack(rows)
    got, scales = held(T.mx_quantize(torch.from_numpy(x).cuda(), fmt))
    want, s = R.quantised(x.astype(np.float64), fmt)
    assert np.array_equal(scales, s) and np.array_equal(got, want)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_quantize_nan_stays_in_its_block(bad, fmt):
    x = normal(4, 3, 200)
    x[1, 70] = bad
    x[2, 199] = bad
    got, scales = held(T.mx_quantize(x, fmt))
    want, s = R.quantised(f64(x), fmt)
    assert np.array_equal(scales, s)
    assert np.array_equal(got, want, equal_nan=True)
    assert np.isnan(got).sum() == 32 + 8


# -------------------------------------------------- row ops into the formats
def check_codes(t, y):
    """t holds rows y (float64), computed in f32 to REL, in its format."""
    got, scales = held(t)
    rows, cols = y.shape
    full = np.zeros((rows, R.up(cols, 32)))
    full[:, :cols] = np.abs(y)
    amax = full.reshape(rows, -1, 32).max(-1)
    lo = R.scale_exponents(amax * (1 - REL), t.format) + 127
    hi = R.scale_exponents(amax * (1 + REL), t.format) + 127
    assert ((scales == lo) | (scales == hi)).all()
    s = np.repeat(np.ldexp(1.0, scales.astype(np.int64) - 127), 32, 1)[:, :cols]
    # half a step: 2^-4 of a value and 2^-10 of the scale, or 2^-2 of both
    half = np.maximum(np.abs(y) * 2.0 ** -4, s * 2.0 ** -10) if t.format == "e4m3" else \
        np.maximum(np.abs(y) * 2.0 ** -2, s * 2.0 ** -2)
    assert (np.abs(got - y) <= half * (1 + REL) + np.abs(y) * REL).all()


def norm_of(x, res, w, eps):
    h = x if res is None else x + res
    y = h / np.sqrt((eps + (h * h).sum(-1, keepdims=True)) / x.shape[1])
    return h, y if w is None else y * w


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 100), (3, 256), (130, 1024), (77, 4100),
                                       (5, 8192), (2, 16384), (3, 33000), (2, 70000)])
def test_residual_rms_norm_mx(rows, cols, dtype, fmt):
    x, res = normal(5, rows, cols, dtype=dtype), normal(6, rows, cols, dtype=dtype, std=2.0)
    w = 1 + normal(7, cols, dtype=dtype, std=0.1)
    h, y = T.residual_rms_norm_mx(x, res, w, 1e-5, format=fmt)
    want_h, want = norm_of(f64(x), f64(res), f64(w), 1e-5)
    assert torch.equal(h, (x.float() + res.float()).to(x.dtype))
    check_codes(y, want)


@pytest.mark.parametrize("has_res,has_w", [(False, False), (False, True), (True, False)])
def test_residual_rms_norm_mx_parts(has_res, has_w):
    x, res = normal(8, 9, 500, dtype="bf16"), normal(9, 9, 500, dtype="bf16")
    w = 1 + normal(10, 500, dtype="bf16", std=0.1)
    h, y = T.residual_rms_norm_mx(x, res if has_res else None, w if has_w else None, 1e-5)
    check_codes(y, norm_of(f64(x), f64(res) if has_res else None, f64(w) if has_w else None,
                           1e-5)[1])
    assert (h is None) == (not has_res)


@pytest.mark.parametrize("cols", [512, 515, 70001])
@pytest.mark.parametrize("into", ["x", "residual"])
def test_residual_rms_norm_mx_in_place(into, cols):
    x, res = normal(11, 4, cols), normal(12, 4, cols)
    want_h, want = norm_of(f64(x), f64(res), None, 1e-5)
    sum_ = x + res
    h, y = T.residual_rms_norm_mx(x, res, None, 1e-5, h_out=x if into == "x" else res)
    assert h is (x if into == "x" else res) and torch.equal(h, sum_)
    check_codes(y, want)


def test_residual_rms_norm_mx_is_the_row_norm():
    """The same f32 rows as residual_rms_norm, which stores them in f32."""
    x, res = normal(13, 50, 4096), normal(14, 50, 4096)
    w = 1 + normal(15, 4096, std=0.1)
    _, y = T.residual_rms_norm(x, res, w, 1e-5)
    _, t = T.residual_rms_norm_mx(x, res, w, 1e-5)
    check_codes(t, f64(y))


def test_residual_rms_norm_mx_of_a_row_with_nan():
    x, res = normal(16, 5, 300), normal(17, 5, 300)
    clean = T.residual_rms_norm_mx(x, res, None, 1e-5)[1]
    want = held(clean)[0]
    x[2, 5] = np.nan
    x[3, 299] = np.inf
    got = held(T.residual_rms_norm_mx(x, res, None, 1e-5)[1])[0]
    assert np.isnan(got[2]).all()  # the whole row's scale is NaN
    # a row's infinity gives a scale of zero: its own block is NaN, the others are 0
    assert np.isnan(got[3, 288:]).all() and (got[3, :288] == 0).all()
    keep = [0, 1, 4]
    assert np.array_equal(got[keep], want[keep])


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 100), (129, 1024), (7, 11008)])
def test_swiglu_mx(rows, cols, dtype, fmt):
    both = normal(18, rows, 2 * cols, dtype=dtype, std=2.0)
    gate, up = both[:, :cols], both[:, cols:]
    t = T.swiglu_mx(gate, up, fmt)
    g, u = f64(gate), f64(up)
    check_codes(t, g / (1 + np.exp(-g)) * u)
    t2 = T.swiglu_mx(gate.contiguous(), up.contiguous(), fmt)
    assert torch.equal(t.codes, t2.codes) and torch.equal(t.scales, t2.scales)


@pytest.mark.parametrize("fmt", FORMATS)
def test_swiglu_mx_is_the_row_op(fmt):
    """swiglu's f32 rows, bit for bit, at gates of all sizes and next to its branches."""
    g = normal(54, 300, 4096) * torch.exp2(
        torch.randint(-60, 12, (300, 4096), generator=gen(55), device="cuda") / 2.0)
    one = torch.ldexp(torch.ones(4096, device="cuda"), torch.arange(4096, device="cuda") % 200 - 140)
    near = torch.nextafter(one, 2 * one)
    g[:4] = torch.stack([one, -one, near, -near])
    g[4] = torch.linspace(79.9, 80.1, 4096, device="cuda")
    g[5] = -torch.linspace(79.9, 110, 4096, device="cuda")
    u = normal(56, 300, 4096)
    t, want = T.swiglu_mx(g, u, fmt), T.mx_quantize(T.swiglu(g, u), fmt)
    assert torch.equal(t.scales, want.scales) and torch.equal(t.codes, want.codes)


# ---------------------------------------------------------------- the product
def linear_of(x, w, bias=None):
    """(x w^T + bias, the bound on sum |x w|'s error) in float64."""
    x, w = (R.values(t.codes.cpu().numpy(), t.scales.cpu().numpy(), t.cols, t.format)
            for t in (x, w))
    y = x @ w.T + (0 if bias is None else f64(bias))
    near = (x.shape[1] / 32 + 40) * 2.0 ** -23 * (np.abs(x) @ np.abs(w).T)
    return y, near


def check_linear(x, w, bias, y):
    want, near = linear_of(x, w, bias)
    half = torch.finfo(y.dtype).eps / 2
    got = f64(y)
    assert got.shape == want.shape
    off = np.abs(got - want) - near - (1 if bias is None else 2) * half * np.abs(want)
    assert off.max(initial=0.0) <= 2.0 ** -140


@pytest.mark.parametrize("xf,wf", [("e4m3", "e4m3"), ("e4m3", "e2m1"), ("e2m1", "e4m3"),
                                   ("e2m1", "e2m1")])
@pytest.mark.parametrize("rows,cols,outs", [
    (1, 128, 128), (1, 32, 1), (16, 256, 128), (17, 128, 130), (2, 4096, 256), (64, 384, 300),
    (65, 100, 16), (128, 1000, 129), (129, 512, 127), (256, 128, 128), (257, 640, 200),
    (700, 300, 1000), (1, 1, 1), (3, 11008, 100)])
def test_linear(rows, cols, outs, xf, wf):
    x = T.mx_quantize(normal(20, rows, cols), xf)
    w = T.mx_quantize(normal(21, outs, cols, std=0.05), wf)
    bias = normal(22, outs)
    check_linear(x, w, None, T.mx_linear(x, w))
    check_linear(x, w, bias, T.mx_linear(x, w, bias, torch.float32))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("off", [0, 3])
@pytest.mark.parametrize("xf,rows,cols,outs", [
    ("e4m3", 1290, 300, 4100), ("e2m1", 1290, 640, 4100), ("e2m1", 1290, 200, 4100),
    ("e4m3", 100, 300, 40007), ("e2m1", 100, 300, 40007), ("e4m3", 30, 1100, 40007),
    ("e2m1", 30, 2100, 40007), ("e4m3", 1, 1024, 57000), ("e4m3", 128, 1024, 40007)])
def test_linear_of_several_tiles_a_cta(xf, rows, cols, outs, off, dtype):
    """More tiles than CTAs, the last of them ragged; rows of y aligned or not."""
    x, w = T.mx_quantize(normal(57, rows, cols), xf), T.mx_quantize(normal(58, outs, cols), "e2m1")
    stride = (outs + 15) // 8 * 8 + off % 2
    y = torch.full((rows, stride), 7.0, dtype=DTYPES[dtype], device="cuda")
    bias = normal(59, outs)
    T.mx_linear(x, w, bias, y=y[:, off:off + outs])
    check_linear(x, w, bias, y[:, off:off + outs])
    assert (y[:, :off] == 7.0).all() and (y[:, off + outs:] == 7.0).all()


@pytest.mark.parametrize("cols,outs", [(1600, 10240), (2600, 6100), (3200, 5100), (3600, 300),
                                       (4200, 700), (1100, 300)])
@pytest.mark.parametrize("xf", FORMATS)
def test_linear_in_parts_of_cols(xf, cols, outs):
    """2 to 8 CTAs a tile, by the number of tiles and of steps."""
    x, w = T.mx_quantize(normal(62, 5, cols), xf), T.mx_quantize(normal(63, outs, cols), "e2m1")
    bias = normal(64, outs)
    y = T.mx_linear(x, w, bias, torch.float32)
    check_linear(x, w, bias, y)
    assert torch.equal(T.mx_linear(x, w, bias, torch.float32), y)


@pytest.mark.parametrize("rows", [2, 200])
def test_linear_of_far_larger_codes_and_scales(rows):
    """Codes and scales that did not come from mx_quantize: every code but NaN, any scale."""
    def raw(seed, rows, cols, fmt):
        t = T.MxTensor.empty(rows, cols, fmt)
        c = torch.randint(0, 256, t.codes.shape, generator=gen(seed), device="cuda")
        if fmt == "e4m3":
            c = torch.where((c & 127) == 127, c - 1, c)
        t.codes.copy_(c)
        t.scales.copy_(torch.randint(90, 160, t.scales.shape, generator=gen(seed), device="cuda"))
        return t
    for xf in FORMATS:
        for wf in FORMATS:
            x, w = raw(60, rows, 384, xf), raw(61, 140, 384, wf)
            check_linear(x, w, None, T.mx_linear(x, w, dtype=torch.float32))


@pytest.mark.parametrize("xf,wf", [("e4m3", "e2m1"), ("e2m1", "e2m1")])
def test_linear_scales_of_all_sizes(xf, wf):
    """Blocks whose scales span f32's exponents: a wrong row's or block's scale shows."""
    def wild(seed, rows, cols):
        e = torch.randint(-50, 50, (rows, -(-cols // 32)), generator=gen(seed), device="cuda")
        return normal(seed, rows, cols) * torch.exp2(e.float()).repeat_interleave(32, 1)[:, :cols]
    for rows, cols, outs in [(5, 500, 140), (300, 1000, 260)]:
        x, w = T.mx_quantize(wild(23, rows, cols), xf), T.mx_quantize(wild(24, outs, cols), wf)
        check_linear(x, w, None, T.mx_linear(x, w, dtype=torch.float32))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [3, 300])
def test_linear_writes_its_rows_only(rows, dtype):
    x = T.mx_quantize(normal(25, rows, 256))
    w = T.mx_quantize(normal(26, 200, 256), "e2m1")
    big = torch.full((rows + 2, 333), 7.0, dtype=DTYPES[dtype], device="cuda")
    y = big[1:-1, 5:205]
    assert T.mx_linear(x, w, y=y) is y
    check_linear(x, w, None, y.clone())
    y.fill_(7.0)
    assert (big == 7.0).all()


def test_linear_of_parts_of_tensors():
    """The first rows of x, and rows of w from a multiple of 128 on, are tensors."""
    x = T.mx_quantize(normal(27, 300, 640))
    w = T.mx_quantize(normal(28, 500, 640), "e2m1")
    whole = T.mx_linear(x, w)
    for n in (1, 40, 256, 290):
        first = T.MxTensor(x.codes[:n], x.scales[:-(-n // 128) * 5 * 512], 640, "e4m3")
        part = T.MxTensor(w.codes[128:], w.scales[5 * 512:], 640, "e2m1")
        check_linear(first, part, None, T.mx_linear(first, part))
        if n == 256:
            assert torch.equal(T.mx_linear(first, w), whole[:n])


@pytest.mark.parametrize("xf,wf", [("e4m3", "e4m3"), ("e4m3", "e2m1"), ("e2m1", "e2m1")])
@pytest.mark.parametrize("rows", [4, 270])
def test_linear_nan_stays_in_its_row_and_column(rows, xf, wf):
    xs, ws = normal(29, rows, 300), normal(30, 150, 300)
    clean = T.mx_linear(T.mx_quantize(xs, xf), T.mx_quantize(ws, wf))
    xs[1, 299] = np.nan
    ws[140, 0] = np.inf
    y = T.mx_linear(T.mx_quantize(xs, xf), T.mx_quantize(ws, wf))
    assert y[1].isnan().all() and y[:, 140].isnan().all()
    clean[1] = np.nan
    clean[:, 140] = np.nan
    assert torch.equal(y.isnan(), clean.isnan())
    assert torch.equal(y.nan_to_num(), clean.nan_to_num())


def test_linear_is_the_same_each_time():
    x = T.mx_quantize(normal(31, 20, 8192))
    w = T.mx_quantize(normal(32, 1000, 8192), "e2m1")
    y = T.mx_linear(x, w)
    for _ in range(5):
        assert torch.equal(T.mx_linear(x, w), y)


def test_empty_calls():
    for fmt in FORMATS:
        t = T.mx_quantize(torch.empty(0, 40, device="cuda"), fmt)
        assert T.mx_dequantize(t).shape == (0, 40)
        w = T.mx_quantize(normal(33, 5, 40), fmt)
        assert T.mx_linear(t, w).shape == (0, 5)
        assert T.mx_linear(w, t).shape == (5, 0)
        assert T.swiglu_mx(torch.empty(0, 40, device="cuda"),
                           torch.empty(0, 40, device="cuda"), fmt).rows == 0
        assert T.residual_rms_norm_mx(torch.empty(0, 40, device="cuda"), None, None, 1e-5,
                                      format=fmt)[1].rows == 0


# ----------------------------------------------------------------- as used
class Mlp:
    """norm -> gate and up -> SwiGLU -> down, as a decoder layer has them."""

    def __init__(self, hidden, inner, fmt):
        self.norm = (1 + 0.1 * normal(40, hidden)).bfloat16()
        self.gate_up = T.mx_quantize(normal(41, 2 * inner, hidden, std=hidden ** -0.5), "e2m1")
        self.down = T.mx_quantize(normal(42, hidden, inner, std=inner ** -0.5), "e2m1")
        self.inner, self.fmt = inner, fmt

    def __call__(self, x, res):
        h, y = T.residual_rms_norm_mx(x, res, self.norm, 1e-5, format=self.fmt)
        both = T.mx_linear(y, self.gate_up)
        act = T.swiglu_mx(both[:, :self.inner], both[:, self.inner:], self.fmt)
        return h, y, both, act, T.mx_linear(act, self.down)

    def check(self, x, res, got):
        h, y, both, act, out = got
        want_h, want = norm_of(f64(x), f64(res), f64(self.norm), 1e-5)
        assert torch.equal(h, (x.float() + res.float()).bfloat16())
        check_codes(y, want)
        check_linear(y, self.gate_up, None, both)
        b = f64(both)
        g, u = b[:, :self.inner], b[:, self.inner:]
        check_codes(act, g / (1 + np.exp(-g)) * u)
        check_linear(act, self.down, None, out)


@pytest.mark.parametrize("rows", [1, 5, 140])
@pytest.mark.parametrize("fmt", FORMATS)
def test_layer(rows, fmt):
    mlp = Mlp(512, 1408, fmt)
    x, res = normal(43, rows, 512, dtype="bf16"), normal(44, rows, 512, dtype="bf16")
    mlp.check(x, res, mlp(x, res))


def test_layer_from_a_graph_beside_another_stream():
    """A captured layer replayed on new inputs while another stream runs the same calls."""
    mlp = Mlp(512, 1408, "e4m3")
    x, res = normal(45, 4, 512, dtype="bf16"), normal(46, 4, 512, dtype="bf16")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        mlp(x, res)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = mlp(x, res)
    x2, res2 = normal(47, 200, 512, dtype="bf16"), normal(48, 200, 512, dtype="bf16")
    torch.cuda.synchronize()
    for seed in (49, 50, 51):
        x.copy_(normal(seed, 4, 512, dtype="bf16"))
        torch.cuda.synchronize()
        graph.replay()
        with torch.cuda.stream(side):
            beside = mlp(x2, res2)
        torch.cuda.synchronize()
        mlp.check(x, res, got)
        mlp.check(x2, res2, beside)


def test_calls_on_a_given_stream():
    side = torch.cuda.Stream()
    x, w = normal(52, 30, 1000), normal(53, 260, 1000)
    torch.cuda.synchronize()
    s = side.cuda_stream
    tx, tw = T.mx_quantize(x, stream=s), T.mx_quantize(w, "e2m1", stream=s)
    y = T.mx_linear(tx, tw, stream=s)
    v = T.mx_dequantize(tx, stream=s)
    side.synchronize()
    check_linear(tx, tw, None, y)
    assert np.array_equal(f64(v), R.quantised(f64(x), "e4m3")[0])
