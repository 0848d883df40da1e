"""The paged 8-bit KV cache (tb_b200_kv8_append, tb_b200_kv8_attention)
against its definition in 64 bits.

append: codes and scales are exact -- scaling by a power of two loses nothing,
so every code is the nearest one of an exact quotient -- and compared for
equality.

attention, per output element, with A = sum_j p_j |v_j| and, per row,
S = scale max_j sum_i |q_i k_ij|:
- a score is off by at most ds = S (d / 16 + 16) 2^-23 + R 2^-22: one f32
  rounding or truncation per group of 16 products and the scalings; and q held
  to 2^-22 of its row's largest element, so R = scale max_i |q_i| max_j sum_i |k_ij|;
- p_j is off by 2 ds relative (its own score and the maximum's), 2^-21 for
  exp2 and its argument, and, for bf16 calls, 2^-11 for p as f16;
- the sum over n keys is accumulated in f32 by groups of 16: (n / 16 + 16) 2^-23;
- the weights p_j scale_j (scale_j the page's for v) are held as f16, or two of
  them, times 2^11 over a power of two that is at most twice the largest: where
  that is subnormal its half step 2^-25 is 2^-35 of the largest, so the output
  is off by 2^-35 max_j(p_j scale_j) sum_j |code_j| however small p_j |v_j| is;
- the output is rounded by 2^-24, or 2^-8 as bf16.
lse: ds and (n / 16 + 16) 2^-23 for the sum, 2^-21 for exp2 and log.
"""
import math

import numpy as np
import pytest

import tb_b200 as T

pytestmark = pytest.mark.gpu
MOST = {"int8": 127.0, "e4m3": 448.0}


@pytest.fixture(scope="module")
def dev(cuda):
    import torch
    torch.cuda.set_device(cuda)
    T.check_status()
    return cuda


def nearest(x, fmt):
    if fmt == "int8":
        return np.rint(x)
    e = np.maximum(np.frexp(x)[1] - 1, -6)
    step = np.ldexp(1.0, e - 3)
    return np.rint(x / step) * step


def scale_for(amax, fmt):
    s = 2.0 ** -100
    while amax > MOST[fmt] * s:
        s *= 2
    return s


class Model:
    """A cache and its batch in 64 bits, beside the device's."""

    def __init__(self, dev, fmt, page, hkv, d, n_pages, seed=0):
        import torch
        self.fmt, self.page, self.hkv, self.d, self.dev = fmt, page, hkv, d, dev
        self.rng = np.random.default_rng(seed + page + d)
        dt = torch.int8 if fmt == "int8" else torch.float8_e4m3fn
        self.cache = T.Kv8Cache.empty(n_pages, hkv, page, d, dt)
        # what was in the memory before: any codes, NaN ones among them
        for t in (self.cache.k, self.cache.v):
            t.view(torch.uint8).copy_(torch.from_numpy(
                self.rng.integers(0, 256, t.shape, dtype=np.uint8)))
        self.cache.k_scale.fill_(float("nan"))
        self.cache.v_scale.fill_(float("nan"))
        self.codes = [f64(t) for t in (self.cache.k, self.cache.v)]
        self.scales = [np.full((n_pages, hkv), np.nan) for _ in range(2)]

    def append(self, xs, starts, lengths, table):
        for x, codes, scales in zip(xs, self.codes, self.scales):
            for i, total in enumerate(lengths):
                rows = x[starts[i]:starts[i + 1]]
                first = total - len(rows)
                for lp in range(max(first, 0) // self.page, -(-total // self.page)):
                    a, b = max(first, lp * self.page, 0), min(total, (lp + 1) * self.page)
                    if a >= b:
                        continue
                    at, slot = table[i][lp], a - lp * self.page
                    part = rows[a - first:b - first]
                    for h in range(self.hkv):
                        p = part[:, h]
                        fin = np.abs(p[np.isfinite(p)])
                        s = scale_for(fin.max() if fin.size else 0.0, self.fmt)
                        if slot:
                            s = max(s, scales[at, h])
                            old = codes[at, h, :slot]
                            codes[at, h, :slot] = nearest(old * (scales[at, h] / s), self.fmt)
                        q = np.clip(np.nan_to_num(p / s, nan=0.0, posinf=1e9, neginf=-1e9),
                                    -MOST[self.fmt], MOST[self.fmt])
                        codes[at, h, slot:slot + len(p)] = nearest(q, self.fmt)
                        scales[at, h] = s

    def same(self):
        for got, want in zip((self.cache.k, self.cache.v), self.codes):
            np.testing.assert_array_equal(f64(got), want)
        for got, want in zip((self.cache.k_scale, self.cache.v_scale), self.scales):
            np.testing.assert_array_equal(f64(got), want)

    def attention(self, q, starts, lengths, table, window=0, scale=None, bad=()):
        """(out, lse, A, tolerance of out, of lse) for f64 q [rows, heads, d]."""
        rows, heads, d = q.shape
        scale = d ** -0.5 if scale is None else scale
        out, lse = np.zeros(q.shape), np.full((rows, heads), -np.inf)
        A, ds, n = np.zeros(q.shape), np.zeros((rows, heads)), np.zeros(rows)
        floor = np.zeros(q.shape)
        for i, total in enumerate(lengths):
            m = starts[i + 1] - starts[i]
            if m <= 0 or total <= 0:
                continue
            pages = table[i][:-(-total // self.page)]
            held = np.repeat([p not in bad for p in pages], self.page)[:total]
            pages = [0 if p in bad else p for p in pages]
            k, v = (np.nan_to_num(c[pages] * s[pages][:, :, None, None]).transpose(
                0, 2, 1, 3).reshape(-1, self.hkv, d)[:total]
                for c, s in zip(self.codes, self.scales))
            vs = np.repeat(self.scales[1][pages], self.page, 0)[:total]
            j = np.arange(total)
            for t in range(m):
                row, p = starts[i] + t, total - m + t
                see = held & (j <= p) & ((j > p - window) if window else True)
                if not see.any():
                    continue
                n[row] = see.sum()
                for h in range(heads):
                    g = h // (heads // self.hkv)
                    s = scale * (k[see, g] @ q[row, h])
                    top = s.max()
                    e = np.exp(s - top)
                    w = e / e.sum()
                    out[row, h] = w @ v[see, g]
                    lse[row, h] = top + math.log(e.sum())
                    A[row, h] = w @ np.abs(v[see, g])
                    floor[row, h] = 2.0 ** -35 * (w * vs[see, g]).max() * (
                        np.abs(v[see, g]) / vs[see, g][:, None]).sum(0)
                    ds[row, h] = abs(scale) * (
                        (np.abs(k[see, g]) @ np.abs(q[row, h])).max() * (d / 16 + 16) * 2.0 ** -23
                        + np.abs(q[row, h]).max() * np.abs(k[see, g]).sum(1).max() * 2.0 ** -22)
        acc = (n[:, None] / 16 + 16) * 2.0 ** -23
        rel = 2 * ds + 2.0 ** -21 + acc
        # what the output may be off by, but for its rounding and p's as f16
        return out, lse, A, A * rel[..., None] + floor, ds + acc + 2.0 ** -21

    def attention_by_head(self, q, starts, lengths, table, window=0, scale=None, bad=()):
        """attention(), a sequence's rows of one k/v head at a time, for many rows."""
        rows, heads, d = q.shape
        scale = d ** -0.5 if scale is None else scale
        group = heads // self.hkv
        out, lse = np.zeros(q.shape), np.full((rows, heads), -np.inf)
        A, floor, ds, n = np.zeros(q.shape), np.zeros(q.shape), np.zeros((rows, heads)), np.zeros(rows)
        for i, total in enumerate(lengths):
            m = starts[i + 1] - starts[i]
            if m <= 0 or total <= 0:
                continue
            at = slice(starts[i], starts[i + 1])
            pages = table[i][:-(-total // self.page)]
            held = np.repeat([p not in bad for p in pages], self.page)[:total]
            pages = np.array([0 if p in bad else p for p in pages])
            p, j = total - m + np.arange(m)[:, None], np.arange(total)
            see = held & (j <= p) & ((j > p - window) if window else True)
            n[at] = see.sum(1)
            for g in range(self.hkv):
                vs = np.repeat(self.scales[1][pages, g], self.page)[:total]
                c = self.codes[1][pages, g].reshape(-1, d)[:total]
                k = (self.codes[0][pages, g] * self.scales[0][pages, g][:, None, None]).reshape(
                    -1, d)[:total]
                k, c, vs = np.nan_to_num(k), np.nan_to_num(c), np.nan_to_num(vs)
                for h in range(g * group, (g + 1) * group):
                    x = q[at, h]
                    s = np.where(see, scale * (x @ k.T), -np.inf)
                    top = np.where(see.any(1), s.max(1), 0.0)[:, None]
                    e = np.exp(s - top)
                    z = e.sum(1, keepdims=True)
                    w = e / np.where(z == 0, 1, z)
                    out[at, h] = (w * vs) @ c
                    with np.errstate(divide="ignore"):
                        lse[at, h] = (top + np.log(z))[:, 0]
                    A[at, h] = (w * vs) @ np.abs(c)
                    floor[at, h] = 2.0 ** -35 * (w * vs).max(1)[:, None] * (see @ np.abs(c))
                    ds[at, h] = abs(scale) * (
                        np.where(see, np.abs(x) @ np.abs(k).T, 0).max(1) * (d / 16 + 16) * 2.0 ** -23
                        + np.abs(x).max(1) * np.where(see, np.abs(k).sum(1), 0).max(1) * 2.0 ** -22)
        acc = (n[:, None] / 16 + 16) * 2.0 ** -23
        rel = 2 * ds + 2.0 ** -21 + acc
        return out, lse, A, A * rel[..., None] + floor, ds + acc + 2.0 ** -21


def f64(t):
    import torch
    t = t.detach()
    if t.dtype == torch.float8_e4m3fn:
        t = t.float()
    return t.double().cpu().numpy()


def i32(a, dev):
    import torch
    return torch.tensor(np.asarray(a), dtype=torch.int32, device=dev)


def tables(rng, lengths, page, n_pages, width=None):
    """Pages of each sequence, at random; unused places name no page."""
    order = rng.permutation(n_pages)
    width = width or max(1, max(-(-t // page) for t in lengths))
    table = np.full((len(lengths), width), -5)
    at = 0
    for i, t in enumerate(lengths):
        n = -(-t // page)
        table[i, :n] = order[at:at + n]
        at += n
    return table


def rows_of(rng, n, heads, d, bf16, dev, pad=0, spread=True):
    import torch
    x = rng.standard_normal((n, heads * d + pad)).astype(np.float32)
    if spread:
        x *= np.exp2(rng.integers(-3, 4, (n, 1))).astype(np.float32)
    t = torch.from_numpy(x).to(torch.bfloat16 if bf16 else torch.float32).to(dev)
    return t[:, :heads * d].unflatten(1, (heads, d))


def starts_of(counts):
    return np.concatenate([[0], np.cumsum(counts)]).astype(int)


def fill(m, lengths, table, bf16=True, spread=True):
    """The sequences' tokens appended in one call."""
    st = starts_of(lengths)
    k, v = (rows_of(m.rng, int(st[-1]), m.hkv, m.d, bf16, m.dev, spread=spread) for _ in range(2))
    T.kv8_append(m.cache, k, v, i32(st, m.dev), i32(lengths, m.dev), i32(table, m.dev))
    m.append([f64(k), f64(v)], st, lengths, table)


# ------------------------------------------------------------------ append
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("page,hkv,d", [(16, 1, 16), (32, 3, 80), (64, 8, 128), (128, 2, 256),
                                        (64, 4, 64)])
def test_append_prompts_then_tokens(dev, fmt, bf16, page, hkv, d):
    """Prompts, then tokens one at a time and a few at once, every code equal;
    pages' scales grow on the way and earlier codes are rescaled."""
    m = Model(dev, fmt, page, hkv, d, 24)
    lengths = np.array([page, 1, 3 * page - 1, 2 * page + 5, 0])
    table = tables(m.rng, lengths + page, page, 24)
    fill(m, lengths, table, bf16)
    m.same()
    for counts in ([1, 1, 1, 1, 1], [0, 5, 3, 0, page - 1], [2, 0, page // 2, 1, 1]):
        counts = np.array(counts)
        counts = np.minimum(counts, table.shape[1] * page - lengths)
        lengths = lengths + counts
        if any((table[i][-(-t // page) - 1] < 0) for i, t in enumerate(lengths) if t):
            break
        st = starts_of(counts)
        k, v = (rows_of(m.rng, int(st[-1]), hkv, d, bf16, dev, pad=3) for _ in range(2))
        T.kv8_append(m.cache, k, v, i32(st, dev), i32(lengths, dev), i32(table, dev))
        m.append([f64(k), f64(v)], st, lengths, table)
        m.same()
    assert T.check_status() == (0, 0)


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_append_scale_borders(dev, fmt):
    """amax at, just under and just over MAX s; zeros; the smallest and the
    largest values; ties."""
    import torch
    most = MOST[fmt]
    up = float(np.nextafter(np.float32(most), np.float32(np.inf)))
    down = float(np.nextafter(np.float32(most), np.float32(0)))
    peaks = [most, up, down, 0.0, 1e-38, 1e-45, 2.0 ** -100 * most, 2.0 ** -101 * most, 3.4e38,
             2.0 ** 127, most * 2.0 ** -20, up * 2.0 ** 30]
    m = Model(dev, fmt, 16, 1, 16, len(peaks))
    x = np.zeros((len(peaks), 1, 16), np.float32)
    for i, p in enumerate(peaks):
        x[i, 0] = np.float32(p) * ((np.arange(16) - 8.0) / 8.0).astype(np.float32)
        x[i, 0, 9:12] = np.float32(p / (2 * most)) * np.array([1, 3, -5], np.float32)
    lengths = np.ones(len(peaks), int)
    table = np.arange(len(peaks))[:, None]
    t = torch.from_numpy(x).to(dev)
    T.kv8_append(m.cache, t, -t, i32(starts_of(lengths), dev), i32(lengths, dev), i32(table, dev))
    m.append([x.astype(np.float64), -x.astype(np.float64)], starts_of(lengths), lengths, table)
    m.same()
    assert T.check_status() == (0, 0)


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_append_nonfinite_is_flagged(dev, fmt):
    import torch
    m = Model(dev, fmt, 16, 2, 32, 2)
    x = m.rng.standard_normal((3, 2, 32)).astype(np.float32)
    x[0, 0, 3], x[1, 0, 4], x[2, 1, 5] = np.nan, np.inf, -np.inf
    t = torch.from_numpy(x).to(dev)
    T.kv8_append(m.cache, t, t, i32([0, 3], dev), i32([3], dev), i32([[1]], dev))
    m.append([x.astype(np.float64)] * 2, [0, 3], [3], [[1]])
    m.same()
    assert T.check_status() == (8, T.FLAG_NONFINITE)


def test_append_padding_and_bounds(dev):
    """Rows before position 0, rows behind the last sequence, pages out of
    range, a table that is too short, and malformed row_start values."""
    import torch
    m = Model(dev, "int8", 16, 2, 64, 6)
    k, v = (rows_of(m.rng, 40, 2, 64, True, dev) for _ in range(2))
    # sequence 0: three rows, one token; sequence 1: none; sequence 2: idle slot
    st, lengths, table = [0, 3, 3, 4], [1, 0, 0], [[2], [0], [1]]
    T.kv8_append(m.cache, k, v, i32(st, dev), i32(lengths, dev), i32(table, dev))
    m.append([f64(k), f64(v)], st, lengths, table)
    m.same()
    assert T.check_status() == (0, 0)
    # a bad page between two good ones
    st, lengths, table = [0, 40], [40], [[3, 6, 4]]
    T.kv8_append(m.cache, k, v, i32(st, dev), i32(lengths, dev), i32(table, dev))
    x = [f64(k), f64(v)]
    m.append([a[:16] for a in x], [0, 16], [16], [[3]])
    m.append([a[32:] for a in x], [0, 8], [8], [[4]])
    m.same()
    assert T.check_status() == (8, T.FLAG_PAGE_RANGE)
    # 40 tokens, room for 32
    T.kv8_append(m.cache, k, v, i32([0, 40], dev), i32([40], dev), i32([[0, 5]], dev))
    m.append([a[:32] for a in x], [0, 32], [32], [[0, 5]])
    m.same()
    assert T.check_status() == (8, T.FLAG_POSITION_RANGE)
    # row_start outside the rows: clamped
    T.kv8_append(m.cache, k, v, i32([-7, 2 ** 30], dev), i32([40], dev), i32([[0, 5, 1]], dev))
    m.append(x, [0, 40], [40], [[0, 5, 1]])
    m.same()
    T.kv8_append(m.cache, k, v, i32([9, 3], dev), i32([40], dev), i32([[0, 5, 1]], dev))
    m.same()
    assert T.check_status() == (0, 0)
    torch.cuda.synchronize()


# --------------------------------------------------------------- attention
def limit(y, A, lim, bf16):
    return lim + (A * 2.0 ** -11 + 2.0 ** -8 * np.abs(y) if bf16 else 2.0 ** -24 * np.abs(y)) + 1e-37


def attend(m, counts, lengths, table, heads, bf16, window=0, scale=None, q=None, bad=(), extra=0,
           pad=0, by_head=False, **kw):
    import torch
    st = starts_of(counts)
    if q is None:
        q = rows_of(m.rng, int(st[-1]) + extra, heads, m.d, bf16, m.dev, pad=pad, spread=False)
    out = torch.full(q.shape, 7.0, dtype=q.dtype, device=m.dev)
    lse = torch.full(q.shape[:2], 7.0, device=m.dev)
    T.kv8_attention(m.cache, q, i32(st, m.dev), i32(lengths, m.dev), i32(table, m.dev),
                    window=window, scale=scale, out=out, lse=lse, **kw)
    f = m.attention_by_head if by_head else m.attention
    y, z, A, lim, tol = f(f64(q), st, lengths, table, window, scale, bad)
    n = int(st[-1])
    o, ls = f64(out)[:n], f64(lse)[:n]
    lim = limit(y, A, lim, bf16)[:n]
    off = np.abs(o - y[:n])
    assert (off <= lim).all(), ("out", (off / lim).max(), np.argwhere(off > lim)[:5])
    np.testing.assert_array_equal(np.isneginf(ls), np.isneginf(z[:n]))
    fin = np.isfinite(z[:n])
    off = np.abs(ls[fin] - z[:n][fin])
    assert (off <= (tol[:n] + 2.0 ** -23 * np.abs(z[:n]))[fin]).all(), ("lse", off.max())
    if extra:  # rows of nobody
        assert bool((out[n:] == 7.0).all()) and bool((lse[n:] == 7.0).all())
    return out, lse


SHAPES = [  # page, heads, kv heads, d
    (16, 4, 4, 64), (64, 64, 8, 128), (32, 7, 1, 80), (128, 2, 2, 256), (64, 12, 4, 96),
    (16, 3, 3, 16), (64, 40, 2, 128), (64, 6, 2, 208)]


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("page,heads,hkv,d", SHAPES)
def test_single_tokens(dev, fmt, bf16, page, heads, hkv, d):
    """One query per sequence, lengths from none to many pages."""
    lengths = [1, 2, page - 1, page, page + 1, 0, 3 * page + 7, 517, 16, 17]
    m = Model(dev, fmt, page, hkv, d, sum(-(-t // page) for t in lengths) + 1)
    table = tables(m.rng, lengths, page, len(m.scales[0]))
    fill(m, lengths, table)
    attend(m, [1] * len(lengths), lengths, table, heads, bf16, extra=2)
    assert T.check_status() == (0, 0)


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("window", [0, 1, 37, 1000])
@pytest.mark.parametrize("page,heads,hkv,d", [(16, 8, 2, 64), (64, 8, 1, 128), (32, 2, 2, 112)])
def test_ragged_queries(dev, fmt, bf16, page, heads, hkv, d, window):
    """None to many queries per sequence, more queries than tokens among them."""
    counts = [1, 0, 5, 17, 70, 33, 4]
    lengths = [300, 40, 5, 120, 70, 333, 2]
    m = Model(dev, fmt, page, hkv, d, sum(-(-t // page) for t in lengths), seed=window)
    table = tables(m.rng, lengths, page, len(m.scales[0]))
    fill(m, lengths, table)
    attend(m, counts, lengths, table, heads, bf16, window=window, pad=5, extra=3)
    assert T.check_status() == (0, 0)


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("window", [0, 3000])
def test_long_sequences(dev, fmt, bf16, window):
    """Rows whose keys are split over the device and joined again."""
    lengths = [9001, 20, 4097]
    m = Model(dev, fmt, 64, 2, 128, 300)
    table = tables(m.rng, lengths, 64, 300, width=200)
    fill(m, lengths, table, spread=False)
    attend(m, [1, 1, 1], lengths, table, 8, bf16, window=window)
    attend(m, [3, 1, 20], lengths, table, 4, bf16, window=window)
    assert T.check_status() == (0, 0)


CHUNKS = [  # page, heads, kv heads, d, rows and lengths of the sequences, window
    (64, 32, 8, 128, [360, 1, 257, 64], [811, 500, 257, 3000], 0),
    (16, 32, 2, 64, [130, 490, 5], [130, 1000, 20], 0),
    (128, 28, 4, 80, [700], [1500], 100),
    (32, 64, 1, 112, [256, 50], [300, 40], 0),
    (64, 24, 8, 128, [900, 3], [2500, 129], 700),
    (16, 16, 16, 16, [1300], [1411], 0)]


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("page,heads,hkv,d,counts,lengths,window", CHUNKS)
def test_chunks_of_prompts(dev, fmt, page, heads, hkv, d, counts, lengths, window):
    """Calls with many rows a sequence, beside ones with few or more than tokens."""
    m = Model(dev, fmt, page, hkv, d, sum(-(-t // page) for t in lengths) + 1)
    table = tables(m.rng, lengths, page, len(m.scales[0]))
    fill(m, lengths, table)
    attend(m, counts, lengths, table, heads, True, window=window, extra=3, pad=8, by_head=True)
    assert T.check_status() == (0, 0)


def test_chunk_scales_strides_and_bounds(dev):
    """Many rows: a zero and a negative scale, unaligned rows, pages of very
    different scales, a page out of range, a NaN row, a sequence past its bounds."""
    import torch
    lengths, counts, heads = [500, 300], [400, 250], 32
    m = Model(dev, "int8", 64, 8, 128, 14)
    table = tables(m.rng, lengths, 64, 14)
    fill(m, lengths, table)
    for scale in (0.0, -0.3, 0.7):
        attend(m, counts, lengths, table, heads, True, scale=scale, by_head=True, pad=3)
    broken = table.copy()
    broken[0, 2], broken[1, 1] = 14, -1
    attend(m, counts, lengths, broken, heads, True, bad=(14, -1), by_head=True)
    attend(m, counts, lengths, broken, heads, True, bad=(14, -1), scale=0.0, by_head=True)
    assert T.check_status() == (8, T.FLAG_PAGE_RANGE)
    st, ln, tb = i32(starts_of(counts), dev), i32(lengths, dev), i32(table, dev)
    q = rows_of(m.rng, sum(counts), heads, 128, True, dev, spread=False).clone()
    want = T.kv8_attention(m.cache, q, st, ln, tb)
    q[77, 5, 100] = float("nan")
    got = T.kv8_attention(m.cache, q, st, ln, tb)
    assert bool(torch.isnan(got[77, 5]).all())
    got[77, 5] = want[77, 5]
    assert torch.equal(got, want)
    out, lse = T.kv8_attention(m.cache, q, st, ln, tb, max_len=499, return_lse=True)
    assert bool((out[:400] == 0).all()) and bool(torch.isneginf(lse[:400]).all())
    assert torch.equal(out[400:], want[400:])
    assert T.check_status() == (8, T.FLAG_POSITION_RANGE)
    # pages 2^30 apart
    for p in range(14):
        e = [0, -30, 12, -5][p % 4]
        m.cache.v_scale[p] *= 2.0 ** e
        m.scales[1][p] *= 2.0 ** e
    attend(m, counts, lengths, table, heads, True, by_head=True)


@pytest.mark.parametrize("bf16", [False, True])
def test_peaked_tiny_and_huge_scores(dev, bf16):
    """One key that takes all the weight, scores far apart, a zero and a
    negative scale, q of very small and very large values."""
    import torch
    lengths = [200, 90]
    m = Model(dev, "int8", 64, 1, 64, 6)
    table = tables(m.rng, lengths, 64, 6)
    fill(m, lengths, table)
    for factor in (50.0, 1e-30, 0.0):
        q = rows_of(m.rng, 2, 4, 64, bf16, dev, spread=False) * factor
        attend(m, [1, 1], lengths, table, 4, bf16, q=q)
    for scale in (0.0, -0.3, 2.0):
        attend(m, [1, 1], lengths, table, 4, bf16, scale=scale)
    q = rows_of(m.rng, 2, 4, 64, bf16, dev, spread=False)
    q[:, :, 5] *= 1e-6  # elements far below their row's largest
    attend(m, [1, 1], lengths, table, 4, bf16, q=q)
    big = torch.full((2, 4, 64), 1e30, device=dev).to(q.dtype) * torch.sign(q)
    attend(m, [1, 1], lengths, table, 4, bf16, q=big, scale=1e-31)


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_pages_of_very_different_scales(dev, fmt):
    """Values of pages 2^60 apart: each page's scale is its own."""
    import torch
    m = Model(dev, fmt, 16, 1, 32, 8)
    table = [[3, 1, 7, 0, 5]]
    x = m.rng.standard_normal((2, 70, 1, 32)).astype(np.float32)
    for p, e in enumerate([0, -60, 30, -30, 0]):
        x[1, 16 * p:16 * p + 16] *= np.float32(2.0 ** e)
        x[0, 16 * p:16 * p + 16] *= np.float32(2.0 ** (e // 30))
    k, v = (torch.from_numpy(a).to(dev) for a in x)
    T.kv8_append(m.cache, k, v, i32([0, 70], dev), i32([70], dev), i32(table, dev))
    m.append([a.astype(np.float64) for a in x], [0, 70], [70], table)
    m.same()
    for counts in ([1], [40]):
        attend(m, counts, [70], table, 2, False)
    for n in (16, 32):  # the small pages alone
        attend(m, [1], [n], table, 2, False, window=16)


def test_bounds_are_flagged(dev):
    import torch
    lengths = [100, 60]
    m = Model(dev, "int8", 16, 2, 64, 12)
    table = tables(m.rng, lengths, 16, 12)
    fill(m, lengths, table)
    # a page out of range: its keys are not attended
    broken = table.copy()
    broken[0, 2], broken[1, 1] = 12, -1
    attend(m, [1, 2], lengths, broken, 4, True, bad=(12, -1))
    assert T.check_status() == (8, T.FLAG_PAGE_RANGE)
    # beyond max_len, max_q and the table: as without keys
    q = rows_of(m.rng, 5, 4, 64, True, dev)
    for kw, n in ((dict(max_len=99), 100), (dict(max_q=2), 100), ({}, 113)):
        out, lse = T.kv8_attention(m.cache, q, i32([0, 3, 5], dev), i32([n, 60], dev),
                                   i32(table, dev), return_lse=True, **kw)
        assert bool((out[:3] == 0).all()) and bool(torch.isneginf(lse[:3]).all())
        assert bool((out[3:] != 0).any()) and bool(torch.isfinite(lse[3:]).all())
        assert T.check_status() == (8, T.FLAG_POSITION_RANGE)


def test_nan_query_stays_its_own(dev):
    import torch
    m = Model(dev, "e4m3", 16, 1, 64, 4)
    table = tables(m.rng, [50], 16, 4)
    fill(m, [50], table)
    q = rows_of(m.rng, 3, 2, 64, True, dev)
    want = T.kv8_attention(m.cache, q, i32([0, 3], dev), i32([50], dev), i32(table, dev))
    q = q.clone()
    q[1, 0, 7] = float("nan")
    got = T.kv8_attention(m.cache, q, i32([0, 3], dev), i32([50], dev), i32(table, dev))
    assert bool(torch.isnan(got[1, 0]).all())
    keep = torch.ones(3, 2, dtype=torch.bool, device=dev)
    keep[1, 0] = False
    assert torch.equal(got[keep], want[keep])


def test_large_page_numbers(dev):
    """Codes more than 2^31 bytes into the cache."""
    n, page, d = 9000, 128, 256
    m = Model.__new__(Model)
    import torch
    m.fmt, m.page, m.hkv, m.d, m.dev = "int8", page, 8, d, dev
    m.rng = np.random.default_rng(3)
    m.cache = T.Kv8Cache.empty(n, 8, page, d, torch.int8)
    used = [8998, 8191, 8999]
    m.codes = [np.zeros((3, 8, page, d)) for _ in range(2)]
    m.scales = [np.zeros((3, 8)) for _ in range(2)]
    lengths = [300]
    st = starts_of(lengths)
    k, v = (rows_of(m.rng, 300, 8, d, True, dev) for _ in range(2))
    T.kv8_append(m.cache, k, v, i32(st, dev), i32(lengths, dev), i32([used], dev))
    m.append([f64(k), f64(v)], st, lengths, [[0, 1, 2]])
    for got, want in zip((m.cache.k, m.cache.v), m.codes):
        np.testing.assert_array_equal(f64(got[used]), want)
    q = rows_of(m.rng, 1, 8, d, True, dev)
    out = T.kv8_attention(m.cache, q, i32([0, 1], dev), i32(lengths, dev), i32([used], dev))
    y, _, A, lim, _ = m.attention(f64(q), [0, 1], lengths, [[0, 1, 2]])
    assert (np.abs(f64(out) - y) <= limit(y, A, lim, True)).all()


# ---------------------------------------------------------------- together
def test_decode_steps_from_a_graph(dev):
    """A prompt, then decode steps as one captured graph: head norms with
    rotary positions, append, attention; lengths and positions advance on the
    device."""
    import torch
    heads, hkv, d, page, seqs = 8, 2, 64, 16, 3
    m = Model(dev, "int8", page, hkv, d, 40)
    lengths = np.array([30, 5, 16])
    table = tables(m.rng, lengths + 20, page, 40)
    fill(m, lengths, table)
    qkv = torch.empty(seqs, heads + 2 * hkv, d, dtype=torch.bfloat16, device=dev)
    q, k, v = qkv[:, :heads], qkv[:, heads:heads + hkv], qkv[:, heads + hkv:]
    w = torch.ones(d, dtype=torch.bfloat16, device=dev)
    fr = T.rotary_freqs(d, 1e4)
    start, length = i32(range(seqs + 1), dev), i32(lengths, dev)
    pos, tab = i32(lengths - 1, dev), i32(table, dev)
    qr, kr = torch.empty_like(q), torch.empty_like(k)
    out = torch.empty_like(qr)
    ws = torch.empty(64 << 20, dtype=torch.uint8, device=dev)

    def step():
        length.add_(1)
        pos.add_(1)
        T.qk_norm_rotary(q, k, w, w, 1e-6, pos, fr, q_out=qr, k_out=kr)
        T.kv8_append(m.cache, kr, v, start, length, tab)
        T.kv8_attention(m.cache, qr, start, length, tab, max_q=1, out=out, workspace=ws)

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for n in range(20):
        qkv.copy_(torch.from_numpy(m.rng.standard_normal(qkv.shape).astype(np.float32)))
        graph.replay()
        lengths = lengths + 1
        m.append([f64(kr), f64(v)], range(seqs + 1), lengths, table)
        y, _, A, lim, _ = m.attention(f64(qr), range(seqs + 1), lengths, table)
        assert (np.abs(f64(out) - y) <= limit(y, A, lim, True)).all()
    m.same()
    assert T.check_status() == (0, 0)


def test_two_streams_and_repeats(dev):
    """Calls at once on two streams, each with its own scratch, and the same
    call again: the same bits."""
    import torch
    lengths = [5000, 3000]
    m = Model(dev, "e4m3", 64, 2, 128, 130)
    table = tables(m.rng, lengths, 64, 130)
    fill(m, lengths, table)
    q = [rows_of(m.rng, 2, 16, 128, True, dev) for _ in range(2)]
    args = (i32([0, 1, 2], dev), i32(lengths, dev), i32(table, dev))
    want = [T.kv8_attention(m.cache, x, *args) for x in q]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            got[i].append(T.kv8_attention(m.cache, q[i], *args, stream=s.cuda_stream))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(want[i], g) for g in got[i])


def test_python_refusals(dev):
    import torch
    m = Model(dev, "int8", 16, 2, 64, 4)
    q = rows_of(m.rng, 2, 4, 64, True, dev)
    k = rows_of(m.rng, 2, 2, 64, True, dev)
    st, ln, tb = i32([0, 1, 2], dev), i32([1, 1], dev), i32([[0], [1]], dev)
    with pytest.raises(TypeError):
        T.kv8_append(m.cache, k, k, st.long(), ln, tb)
    with pytest.raises(TypeError):
        T.kv8_append(m.cache, k, k.float(), st, ln, tb)
    with pytest.raises(ValueError):
        T.kv8_append(m.cache, q, q, st, ln, tb)
    with pytest.raises(ValueError):
        T.kv8_append(m.cache, k, k, st[:2], ln, tb)
    with pytest.raises(ValueError):
        T.kv8_attention(m.cache, q[:, :, :32], st, ln, tb)
    with pytest.raises(T.TbError):
        T.kv8_attention(m.cache, q[:, :3], st, ln, tb)
    with pytest.raises(T.TbError):
        T.kv8_attention(m.cache, q, st, ln, tb, out=q)
    with pytest.raises(TypeError):
        T.kv8_attention(m.cache, q.half(), st, ln, tb)
    with pytest.raises(TypeError):
        T.Kv8Cache(m.cache.k.view(torch.uint8), m.cache.v, m.cache.k_scale, m.cache.v_scale)


# ------------------------------------------------ calls at the edges of the rules
def test_rows_before_the_first_sequence(dev):
    """row_start[0] > 0: rows of nobody in front, and pages of the sequence that
    the call does not touch, given back, with no scale or of no number."""
    m = Model(dev, "int8", 16, 2, 64, 8)
    for t, s in zip((m.cache.k_scale, m.cache.v_scale), m.scales):
        t.fill_(0.0)
        s[:] = 0.0
    k, v = (rows_of(m.rng, 70, 2, 64, True, dev) for _ in range(2))
    x = [f64(k), f64(v)]
    for table in ([[1, 2, 3, 4, 5, 6, 7]], [[-1, -1, 9, -1, -1, 6, 7]]):
        st, lengths = [40, 70], [110]  # positions 80 .. 109, in its last two pages
        T.kv8_append(m.cache, k, v, i32(st, dev), i32(lengths, dev), i32(table, dev))
        m.append(x, st, lengths, table)
        m.same()
        assert T.check_status() == (0, 0)
    q = rows_of(m.rng, 70, 4, 64, True, dev)
    out, lse = T.kv8_attention(m.cache, q, i32([40, 70], dev), i32([110], dev), i32(table, dev),
                               window=3, out=q.new_full(q.shape, 7.0), return_lse=True)
    y, z, A, lim, _ = m.attention(f64(q), [40, 70], [110], table, window=3, bad=(-1, 9))
    assert (np.abs(f64(out) - y) <= limit(y, A, lim, True))[42:].all()
    assert bool((out[:40] == 7.0).all())
    assert T.check_status()[1] in (0, T.FLAG_PAGE_RANGE)  # of rows 40 and 41


@pytest.mark.parametrize("n", [129, 1500])
def test_many_sequences(dev, n):
    """More sequences than threads of a CTA and than 32 times 32."""
    m = Model(dev, "e4m3", 16, 1, 32, 3 * n)
    lengths = m.rng.integers(0, 41, n)
    table = tables(m.rng, lengths + 3, 16, 3 * n)
    fill(m, lengths, table)
    m.same()
    counts = m.rng.integers(0, 4, n)
    lengths = lengths + counts
    st = starts_of(counts)
    k, v = (rows_of(m.rng, int(st[-1]), 1, 32, True, dev) for _ in range(2))
    T.kv8_append(m.cache, k, v, i32(st, dev), i32(lengths, dev), i32(table, dev))
    m.append([f64(k), f64(v)], st, lengths, table)
    m.same()
    attend(m, counts, lengths, table, 2, True, extra=1)
    attend(m, counts, lengths, table, 2, False, max_q=3, max_len=48)
    assert T.check_status() == (0, 0)


@pytest.mark.parametrize("heads,hkv,counts,lengths", [(4, 2, [9, 3], [5, 60]),
                                                     (32, 8, [700, 20], [300, 60])])
def test_windows_beyond_every_length(dev, heads, hkv, counts, lengths):
    """The widest windows are none, for rows before position 0 beside others too."""
    import torch
    m = Model(dev, "int8", 16, hkv, 64, 30)
    table = tables(m.rng, lengths, 16, 30)
    fill(m, lengths, table)
    q = rows_of(m.rng, sum(counts), heads, 64, True, dev, spread=False)
    want = attend(m, counts, lengths, table, heads, True, q=q, by_head=True)
    for window in (2 ** 31 - 1, 2 ** 31 - 4, 2 ** 40 + 7, max(lengths)):
        got = attend(m, counts, lengths, table, heads, True, q=q, window=window, by_head=True)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert T.check_status() == (0, 0)


def test_chunk_rows_past_the_bound(dev):
    """A sequence with more rows than max_q: all its rows are as without keys."""
    import torch
    counts, lengths, heads = [700, 100], [720, 100], 32
    m = Model(dev, "e4m3", 64, 8, 128, 16)
    table = tables(m.rng, lengths, 64, 16)
    fill(m, lengths, table)
    q = rows_of(m.rng, 800, heads, 128, True, dev, spread=False)
    args = (i32(starts_of(counts), dev), i32(lengths, dev), i32(table, dev))
    want = T.kv8_attention(m.cache, q, *args)
    out, lse = torch.full_like(want, 7.0), torch.full((800, heads), 7.0, device=dev)
    T.kv8_attention(m.cache, q, *args, max_q=250, out=out, lse=lse)
    assert bool((out[:700] == 0).all()) and bool(torch.isneginf(lse[:700]).all())
    assert torch.equal(out[700:], want[700:]) and bool(torch.isfinite(lse[700:]).all())
    assert T.check_status() == (8, T.FLAG_POSITION_RANGE)


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("heads,hkv,counts", [(4, 2, [40, 1]), (32, 8, [600, 30])])
def test_values_of_zero_beside_huge_ones(dev, fmt, heads, hkv, counts):
    """Pages of zero values, at the smallest scale, keep their place in the sum."""
    import torch
    lengths = [620, 90]
    m = Model(dev, fmt, 32, hkv, 64, 24)
    table = tables(m.rng, lengths, 32, 24)
    st = starts_of(lengths)
    k, v = (rows_of(m.rng, 710, hkv, 64, False, dev, spread=False) for _ in range(2))
    v = v * 2.0 ** 100
    zero = torch.arange(710, device=dev) // 32 % 3 != 1
    v[zero] = 0.0
    T.kv8_append(m.cache, k, v, i32(st, dev), i32(lengths, dev), i32(table, dev))
    m.append([f64(k), f64(v)], st, lengths, table)
    m.same()
    attend(m, counts, lengths, table, heads, True, by_head=True)
    attend(m, counts, lengths, table, heads, False, by_head=True)
    assert T.check_status() == (0, 0)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_wide_heads_over_long_sequences(dev, fmt, bf16):
    """Heads of 256 and of 208, split over the device and joined."""
    for d, page in ((256, 128), (208, 16)):
        lengths = [4001, 700]
        m = Model(dev, fmt, page, 1, d, 320)
        table = tables(m.rng, lengths, page, 320)
        fill(m, lengths, table, spread=False)
        attend(m, [1, 1], lengths, table, 3, bf16)
        attend(m, [9, 2], lengths, table, 3, bf16, window=2500)
    assert T.check_status() == (0, 0)


@pytest.mark.parametrize("heads,hkv,d,counts,lengths", [
    (8, 2, 128, [1, 1, 3], [5000, 30, 700]), (32, 8, 64, [600, 30, 1], [620, 50, 90])])
def test_unaligned_rows_and_strided_tables(dev, heads, hkv, d, counts, lengths):
    """q and out rows of any start and stride, a page table that is part of a wider
    one: the bits of the aligned call, and nothing beside them written."""
    import torch
    m = Model(dev, "e4m3", 64, hkv, d, 100)
    table = tables(m.rng, lengths, 64, 100)
    fill(m, lengths, table)
    n = sum(counts)
    q = rows_of(m.rng, n, heads, d, True, dev, spread=False)
    st, ln = i32(starts_of(counts), dev), i32(lengths, dev)
    want, lse = T.kv8_attention(m.cache, q, st, ln, i32(table, dev), return_lse=True)
    wide = torch.full((3, table.shape[1] + 5), -9, dtype=torch.int32, device=dev)
    wide[:, 2:2 + table.shape[1]] = i32(table, dev)
    part = wide[:, 2:2 + table.shape[1]]
    for pad, at in ((1, 1), (8, 3), (8, 8), (3, 0)):
        w = heads * d
        qs = torch.zeros(n * (w + pad) + at, dtype=q.dtype, device=dev)
        os_ = torch.full_like(qs, 7.0)
        view = [torch.as_strided(t, (n, heads, d), (w + pad, d, 1), at) for t in (qs, os_)]
        view[0].copy_(q)
        got, ls = T.kv8_attention(m.cache, view[0], st, ln, part, out=view[1], return_lse=True)
        assert torch.equal(got, want) and torch.equal(ls, lse)
        view[1].fill_(7.0)
        assert bool((os_ == 7.0).all())
    assert T.check_status() == (0, 0)


def test_empty_batches_and_tables(dev):
    import torch
    m = Model(dev, "int8", 16, 2, 64, 4)
    none = i32(np.zeros((2, 0)), dev)
    q, k = (rows_of(m.rng, 3, h, 64, True, dev) for h in (4, 2))
    # rows that are padding, or of nobody, need no page
    T.kv8_append(m.cache, k, k, i32([0, 2, 2], dev), i32([0, 0], dev), none)
    out, lse = T.kv8_attention(m.cache, q, i32([0, 2, 2], dev), i32([0, 0], dev), none,
                               out=torch.full_like(q, 7.0), return_lse=True)
    assert bool((out[:2] == 0).all()) and bool((out[2] == 7.0).all())
    assert bool(torch.isneginf(lse[:2]).all()) and T.check_status() == (0, 0)
    # a token and no table
    T.kv8_append(m.cache, k, k, i32([0, 2, 3], dev), i32([2, 1], dev), none)
    assert T.check_status() == (8, T.FLAG_POSITION_RANGE)
    m.same()
    # no rows, no sequences
    T.kv8_append(m.cache, k[:0], k[:0], i32([0], dev), i32([], dev), none[:0])
    assert T.kv8_attention(m.cache, q[:0], i32([0], dev), i32([], dev), none[:0]).shape[0] == 0
    assert T.check_status() == (0, 0)
    with pytest.raises(T.TbError):  # a cache of no pages
        T.kv8_append(T.Kv8Cache.empty(0, 2, 16, 64, torch.int8), k, k, i32([0, 2, 3], dev),
                     i32([2, 1], dev), i32([[0], [0]], dev))


def test_workspace_refusals(dev):
    import torch
    m = Model(dev, "int8", 64, 2, 64, 100)
    table = tables(m.rng, [6000], 64, 100)
    fill(m, [6000], table)
    q = rows_of(m.rng, 1, 8, 64, True, dev)
    args = (i32([0, 1], dev), i32([6000], dev), i32(table, dev))
    want = T.kv8_attention(m.cache, q, *args)
    ws = torch.empty(64 << 20, dtype=torch.uint8, device=dev)
    assert torch.equal(T.kv8_attention(m.cache, q, *args, workspace=ws), want)
    for bad in (ws[:256], ws[8:]):
        with pytest.raises(T.TbError):
            T.kv8_attention(m.cache, q, *args, workspace=bad)
    with pytest.raises(ValueError):
        T.kv8_attention(m.cache, q, *args, workspace=ws[::2])


@pytest.mark.parametrize("heads,hkv,counts,lengths", [
    (16, 2, [1, 1], [5000, 3000]), (32, 8, [600, 30], [900, 1000])])
def test_graphs_at_once(dev, heads, hkv, counts, lengths):
    """Two captured calls, replayed over and over on two streams beside each other
    and an eager one: each has scratch of its own."""
    import torch
    m = Model(dev, "int8", 64, hkv, 128, 130)
    table = tables(m.rng, lengths, 64, 130)
    fill(m, lengths, table)
    args = (i32(starts_of(counts), dev), i32(lengths, dev), i32(table, dev))
    q = [rows_of(m.rng, sum(counts), heads, 128, True, dev) for _ in range(3)]
    want = [T.kv8_attention(m.cache, x, *args, return_lse=True) for x in q]
    graphs, got, streams = [], [], [torch.cuda.Stream() for _ in range(2)]
    for x in q[:2]:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            got.append(T.kv8_attention(m.cache, x, *args, return_lse=True))
        graphs.append(g)
    torch.cuda.synchronize()
    for _ in range(10):
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        eager = T.kv8_attention(m.cache, q[2], *args, return_lse=True)
    torch.cuda.synchronize()
    for w, g in zip(want, got + [eager]):
        assert torch.equal(w[0], g[0]) and torch.equal(w[1], g[1])
    assert T.check_status() == (0, 0)


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_single_tokens_of_many_heads(dev, fmt):
    """64 heads on one k/v head: enough rows a sequence and sequences for the kernel
    of many rows, a token each, empty sequences among them."""
    m = Model(dev, fmt, 32, 1, 128, 700)
    lengths = m.rng.integers(0, 200, 130)
    lengths[[3, 77, 129]] = 0
    lengths[50] = 513
    table = tables(m.rng, lengths, 32, 700)
    fill(m, lengths, table)
    attend(m, [1] * 130, lengths, table, 64, True, extra=1, by_head=True)
    counts = m.rng.integers(0, 3, 130)
    attend(m, counts, lengths, table, 64, True, window=40, by_head=True)
    assert T.check_status() == (0, 0)


def test_chunk_rows_in_front_and_clamped_starts(dev):
    """Many rows: rows of nobody in front of the first sequence, row_start values
    outside the rows, and the loosest bounds beside the tightest."""
    import torch
    m = Model(dev, "e4m3", 32, 8, 64, 80)
    lengths = [700, 400, 0, 900]
    table = tables(m.rng, lengths, 32, 80)
    fill(m, lengths, table)
    q = rows_of(m.rng, 1300, 32, 64, True, dev, spread=False)
    ln, tb = i32(lengths, dev), i32(table, dev)
    st = np.array([0, 600, 601, 601, 1000])
    want, lse = T.kv8_attention(m.cache, q[300:], i32(st, dev), ln, tb, max_q=600, max_len=900,
                                return_lse=True)
    attend(m, st[1:] - st[:-1], lengths, table, 32, True, q=q[:1000], by_head=True)
    out, ls = torch.full_like(q, 7.0), torch.full((1300, 32), 7.0, device=dev)
    T.kv8_attention(m.cache, q, i32(st + 300, dev), ln, tb, out=out, lse=ls)
    assert torch.equal(out[300:], want) and torch.equal(ls[300:], lse)
    assert bool((out[:300] == 7.0).all()) and bool((ls[:300] == 7.0).all())
    one = T.kv8_attention(m.cache, q, i32([0, 1300], dev), ln[3:], tb[3:])
    out.fill_(7.0)
    T.kv8_attention(m.cache, q, i32([-9, 2 ** 31 - 1, 40], dev), ln[[3, 0]], tb[[3, 0]], out=out)
    assert torch.equal(out, one)
    assert T.check_status() == (0, 0)


FIRST_CALL = """
import sys, torch
sys.path.insert(0, {repo!r})
import perf.operators as M
M.own = True
case = [c for c in M.listed() if c["name"] == {name!r}][0]
state = M.prepare(case, 1)
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    got = M.run(state)
graph.replay()
want = M.run(state)
for a, b in zip(got, want):
    assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
"""


@pytest.mark.parametrize("name", ["attention long", "attention chunk", "qk_norm decode 256"])
def test_first_call_is_captured(dev, name):
    """A process whose first call of the library is captured into a graph."""
    import os
    import subprocess
    import sys
    repo = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    subprocess.run([sys.executable, "-c", FIRST_CALL.format(repo=repo, name=name)], cwd=repo,
                   check=True, timeout=300)


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("page,hkv,d", [(16, 5, 128), (32, 3, 64), (16, 9, 96), (32, 5, 128)])
def test_append_units_that_share_a_cta(dev, fmt, bf16, page, hkv, d):
    """Small pages, whose heads share CTAs: prompts, then more rows, aligned and not,
    one head of them with an infinity and a NaN."""
    m = Model(dev, fmt, page, hkv, d, 40)
    lengths = np.array([5 * page + 3, page - 1, 0, 2 * page])
    table = tables(m.rng, lengths + 3 * page, page, 40)
    fill(m, lengths, table, bf16)
    m.same()
    for pad in (0, 3):
        counts = np.array([page, page + 1, 1, page // 2])
        lengths = lengths + counts
        st = starts_of(counts)
        k, v = (rows_of(m.rng, int(st[-1]), hkv, d, bf16, dev, pad=pad) for _ in range(2))
        k[2, 1, 5], v[3, 2, 6] = float("inf"), float("nan")
        T.kv8_append(m.cache, k, v, i32(st, dev), i32(lengths, dev), i32(table, dev))
        m.append([f64(k), f64(v)], st, lengths, table)
        m.same()
        assert T.check_status() == (8, T.FLAG_NONFINITE)


# ---------------------------------------------------------- in front of a window
def spoil(m, table, keys):
    """Anything in the slots of sequence 0's `keys`: NaN codes of e4m3 (127 and -1 as
    int8 codes), beside scales that stay as they were."""
    import torch
    for c in (m.cache.k, m.cache.v):
        c = c.view(torch.uint8)
        for j in keys:
            c[int(table[0][j // m.page]), :, j % m.page] = 0x7f if j % 2 else 0xff


def front_of_window(dev, fmt, bf16, page, heads, hkv, d, rows, length, window):
    """A sequence whose rows do not see its first keys: with those spoilt, then their
    whole pages given back, the same bits and no flag."""
    import torch
    m = Model(dev, fmt, page, hkv, d, -(-length // page) + 2)
    table = tables(m.rng, [length], page, len(m.scales[0]))
    fill(m, [length], table)
    q = rows_of(m.rng, rows, heads, d, bf16, dev, spread=False)
    kw = dict(window=window, q=q, by_head=True)
    want = attend(m, [rows], [length], table, heads, bf16, **kw)
    first = max(length - rows - window + 1, 0)  # the first key that a row sees
    assert first > page
    spoil(m, table, range(first))
    st, ln = i32([0, rows], dev), i32([length], dev)
    for gone in (-1, len(m.scales[0])):
        got = T.kv8_attention(m.cache, q, st, ln, i32(table, dev), window=window, return_lse=True)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        assert T.check_status() == (0, 0)
        table = table.copy()
        table[0, :first // page] = gone
    # one page more: the first row sees its last key
    table[0, first // page] = gone
    attend(m, [rows], [length], table, heads, bf16, bad=(gone, -1), **kw)
    assert T.check_status() == (8, T.FLAG_PAGE_RANGE)


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("page,heads,hkv,d,rows,length,window", [
    (16, 8, 1, 64, 1, 121, 5),      # a step's first half in front
    (16, 4, 2, 128, 1, 200, 16), (32, 4, 4, 80, 1, 300, 31),
    (16, 3, 1, 256, 1, 222, 13),    # a step of 16 in front
    (64, 3, 1, 208, 2, 333, 40), (128, 2, 2, 128, 5, 400, 77),
    (16, 4, 2, 64, 30, 177, 1),     # blocks of 8 tokens
    (64, 8, 8, 128, 1, 9000, 4500)])  # cut into shares
def test_pages_in_front_of_a_window(dev, fmt, bf16, page, heads, hkv, d, rows, length, window):
    front_of_window(dev, fmt, bf16, page, heads, hkv, d, rows, length, window)


@pytest.mark.parametrize("bf16", [False, True])
def test_keys_after_a_blocks_rows(dev, bf16):
    """What rows of later tokens alone attend: NaN codes there leave the rows of
    earlier blocks as they were."""
    import torch
    m = Model(dev, "e4m3", 32, 1, 64, 6)
    table = tables(m.rng, [150], 32, 6)
    fill(m, [150], table)
    q = rows_of(m.rng, 50, 1, 64, bf16, dev, spread=False)  # blocks of 16 tokens, from 100
    args = (i32([0, 50], dev), i32([150], dev), i32(table, dev))
    want = T.kv8_attention(m.cache, q, *args)
    spoil(m, table, range(116, 150))
    got = T.kv8_attention(m.cache, q, *args)
    assert torch.equal(got[:16], want[:16]) and bool(torch.isnan(got[-1]).any())
    assert T.check_status() == (0, 0)


def test_attended_bad_page_is_flagged(dev):
    """Rows whose window ends in a page of number -1 are flagged and attend the rest;
    rows behind it are not (the calls of test_rows_before_the_first_sequence, apart)."""
    m = Model(dev, "int8", 16, 2, 64, 8)
    table = [[-1, -1, 9, -1, 5, 6, 7]]
    k, v = (rows_of(m.rng, 46, 2, 64, True, dev) for _ in range(2))
    T.kv8_append(m.cache, k, v, i32([0, 46], dev), i32([110], dev), i32(table, dev))
    m.append([f64(k), f64(v)], [0, 46], [110], table)
    broken = [[-1, -1, 9, -1, -1, 6, 7]]
    attend(m, [30], [110], broken, 4, True, window=3, bad=(-1, 9))  # positions 80 ..
    assert T.check_status() == (8, T.FLAG_PAGE_RANGE)
    attend(m, [28], [110], broken, 4, True, window=3, bad=(-1, 9))  # positions 82 ..
    assert T.check_status() == (0, 0)
    attend(m, [1], [110], broken, 4, True, window=3, bad=(-1, 9))
    assert T.check_status() == (0, 0)


CHUNK_WINDOWS = [  # page, heads, kv heads, d, rows, length, window
    (16, 32, 8, 128, 300, 700, 40), (64, 32, 8, 64, 400, 1000, 100),
    (128, 32, 4, 96, 300, 900, 7), (32, 64, 1, 112, 256, 600, 33)]


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("page,heads,hkv,d,rows,length,window", CHUNK_WINDOWS)
def test_chunk_pages_in_front_of_a_window(dev, fmt, page, heads, hkv, d, rows, length, window):
    """The same with many rows, whose steps begin up to 127 keys early."""
    front_of_window(dev, fmt, True, page, heads, hkv, d, rows, length, window)


def test_keys_after_a_chunks_rows(dev):
    import torch
    m = Model(dev, "e4m3", 32, 16, 80, 24)
    table = tables(m.rng, [700], 32, 24)
    fill(m, [700], table)
    q = rows_of(m.rng, 600, 16, 80, True, dev, spread=False)  # blocks of 256 tokens, from 100
    args = (i32([0, 600], dev), i32([700], dev), i32(table, dev))
    want = T.kv8_attention(m.cache, q, *args)
    spoil(m, table, range(356, 700))
    got = T.kv8_attention(m.cache, q, *args)
    assert torch.equal(got[:256], want[:256]) and bool(torch.isnan(got[-1]).any())
    assert T.check_status() == (0, 0)


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("bf16,counts", [(False, [1, 9]), (True, [1, 9]), (True, [300, 80])])
def test_pages_that_nobody_wrote(dev, fmt, bf16, counts):
    """Pages as Kv8Cache.empty leaves them, of scale 0 and codes 0, are keys and values
    of zero: scores of 0, which count, by few rows and by many."""
    lengths, heads = [500, 200], 32
    m = Model(dev, fmt, 32, 8, 128, 24)
    table = tables(m.rng, lengths, 32, 24)
    fill(m, lengths, table, spread=False)
    for page in (table[0, 3], table[0, 4], table[1, 0], table[1, 6]):
        for t, own in zip((m.cache.k, m.cache.v, m.cache.k_scale, m.cache.v_scale),
                          (*m.codes, *m.scales)):
            t[int(page)] = 0
            own[page] = 0.0
    attend(m, counts, lengths, table, heads, bf16, by_head=True)
    attend(m, counts, lengths, table, heads, bf16, by_head=True, window=64)
    assert T.check_status() == (0, 0)


def test_scratch_of_the_threads_stream(dev):
    """Calls on the stream that tb_b200_set_stream chose take their scratch and outputs
    from that stream's pool, where freed memory waits for the call."""
    import torch
    m = Model(dev, "int8", 64, 2, 64, 100)
    table = tables(m.rng, [6000], 64, 100)
    fill(m, [6000], table)
    q = rows_of(m.rng, 1, 8, 64, True, dev)
    args = (i32([0, 1], dev), i32([6000], dev), i32(table, dev))
    want = T.kv8_attention(m.cache, q, *args)
    fr = T.rotary_freqs(64, 1e4)
    pos = i32([7], dev)

    def taken(call, **kw):
        """The streams of the memory that a call takes, on a new stream s, and s."""
        torch.cuda.synchronize()
        torch.cuda.empty_cache()
        s = torch.cuda.Stream()
        before = {x["address"] for x in torch.cuda.memory_snapshot()}
        T.lib().tb_b200_set_stream(s.cuda_stream)
        try:
            got = call(**kw)
        finally:
            T.lib().tb_b200_set_stream(None)
        torch.cuda.synchronize()
        mine = [x["stream"] for x in torch.cuda.memory_snapshot() if x["stream"] == s.cuda_stream]
        other = [x for x in torch.cuda.memory_snapshot()
                 if x["stream"] != s.cuda_stream and x["address"] not in before]
        assert mine and not other
        return got

    out = torch.empty_like(want)
    for kw in ({}, dict(stream=0)):
        taken(lambda **k: T.kv8_attention(m.cache, q, *args, out=out, **k), **kw)
        assert torch.equal(out, want)
        out.zero_()
        got = taken(lambda **k: T.kv8_attention(m.cache, q, *args, return_lse=True, **k), **kw)
        assert torch.equal(got[0], want)
        taken(lambda **k: T.rotary(q, q, pos, fr, **k), **kw)
        taken(lambda **k: T.rotary_freqs(64, 1e4, **k), **kw)
    # a call's own stream comes before the thread's
    s, own = torch.cuda.Stream(), torch.cuda.Stream()
    T.lib().tb_b200_set_stream(s.cuda_stream)
    try:
        got = [T.kv8_attention(m.cache, q, *args, stream=own.cuda_stream)]
        with torch.cuda.stream(own):
            got.append(T.kv8_attention(m.cache, q, *args))
    finally:
        T.lib().tb_b200_set_stream(None)
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got)


def test_counts_past_an_int(dev):
    """Bounds that a C int does not hold are what they say, not their low 32 bits."""
    import torch
    m = Model(dev, "int8", 16, 2, 64, 8)
    table = tables(m.rng, [100], 16, 8)
    fill(m, [100], table)
    q = rows_of(m.rng, 3, 4, 64, True, dev)
    args = (i32([0, 3], dev), i32([100], dev), i32(table, dev))
    want = T.kv8_attention(m.cache, q, *args)
    for n in (2 ** 31 - 1, 2 ** 31, 2 ** 32, 2 ** 32 + 1, 2 ** 63):
        assert torch.equal(T.kv8_attention(m.cache, q, *args, max_q=n), want)
        assert torch.equal(T.kv8_attention(m.cache, q, *args, window=n), want)
        with pytest.raises(T.TbError):  # more than 2^30
            T.kv8_attention(m.cache, q, *args, max_len=n)
    for bad in (-1, -2 ** 31, -2 ** 32, -2 ** 32 + 50, -2 ** 64 + 100):
        for name in ("max_q", "max_len", "window"):
            with pytest.raises(T.TbError):
                T.kv8_attention(m.cache, q, *args, **{name: bad})
        with pytest.raises(T.TbError):
            T.rotary(q, q, i32([0, 1, 2], dev), T.rotary_freqs(64, 1e4), layout=bad)
    with pytest.raises(T.TbError):
        T.rotary(q, q, i32([0, 1, 2], dev), T.rotary_freqs(64, 1e4), layout=2 ** 32)
    assert T.check_status() == (0, 0)
