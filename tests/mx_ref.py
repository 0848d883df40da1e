"""Definitions in 64 bits of the microscaled formats and of filtered sampling (numpy, CPU)."""
import numpy as np

LARGEST = {"e4m3": 448.0, "e2m1": 6.0}
CODES = {"e4m3": [], "e2m1": []}  # value of each code
for _c in range(256):
    e, m = _c >> 3 & 15, _c & 7
    v = m / 8 * 2.0 ** -6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7)
    CODES["e4m3"].append((-v if _c & 128 else v) if _c & 127 != 127 else np.nan)
for _c in range(16):
    v = (0, 0.5, 1, 1.5, 2, 3, 4, 6)[_c & 7]
    CODES["e2m1"].append(-v if _c & 8 else v)
CODES = {k: np.array(v, dtype=np.float64) for k, v in CODES.items()}


def up(n, to):
    return -(-n // to) * to


def scale_places(rows, cols):
    """Byte of each row's block scales, [rows, ceil(cols / 32)]."""
    t = -(-cols // 128)
    r, b = np.arange(rows)[:, None], np.arange(-(-cols // 32))[None]
    return (r // 128 * t + b // 4) * 512 + r % 32 * 16 + r % 128 // 32 * 4 + b % 4


def values(codes, scales, cols, fmt):
    """What codes [rows, pitch] and tiled scales stand for (uint8 arrays), [rows, cols]."""
    rows = codes.shape[0]
    if fmt == "e2m1":
        codes = np.stack([codes & 15, codes >> 4], -1).reshape(rows, -1)
    s = scales[scale_places(rows, cols)].astype(np.int64)
    s = np.where(s == 255, np.nan, np.ldexp(1.0, s - 127))
    return CODES[fmt][codes[:, :cols]] * np.repeat(s, 32, 1)[:, :cols]


def scale_exponents(amax, fmt):
    """The least e >= -127 with amax <= MAX 2^e."""
    m, e = np.frexp(amax / LARGEST[fmt])  # exact next to powers of two: amax is a float32
    return np.maximum(np.where(amax > 0, e - (m == 0.5), -127), -127)


def nearest(v, fmt):
    """v to the format's values, ties to the even code."""
    table = CODES[fmt][:127] if fmt == "e4m3" else CODES[fmt][:8]
    a = np.abs(v)
    hi = np.minimum(np.searchsorted(table, a), len(table) - 1)
    lo = np.maximum(hi - 1, 0)
    to_lo, to_hi = a - table[lo], table[hi] - a
    pick = np.where((to_hi < to_lo) | ((to_hi == to_lo) & (hi % 2 == 0)), hi, lo)
    return np.copysign(table[pick], v)


def quantised(x, fmt):
    """(values, scale bytes [rows, blocks]) of x [rows, cols] in float64."""
    rows, cols = x.shape
    full = np.zeros((rows, up(cols, 32)))
    full[:, :cols] = x
    blocks = full.reshape(rows, -1, 32)
    bad = ~np.isfinite(blocks).all(-1)
    amax = np.abs(np.where(bad[..., None], 0.0, blocks)).max(-1)
    e = scale_exponents(amax, fmt)
    with np.errstate(invalid="ignore"):
        v = nearest(np.ldexp(blocks, -e[..., None]), fmt) * np.ldexp(1.0, e)[..., None]
    v[bad] = np.nan
    return v.reshape(rows, -1)[:, :cols], np.where(bad, 255, e + 127).astype(np.uint8)


def draw(x, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """The token of one row of logits, by the definition."""
    x = np.asarray(x, dtype=np.float64)
    ok = ~np.isnan(x) & (x > -np.inf)
    if not ok.any():
        return 0
    top = x[ok].max()
    if not temperature >= 2.0 ** -126:
        return int(np.flatnonzero(x == top)[0])
    with np.errstate(invalid="ignore"):
        w = np.where(x == top, 1.0, np.exp((x - top) / temperature))
    w[~ok] = 0.0
    w[np.isnan(w)] = 0.0
    order = np.lexsort((np.arange(len(x)), -np.where(ok, x, -np.inf)))
    order = order[:ok.sum()]
    if 0 < top_k < len(order):
        order = order[:top_k]
    if top_p < 1:
        sums = np.concatenate([[0.0], np.cumsum(w[order])])
        order = order[:max(1, int((sums[:-1] < top_p * sums[-1]).sum()))]
    if min_p > 0:
        order = np.concatenate([order[:1], order[1:][w[order[1:]] >= min_p]])
    kept = np.sort(order)
    sums = np.cumsum(w[kept])
    at = np.searchsorted(sums, u * sums[-1], side="right")
    return int(kept[min(at, len(kept) - 1)])
