"""Linear layers in microscaled formats and the sampling behind the last of them, as cases that
can be run in two ways: in elementary torch operations (`own` false) and through the library's
entry points (`own` true).

  quantize   rows to 8- or 4-bit codes with a power-of-two scale for each 32 elements
             (tb_b200_mx_quantize; 4-bit codes come back as their values, tb_b200_mx_dequantize)
  norm       residual add and RMSNorm with such an output (tb_b200_residual_rms_norm_mx)
  swiglu     SwiGLU with such an output (tb_b200_swiglu_mx)
  linear     the product of such rows with such weights (tb_b200_mx_linear)
  sample     temperature, top-k, top-p and min-p sampling of logits (tb_b200_sample)

Sizes are the repository's workloads (workloads.py: mock, 7b, decode, 70b) and generic ones
around them.
"""
import math
import os
import sys

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
LARGEST = {"e4m3": 448.0, "e2m1": 6.0}
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
EPS = 1e-5


def _T():
    """The library's Python binding."""
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                       "tensorbit-run_b200")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import tb_b200
    return tb_b200


# ------------------------------------------------------------------ cases
def _rows(name, op, rows, cols, dtype, fmt):
    return {"name": name, "op": op, "rows": rows, "cols": cols, "dtype": dtype, "format": fmt}


def _linear(name, rows, cols, outs, xf, wf, dtype, bias=False):
    return {"name": name, "op": "linear", "rows": rows, "cols": cols, "outs": outs, "x": xf,
            "w": wf, "dtype": dtype, "bias": bias}


def _sample(name, rows, vocab, dtype, std, most_k, least_p, most_min_p, greedy):
    return {"name": name, "op": "sample", "rows": rows, "vocab": vocab, "dtype": dtype, "std": std,
            "most_k": most_k, "least_p": least_p, "most_min_p": most_min_p, "greedy": greedy}


def listed():
    return [
        # one token's hidden state on its way into a projection at the 7B shape
        _rows("quantize token", "quantize", 1, 4096, "bf16", "e4m3"),
        # the 70B shape's gate projection, quantised as a model is loaded, and looked at
        _rows("quantize weight 70b", "quantize", 28672, 8192, "bf16", "e2m1"),
        # a decode batch of 256 tokens at the 70B shape, in front of QKV or gate and up
        _rows("norm decode 256", "norm", 256, 8192, "bf16", "e4m3"),
        # a 70B prefill
        _rows("norm prefill 70b", "norm", 16384, 8192, "bf16", "e4m3"),
        # a short prompt in f32, an odd number of rows
        _rows("swiglu odd f32", "swiglu", 777, 11008, "f32", "e4m3"),
        # a 70B prefill chunk, in front of the down projection
        _rows("swiglu prefill 70b", "swiglu", 4096, 28672, "bf16", "e4m3"),
        # one token through a 7B projection
        _linear("linear token", 1, 4096, 4096, "e4m3", "e2m1", "bf16"),
        # a decode batch of 64 tokens to logits at the 70B shape
        _linear("linear head 64", 64, 8192, 128256, "e4m3", "e2m1", "f32"),
        # a 70B prefill chunk through the gate projection, 8-bit rows
        _linear("linear prefill", 4096, 8192, 28672, "e4m3", "e2m1", "bf16"),
        # an odd prompt through the down projection, both sides in 4 bits
        _linear("linear odd 4 bits", 3001, 28672, 8192, "e2m1", "e2m1", "bf16"),
        # one request of a 32000-word vocabulary
        _sample("sample token", 1, 32000, "f32", 3.0, 50, 0.9, 0.0, False),
        # a decode batch of 256 requests of all kinds at the 70B shape's vocabulary
        _sample("sample decode 256", 256, 128256, "f32", 3.0, 100, 0.8, 0.1, True),
    ]


def _between(rng, lo, hi):
    """A whole number of [lo, hi], evenly over its logarithm."""
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5))))))


def draw(rng):
    while True:
        op = rng.choice(["quantize", "norm", "swiglu", "linear", "linear", "sample", "sample"])
        dtype = rng.choice(["bf16", "bf16", "f32"])
        fmt = rng.choice(["e4m3", "e4m3", "e2m1"])
        if op in ("quantize", "norm", "swiglu"):
            c = _rows("", op, _between(rng, 1, 16384), _between(rng, 64, 28672), dtype, fmt)
            fits = c["rows"] * c["cols"] <= 117e6
        elif op == "linear":
            xf, wf = rng.choice([("e4m3", "e2m1"), ("e4m3", "e2m1"), ("e2m1", "e2m1"),
                                 ("e4m3", "e4m3")])
            c = _linear("", _between(rng, 1, 4096), _between(rng, 64, 28672),
                        _between(rng, 16, 65536), xf, wf, dtype, rng.random() < 0.3)
            fits = c["cols"] * c["outs"] <= 250e6 and work(c)["flops"] <= 1e12
        else:
            c = _sample("", _between(rng, 1, 1024), _between(rng, 100, 200000), dtype,
                        rng.choice([1.0, 2.0, 3.0, 6.0]), rng.choice([0, 1, 20, 50, 1000]),
                        rng.choice([1.0, 0.95, 0.9, 0.5]), rng.choice([0.0, 0.0, 0.05, 0.3]),
                        rng.random() < 0.5)
            fits = c["rows"] * c["vocab"] <= 33e6
        if fits:
            del c["name"]
            return c


def _up(n, to):
    return -(-n // to) * to


def _held(rows, cols, fmt):
    """Bytes of rows in a format: codes and scales."""
    return rows * cols * (1 if fmt == "e4m3" else 0.5) + rows * (-(-cols // 32))


def work(case):
    s = 4 if case["dtype"] == "f32" else 2
    rows = case["rows"]
    if case["op"] == "linear":
        k, n = case["cols"], case["outs"]
        return {"bytes": _held(rows, k, case["x"]) + _held(n, k, case["w"]) + rows * n * s
                + 4 * n * case["bias"], "flops": 2 * rows * n * k}
    if case["op"] == "sample":
        return {"bytes": rows * (case["vocab"] * s + 28), "flops": 2 * rows * case["vocab"]}
    n, fmt = rows * case["cols"], case["format"]
    reads = {"quantize": 1, "norm": 2, "swiglu": 2}[case["op"]]
    size = n * s * (reads + (case["op"] == "norm")) + _held(rows, case["cols"], fmt)
    if fmt == "e2m1":  # read again, and their values written
        size += _held(rows, case["cols"], fmt) + n * 2
    return {"bytes": size, "flops": 4 * n}


# ----------------------------------------------------------------- inputs
def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    st = dict(case)
    rows = case["rows"]
    if case["op"] == "sample":
        n, p = case["vocab"], torch.rand(rows, 4, generator=g, device="cuda")
        st["logits"] = (normal(rows, n) * case["std"]).to(dt)
        st["uniforms"] = torch.rand(rows, generator=g, device="cuda", dtype=torch.float64)
        # requests with settings of their own
        st["temperature"] = 0.5 + p[:, 0]
        if case["greedy"]:
            st["temperature"][p[:, 0] < 0.1] = 0.0
        st["top_k"] = (p[:, 1] * (case["most_k"] + 1)).int()  # 0: all
        st["top_p"] = case["least_p"] + (1 - case["least_p"]) * p[:, 2] * 1.25  # 1 and over: all
        st["min_p"] = (case["most_min_p"] * (2 * p[:, 3] - 1)).clamp(min=0.0)  # 0: all
        return st
    cols = case["cols"]
    if case["op"] == "linear":
        # activations a few of whose features are large, as behind a norm; weights as trained
        wide = 1 + 8 * (torch.rand(cols, generator=g, device="cuda") < 0.01)
        st["x_codes"], st["x_scales"] = _quantized(normal(rows, cols) * wide, case["x"])
        parts = [_quantized(normal(min(8192, case["outs"] - at), cols) * 0.02, case["w"])
                 for at in range(0, case["outs"], 8192)]  # 8192: whole tiles of scales
        st["w_codes"] = torch.cat([p[0] for p in parts])
        st["w_scales"] = torch.cat([p[1] for p in parts])
        st["bias_values"] = normal(case["outs"]) if case["bias"] else None
        return st
    if case["op"] == "swiglu":  # as the joint product of gate and up leaves them
        both = (normal(rows, 2 * cols) * 1.5).to(dt)
        st["gate"], st["up"] = both[:, :cols], both[:, cols:]
        return st
    st["x"] = (normal(rows, cols) * (1 + 8 * (torch.rand(cols, generator=g, device="cuda")
                                              < 0.01))).to(dt)
    if case["op"] == "norm":
        st["residual"] = (3 * normal(rows, cols)).to(dt)
        st["weight"] = (1 + 0.1 * normal(cols)).to(dt)
    return st


# -------------------------------------------------------------- plain form
def _tiled(scales):
    """Scale bytes [rows, blocks] in tiles of 128 rows and 4 blocks: byte 16 (r % 32) +
    4 (r % 128 / 32) + b % 4 of tile (r / 128, b / 4) is row r's block b."""
    rows, blocks = scales.shape
    s = torch.zeros(_up(rows, 128), _up(blocks, 4), dtype=torch.uint8, device=scales.device)
    s[:rows, :blocks] = scales
    s = s.view(s.shape[0] // 128, 4, 32, s.shape[1] // 4, 4)
    return s.permute(0, 3, 2, 1, 4).reshape(-1)


def _scale_values(tiled, rows, cols):
    """Scales [rows, blocks] in f32 of their tiles."""
    s = tiled.view(_up(rows, 128) // 128, -1, 32, 4, 4).permute(0, 3, 2, 1, 4)
    s = s.reshape(_up(rows, 128), -1)[:rows, :-(-cols // 32)]
    return torch.exp2(s.double() - 127).float()


def _codes_of(x, fmt):
    """Values x in f32, scaled into the format's range, to the nearest code, ties to even."""
    if fmt == "e4m3":
        return x.to(torch.float8_e4m3fn).view(torch.uint8)
    a = x.abs()
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    a = (a / step).round() * step
    code = torch.where(a < 2, 2 * a, torch.where(a < 4, a + 2, a / 2 + 4)).to(torch.uint8)
    code |= torch.signbit(x).to(torch.uint8) << 3
    return code[:, 0::2] | code[:, 1::2] << 4


def _quantized(x, fmt):
    """(codes, tiled scales) of rows x in f32, their columns filled up to a multiple of 128."""
    rows, cols = x.shape
    x = torch.nn.functional.pad(x, (0, _up(cols, 128) - cols))
    x = x.view(rows, -1, 32)
    m, e = torch.frexp(x.abs().amax(-1).double() / LARGEST[fmt])  # next to a power of two: 64 bits
    e = torch.where(m == 0, -127, (e - (m == 0.5).to(e.dtype))).clamp(min=-127)
    scale = torch.ldexp(torch.ones_like(m), e).float()
    codes = _codes_of((x / scale[..., None]).view(rows, -1), fmt)
    return codes, _tiled((e + 127).to(torch.uint8))


def _values(codes, tiled, cols, fmt):
    """The f32 values [rows, cols] that codes and scales stand for."""
    rows = codes.shape[0]
    if fmt == "e4m3":
        v = codes[:, :cols].view(torch.float8_e4m3fn).float()
    else:
        table = torch.tensor(E2M1 + tuple(-v for v in E2M1), device=codes.device)
        v = torch.stack((table[(codes & 15).int()], table[(codes >> 4).int()]), -1)
        v = v.view(rows, -1)[:, :cols]
    s = _scale_values(tiled, rows, cols).repeat_interleave(32, 1)[:, :cols]
    return v * s


def _returned(codes, tiled, cols, fmt):
    """8-bit codes and scales as the 8-bit floats that they are, 4-bit ones as their values."""
    if fmt == "e4m3":
        return [codes.view(torch.float8_e4m3fn), tiled.view(torch.float8_e8m0fnu)]
    return [_values(codes, tiled, cols, fmt).to(torch.bfloat16)]


def _sample_plain(st):
    x = st["logits"].double()
    rows, n = x.shape
    t = st["temperature"].double()[:, None]
    top = x.amax(-1, keepdim=True)
    x, order = x.sort(dim=-1, descending=True, stable=True)  # equal logits in their order
    w = ((x - top) / torch.where(t > 0, t, 1.0)).exp()
    k = st["top_k"].long()[:, None]
    w = torch.where((k > 0) & (torch.arange(n, device=x.device) >= k), 0.0, w)
    before = w.cumsum(-1) - w
    p = st["top_p"].double()[:, None]
    keep = (p >= 1) | (before < p * w.sum(-1, keepdim=True))
    keep[:, 0] = True
    keep &= w >= st["min_p"].double()[:, None]
    w = torch.zeros_like(w).scatter_(-1, order, torch.where(keep, w, 0.0))
    c = w.cumsum(-1)
    past = c > st["uniforms"][:, None] * c[:, -1:]
    drawn = torch.where(past & (w > 0), torch.arange(n, device=x.device), n).amin(-1)
    last = torch.where(w > 0, torch.arange(n, device=x.device), 0).amax(-1)
    drawn = torch.minimum(drawn, last)
    return [torch.where(t[:, 0] > 0, drawn, order[:, 0]).int()]


def _plain(st):
    op = st["op"]
    if op == "sample":
        return _sample_plain(st)
    if op == "linear":
        x = _values(st["x_codes"], st["x_scales"], st["cols"], st["x"])
        w = _values(st["w_codes"], st["w_scales"], st["cols"], st["w"])
        y = x @ w.T
        if st["bias"]:
            y = y + st["bias_values"]
        return [y.to(DTYPES[st["dtype"]])]
    out = []
    if op == "quantize":
        y = st["x"].float()
    elif op == "norm":
        h = st["x"].float() + st["residual"].float()
        out.append(h.to(st["x"].dtype))
        y = h / ((h.square().sum(-1, keepdim=True) + EPS) / st["cols"]).sqrt()
        y = y * st["weight"].float()
    else:
        gate = st["gate"].float()
        y = gate / (1 + (-gate).exp()) * st["up"].float()
    codes, scales = _quantized(y, st["format"])
    return out + _returned(codes, scales, st["cols"], st["format"])


# --------------------------------------------------------------- the calls
def _own(st):
    T = _T()
    op = st["op"]
    if op == "sample":
        return [T.sample(st["logits"], st["uniforms"], st["temperature"], st["top_k"],
                         st["top_p"], st["min_p"])]
    if op == "linear":
        x = T.MxTensor(st["x_codes"], st["x_scales"], st["cols"], st["x"])
        w = T.MxTensor(st["w_codes"], st["w_scales"], st["cols"], st["w"])
        return [T.mx_linear(x, w, bias=st["bias_values"], dtype=DTYPES[st["dtype"]])]
    out = []
    if op == "quantize":
        y = T.mx_quantize(st["x"], st["format"])
    elif op == "norm":
        h, y = T.residual_rms_norm_mx(st["x"], st["residual"], st["weight"], EPS,
                                      format=st["format"])
        out.append(h)
    else:
        y = T.swiglu_mx(st["gate"], st["up"], st["format"])
    if st["format"] == "e2m1":
        return out + [T.mx_dequantize(y, torch.bfloat16)]
    return out + [y.codes.view(torch.float8_e4m3fn), y.scales.view(torch.float8_e8m0fnu)]


def run(state):
    """One pass.  8-bit codes come back in their own 8-bit type beside their scales in theirs, in
    the layout in which the product reads them; 4-bit codes as the values that they stand for."""
    return _own(state) if own else _plain(state)


# ------------------------------------------------------ 64-bit definitions
def _exact_mx(y, fmt):
    """The values of rows y (in 64 bits) in a format: codes [rows, columns in whole tiles] before
    scaling, scales [rows in whole tiles, blocks in whole tiles] in their tiles."""
    rows, cols = y.shape
    wide, tall = _up(cols, 128), _up(rows, 128)
    full = torch.zeros(rows, wide, dtype=torch.float64, device=y.device)
    full[:, :cols] = y
    blocks = full.unflatten(1, (wide // 32, 32))
    amax = blocks.abs().max(2).values
    top = LARGEST[fmt]
    e = torch.log2(amax / top).ceil().nan_to_num(neginf=-127.0).clamp(min=-127.0)
    e = torch.where(torch.exp2(e - 1) * top >= amax, e - 1, e).clamp(min=-127.0)
    e = torch.where(torch.exp2(e) * top < amax, e + 1, e)
    v = blocks / torch.exp2(e)[..., None]
    least, bits = (-6, 3) if fmt == "e4m3" else (0, 1)
    power = torch.frexp(v)[1] - 1
    unit = torch.exp2(power.clamp(min=least).double() - bits)
    v = (v / unit).round() * unit
    scales = torch.full((tall, wide // 32), 2.0 ** -127, dtype=torch.float64, device=y.device)
    scales[:rows] = torch.exp2(e)
    if fmt == "e2m1":
        return [(v * scales[:rows, :, None]).flatten(1)[:, :cols]]
    r = torch.arange(tall, device=y.device)[:, None]
    b = torch.arange(wide // 32, device=y.device)
    at = (r // 128 * (wide // 128) + b // 4) * 512 + r % 32 * 16 + r % 128 // 32 * 4 + b % 4
    placed = torch.empty(scales.numel(), dtype=torch.float64, device=y.device)
    placed[at.flatten()] = scales.flatten()
    return [v.flatten(1), placed]


def _exact_values(codes, tiled, cols, fmt):
    rows = codes.shape[0]
    j = torch.arange(cols, device=codes.device)
    if fmt == "e4m3":
        bits = codes[:, :cols].int()
        e, m, sign, bias, steps = bits >> 3 & 15, bits & 7, bits >> 7, 7, 8
    else:
        bits = (codes[:, j // 2].int() >> (j % 2 * 4)) & 15
        e, m, sign, bias, steps = bits >> 1 & 3, bits & 1, bits >> 3, 1, 2
    v = torch.where(e > 0, torch.exp2((e - bias).double()) * (1 + m.double() / steps),
                    2.0 ** (1 - bias) * m.double() / steps)
    r, b = torch.arange(rows, device=codes.device)[:, None], j // 32
    at = (r // 128 * (_up(cols, 128) // 128) + b // 4) * 512 + r % 32 * 16
    at = at + r % 128 // 32 * 4 + b % 4
    return torch.where(sign > 0, -v, v) * torch.exp2(tiled[at].double() - 127)


def _exact_sample(st):
    rows, n = st["logits"].shape
    out = torch.zeros(rows, dtype=torch.int32)
    t, k, p, least = (st[a].double().tolist() for a in ("temperature", "top_k", "top_p", "min_p"))
    u = st["uniforms"].tolist()
    for i in range(rows):
        x = st["logits"][i].double()
        if not t[i] > 0:
            out[i] = int((x == x.max()).nonzero()[0])
            continue
        w = torch.exp((x - x.max()) / t[i])
        rank = torch.empty(n, dtype=torch.int64, device=x.device)
        rank[torch.argsort(-x, stable=True)] = torch.arange(n, device=x.device)
        among = rank < k[i] if k[i] >= 1 else rank >= 0
        if p[i] < 1:
            by_rank = torch.zeros(n, dtype=torch.float64, device=x.device)
            by_rank[rank] = torch.where(among, w, 0.0)
            sums = torch.cat((torch.zeros(1, dtype=torch.float64, device=x.device),
                              torch.cumsum(by_rank, 0)))
            taken = max(1, int((sums[:-1] < p[i] * sums[-1]).sum()))
            among = among & (rank < taken)
        among = among & (w >= least[i])
        index = among.nonzero()[:, 0]
        sums = torch.cumsum(w[index], 0)
        place = int(torch.searchsorted(sums, u[i] * sums[-1], right=True))
        out[i] = int(index[min(place, len(index) - 1)])
    return [out.to(st["logits"].device)]


def exact(case, seed):
    st = prepare(case, seed)
    op = case["op"]
    if op == "sample":
        return _exact_sample(st)
    if op == "linear":
        w = [_exact_values(st["w_codes"][at:at + 8192],
                           st["w_scales"][at // 128 * (_up(case["cols"], 128) // 128) * 512:],
                           case["cols"], case["w"]) for at in range(0, case["outs"], 8192)]
        x = _exact_values(st["x_codes"], st["x_scales"], case["cols"], case["x"])
        y = torch.cat([torch.einsum("rk,nk->rn", x, part) for part in w], 1)
        return [y if st["bias_values"] is None else y + st["bias_values"].double()]
    out = []
    if op == "quantize":
        y = st["x"].double()
    elif op == "norm":
        h = st["x"].double() + st["residual"].double()
        out.append(h)
        y = h * torch.rsqrt((torch.linalg.vector_norm(h, dim=-1, keepdim=True) ** 2 + EPS)
                            / case["cols"]) * st["weight"].double()
    else:
        gate = st["gate"].double()
        y = gate * torch.sigmoid(gate) * st["up"].double()
    return out + _exact_mx(y, case["format"])
