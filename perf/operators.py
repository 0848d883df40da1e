"""The operators between a decoder's QKV projection and its attention output,
as cases that can be run in two ways: in elementary torch operations (`own`
false) and through the library's entry points (`own` true).

  rotary     rotary positions of Q and K rows (tb_b200_rotary)
  qk_norm    RMSNorm of each Q and K head, then rotary positions, in one pass
             (tb_b200_qk_norm_rotary)
  append     K and V rows into a paged 8-bit cache with one power-of-two scale
             per page and head (tb_b200_kv8_append)
  attention  attention over that cache (tb_b200_kv8_attention)

Sizes are the repository's workloads (workloads.py: mock, 7b, decode, 70b) and
generic ones around them.
"""
import math
import os
import random
import sys

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
CODES = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
LARGEST_CODE = {"int8": 127.0, "e4m3": 448.0}
LEAST_SCALE = 2.0 ** -100


def _T():
    """The library's Python binding."""
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                       "tensorbit-run_b200")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import tb_b200
    return tb_b200


# ------------------------------------------------------------------ cases
def _rope(name, op, rows, hq, hkv, d, r, dtype, layout, scaling, theta, first=0, fresh=False):
    return {"name": name, "op": op, "rows": rows, "hq": hq, "hkv": hkv, "d": d, "r": r,
            "dtype": dtype, "layout": layout, "scaling": scaling, "theta": theta,
            "first": first, "fresh": fresh}


def _append(name, seqs, least, most, held, hkv, d, page, dtype, fmt):
    return {"name": name, "op": "append", "seqs": seqs, "least": least, "most": most,
            "held": held, "hkv": hkv, "d": d, "page": page, "dtype": dtype, "format": fmt}


def _attention(name, seqs, least_q, most_q, least, most, hq, hkv, d, page, window, dtype, fmt):
    return {"name": name, "op": "attention", "seqs": seqs, "least_q": least_q, "most_q": most_q,
            "least": least, "most": most, "hq": hq, "hkv": hkv, "d": d, "page": page,
            "window": window, "dtype": dtype, "format": fmt}


def listed():
    return [
        # one token of the mock model, its frequencies following the length
        _rope("rotary token dynamic", "rotary", 1, 4, 4, 64, 64, "f32", "interleaved", "ntk", 1e4,
              first=5000, fresh=True),
        # a short prompt of a model that rotates part of an 80-wide head
        _rope("rotary partial f32", "rotary", 777, 32, 32, 80, 32, "f32", "half", "none", 1e4),
        # a 16384-token prefill chunk at the 70B shape, behind 114688 tokens of a long context
        _rope("rotary prefill 70b", "rotary", 16384, 64, 8, 128, 128, "bf16", "half", "bands",
              5e5, first=114688),
        # a decode batch of 256 tokens at the 7B shape
        _rope("qk_norm decode 256", "qk_norm", 256, 32, 32, 128, 128, "bf16", "interleaved",
              "none", 1e4, first=4000),
        # a 7B prefill in f32, an odd number of rows, half of each head rotated
        _rope("qk_norm prefill f32", "qk_norm", 4095, 32, 32, 128, 64, "f32", "half", "yarn", 1e4,
              first=1 << 15),
        # one new token for each of 256 sequences at the 70B shape's eight kv heads
        _append("append decode 256", 256, 1, 1, 1000, 8, 128, 64, "bf16", "int8"),
        # five prompts, 16000 tokens or so, behind nothing or a shared prefix
        _append("append prefill", 5, 700, 5700, 90, 8, 128, 64, "bf16", "e4m3"),
        # one token of the mock model over a short cache
        _attention("attention token f32", 1, 1, 1, 57, 57, 4, 4, 64, 16, 0, "f32", "int8"),
        # a decode batch of 64 sequences of up to 8192 tokens at the 70B shape
        _attention("attention decode 64", 64, 1, 1, 1, 8191, 64, 8, 128, 64, 0, "bf16", "int8"),
        # one sequence of a long context at the 70B shape
        _attention("attention long", 1, 1, 1, 131071, 131071, 64, 8, 128, 64, 0, "bf16", "e4m3"),
        # drafts of one to eight tokens checked at once, a window of 1000 tokens, small pages
        _attention("attention drafts", 48, 1, 8, 100, 3000, 32, 8, 64, 16, 1000, "bf16", "e4m3"),
        # a chunk of a prompt behind 6144 cached tokens
        _attention("attention chunk", 1, 2048, 2048, 8192, 8192, 32, 8, 128, 64, 0, "bf16",
                   "int8"),
    ]


def _between(rng, lo, hi):
    """A whole number of [lo, hi], evenly over its logarithm."""
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5))))))


def draw(rng):
    while True:
        op = rng.choice(["rotary", "qk_norm", "append", "attention", "attention"])
        d = rng.choice([64, 64, 80, 96, 128, 128, 128, 256])
        hkv = rng.choice([1, 2, 4, 8, 8])
        hq = hkv * rng.choice([1, 1, 2, 4, 7, 8])
        dtype = rng.choice(["bf16", "bf16", "f32"])
        fmt = rng.choice(["int8", "e4m3"])
        page = rng.choice([16, 32, 64, 64, 128])
        if op in ("rotary", "qk_norm"):
            c = _rope("", op, _between(rng, 1, 16384), hq, hkv, d, rng.choice([d, d, d // 2, 16]),
                      dtype, rng.choice(["half", "interleaved"]),
                      rng.choice(["none", "linear", "ntk", "bands", "yarn"]),
                      rng.choice([1e4, 5e5, 1e6]), first=rng.choice([0, _between(rng, 1, 1 << 20)]),
                      fresh=op == "rotary" and rng.random() < 0.3)
        elif op == "append":
            least = _between(rng, 1, 4000)
            c = _append("", _between(rng, 1, 256), least, _between(rng, least, 4 * least),
                        rng.choice([0, _between(rng, 1, 1000)]), hkv, d, page, dtype, fmt)
        else:
            least_q = rng.choice([1, 1, 1, _between(rng, 1, 300)])
            most_q = least_q if rng.random() < 0.5 else _between(rng, least_q, 4 * least_q)
            least = _between(rng, most_q, most_q + 8000)
            most = _between(rng, least, max(least, 60000))
            c = _attention("", _between(rng, 1, 128), least_q, most_q, least, most, hq, hkv, d,
                           page, rng.choice([0, 0, _between(rng, 16, 4096)]), dtype, fmt)
        w = work(c)
        if op == "attention":  # what the plain form lays out
            scores = c["seqs"] * c["hq"] * c["most_q"] * c["most"]
            keys = c["seqs"] * c["most"] * hkv * d
            if scores > 600e6 or keys > 600e6 or w["flops"] > 2.5e11:
                continue
        if w["bytes"] <= 600e6:
            del c["name"]
            return c


def _counts(case):
    """(new rows, held or total tokens) of each sequence: the case's own, whatever the seed."""
    rng = random.Random("%(seqs)d %(page)d %(hkv)d %(d)d" % case)
    if case["op"] == "append":
        new = [rng.randint(case["least"], case["most"]) for _ in range(case["seqs"])]
        return new, [n + rng.randint(0, case["held"]) for n in new]
    total = [rng.randint(case["least"], case["most"]) for _ in range(case["seqs"])]
    new = [min(t, rng.randint(case["least_q"], case["most_q"])) for t in total]
    return new, total


def work(case):
    s = 4 if case["dtype"] == "f32" else 2
    d = case["d"]
    if case["op"] in ("rotary", "qk_norm"):
        n = case["rows"] * (case["hq"] + case["hkv"]) * d
        return {"bytes": 2 * n * s + 4 * case["rows"] + 8 * (case["r"] // 2), "flops": 3 * n}
    new, total = _counts(case)
    hkv, page = case["hkv"], case["page"]
    if case["op"] == "append":
        n = 2 * sum(new) * hkv * d
        pages = sum((t - 1) // page - (t - m) // page + 1 for m, t in zip(new, total))
        return {"bytes": n * (s + 1) + 8 * pages * hkv, "flops": 2 * n}
    keys = pairs = 0
    for m, t in zip(new, total):
        w = case["window"] or t
        keys += min(t, w + m - 1)  # the keys that some query of the sequence sees
        first = t - m + 1          # keys the first and the last query may see: first .. t
        full = max(0, t - max(first, w) + 1)
        short = m - full
        pairs += full * w + short * first + short * (short - 1) // 2
    rows = sum(new)
    return {"bytes": 2 * keys * hkv * d + 8 * hkv * (keys // page) + 2 * rows * case["hq"] * d * s,
            "flops": 4 * d * case["hq"] * pairs}


# ----------------------------------------------------------------- inputs
SCALING = {  # factor, positions of training, low, high
    "none": (1.0, 4096, 0.0, 0.0), "linear": (4.0, 4096, 0.0, 0.0), "ntk": (8.0, 4096, 0.0, 0.0),
    "bands": (8.0, 8192, 1.0, 4.0), "yarn": (16.0, 4096, 1.0, 32.0)}


def _freqs(r, theta, scaling, device):
    """Angle per position of each pair, in 64 bits."""
    factor, trained, low, high = SCALING[scaling]
    if scaling == "ntk":
        theta = theta * factor ** (r / (r - 2))
    i = torch.arange(r // 2, dtype=torch.float64, device=device)
    f = theta ** (-2 * i / r)
    if scaling == "linear":
        f = f / factor
    elif scaling == "bands":
        turns = trained * f / (2 * math.pi)
        keep = ((turns - low) / (high - low)).clamp(0, 1)
        f = f * ((1 - keep) / factor + keep)
    elif scaling == "yarn":
        at = lambda turns: r * math.log(trained / (turns * 2 * math.pi)) / (2 * math.log(theta))  # noqa: E731
        lo, hi = max(math.floor(at(high)), 0), min(math.ceil(at(low)), r - 1)
        ramp = ((i - lo) / ((hi - lo) or 0.001)).clamp(0, 1)
        f = f * (1 - ramp) + f / factor * ramp
    return f


def _attention_factor(scaling):
    return 0.1 * math.log(SCALING[scaling][0]) + 1 if scaling == "yarn" else 1.0


def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    st = dict(case)
    d, hkv = case["d"], case["hkv"]
    if case["op"] in ("rotary", "qk_norm"):
        hq, rows = case["hq"], case["rows"]
        # one packed projection, as a decoder's QKV product leaves it
        qkv = (normal(rows, hq + 2 * hkv, d) * 1.5).to(dt)
        st["q"], st["k"] = qkv[:, :hq], qkv[:, hq:hq + hkv]
        first = case["first"]
        if rows > 1 and rows <= 256:  # a decode batch: positions of their own
            st["positions"] = torch.randint(0, first + rows, (rows,), generator=g, device="cuda",
                                            dtype=torch.int32)
        else:
            st["positions"] = torch.arange(first, first + rows, device="cuda", dtype=torch.int32)
        st["freqs"] = _freqs(case["r"], case["theta"], case["scaling"], "cuda")
        st["q_weight"] = (1 + 0.1 * normal(d)).to(dt)
        st["k_weight"] = (1 + 0.1 * normal(d)).to(dt)
        return st
    page, seqs = case["page"], case["seqs"]
    new, total = _counts(case)
    width = -(-max(total) // page)
    each = [-(-t // page) for t in total]
    pages = sum(each) + 1  # page 0 belongs to nobody: unused places of the table name it
    order = 1 + torch.randperm(pages - 1, generator=g, device="cuda").to(torch.int32)
    used = torch.arange(width, device="cuda") < torch.tensor(each, device="cuda")[:, None]
    table = torch.zeros(seqs, width, dtype=torch.int32, device="cuda")
    table[used] = order
    st["page_table"] = table
    st["lengths"] = torch.tensor(total, dtype=torch.int32, device="cuda")
    st["q_start"] = torch.tensor([0] + [sum(new[:i + 1]) for i in range(seqs)], dtype=torch.int32,
                                 device="cuda")
    st["new"], st["max_q"], st["max_len"] = sum(new), max(new), max(total)
    largest = LARGEST_CODE[case["format"]]

    def held():
        x = normal(pages, hkv, page, d) * (0.5 + normal(pages, hkv, 1, 1).abs())
        scale = _power_of_two_over(x.abs().amax((2, 3)), largest)
        return _coded(x / scale[:, :, None, None], case["format"]), scale

    st["k_codes"], st["k_scale"] = held()
    st["v_codes"], st["v_scale"] = held()
    if case["op"] == "append":
        # a batch's values grow now and then: about a fifth of the pages that a token joins
        # need a larger scale
        kv = (normal(st["new"], 2, hkv, d) * (0.5 + normal(st["new"], 1, hkv, 1).abs())).to(dt)
        st["k"], st["v"] = kv[:, 0], kv[:, 1]
    else:
        st["q"] = (2 * normal(st["new"], case["hq"], d)).to(dt)
    return st


# -------------------------------------------------------------- plain form
def _power_of_two_over(amax, largest):
    """The least power of two (2^-100 or more) that takes amax to `largest` or below; in 64
    bits, since amax / largest is next to a power of two now and then."""
    m, e = torch.frexp(amax.double() / largest)
    s = torch.ldexp(torch.ones_like(m), e - (m == 0.5).to(e.dtype))
    return s.clamp(min=LEAST_SCALE).float()


def _coded(x, fmt):
    if fmt == "int8":
        return x.round().clamp(-127, 127).to(torch.int8)
    return x.clamp(-448, 448).to(torch.float8_e4m3fn)


def _rotated(x, cos, sin, r, layout):
    x, rest = x[..., :r], x[..., r:]
    if layout == "interleaved":
        a, b = x[..., 0::2], x[..., 1::2]
        y = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = x[..., :r // 2], x[..., r // 2:]
        y = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((y, rest), -1)


def _rotary_plain(st):
    freqs = _freqs(st["r"], st["theta"], st["scaling"], "cuda") if st["fresh"] else st["freqs"]
    angle = st["positions"].double()[:, None, None] * freqs  # far positions: 64 bits
    m = _attention_factor(st["scaling"])
    cos, sin = (m * angle.cos()).float(), (m * angle.sin()).float()
    out = []
    for x, w in ((st["q"], st["q_weight"]), (st["k"], st["k_weight"])):
        y = x.float()
        if st["op"] == "qk_norm":
            y = y / (y.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w.float()
        out.append(_rotated(y, cos, sin, st["r"], st["layout"]).to(x.dtype))
    return out + ([freqs] if st["fresh"] else [])


def _append_plain(st):
    page = st["page"]
    largest = LARGEST_CODE[st["format"]]
    start = st["q_start"][:-1].long()
    count = st["q_start"][1:].long() - start
    total = st["lengths"].long()
    first = total - count  # the position of each sequence's first new row
    units = min((st["max_q"] - 2) // page + 2, st["page_table"].shape[1])
    logical = first[:, None] // page + torch.arange(units, device="cuda")
    touched = logical * page < total[:, None]
    at = torch.where(touched, st["page_table"].long().gather(
        1, logical.clamp(max=st["page_table"].shape[1] - 1)), 0).flatten()
    pos = logical[..., None] * page + torch.arange(page, device="cuda")  # seq, unit, slot
    fresh = touched[..., None] & (pos >= first[:, None, None]) & (pos < total[:, None, None])
    row = torch.where(fresh, start[:, None, None] + pos - first[:, None, None], 0)
    fresh = fresh.flatten(0, 1)[:, None, :, None]
    before = (touched[..., None] & (pos < first[:, None, None])).flatten(0, 1)[:, None, :, None]
    for name in ("k", "v"):
        x = st[name][row.flatten()].view(-1, page, st["hkv"], st["d"]).transpose(1, 2).float()
        x = torch.where(fresh, x, 0.0)
        codes, scale = st[name + "_codes"], st[name + "_scale"]
        held = codes[at].float()
        old = torch.where(before.any(2).squeeze(-1), scale[at], 0.0)
        s = torch.maximum(old, _power_of_two_over(x.abs().amax((2, 3)), largest))
        ratio = (old / s)[:, :, None, None]
        y = torch.where(fresh, x / s[:, :, None, None], torch.where(before, held * ratio, held))
        keep = at == 0
        s = torch.where(keep[:, None], scale[at], s)
        raw = codes.view(torch.uint8)
        raw[at] = _coded(y, st["format"]).view(torch.uint8)
        scale[at] = s
    return [st["k_codes"], st["v_codes"], st["k_scale"], st["v_scale"]]


def _attention_plain(st):
    page, hq, hkv, d = st["page"], st["hq"], st["hkv"], st["d"]
    table = st["page_table"].long()
    seqs, width = table.shape
    start = st["q_start"][:-1].long()
    count = st["q_start"][1:].long() - start
    total = st["lengths"].long()

    def laid_out(codes, scale):  # seqs, hkv, tokens, d
        x = codes[table].float() * scale[table][..., None, None]
        return x.transpose(1, 2).reshape(seqs, hkv, width * page, d)

    t = torch.arange(st["max_q"], device="cuda")
    there = t < count[:, None]
    row = torch.where(there, start[:, None] + t, 0)
    q = st["q"][row].float()  # seqs, max_q, hq, d
    q = q.view(seqs, -1, hkv, hq // hkv, d).permute(0, 2, 3, 1, 4).reshape(seqs, hkv, -1, d)
    s = q @ laid_out(st["k_codes"], st["k_scale"]).transpose(-1, -2) / math.sqrt(d)
    s = s.view(seqs, hkv, hq // hkv, st["max_q"], width * page)
    p = (total - count)[:, None] + t  # position of each query
    j = torch.arange(width * page, device="cuda")
    seen = (j <= p[..., None]) & there[..., None]
    if st["window"]:
        seen &= j > p[..., None] - st["window"]
    seen = seen[:, None, None]
    s = s.masked_fill_(~seen, -math.inf)
    top = s.amax(-1, keepdim=True)
    e = (s - torch.where(top == -math.inf, 0.0, top)).exp_()
    z = e.sum(-1, keepdim=True)
    o = e.view(seqs, hkv, -1, width * page) @ laid_out(st["v_codes"], st["v_scale"])
    o = o.view(seqs, hkv, hq // hkv, -1, d) / torch.where(z == 0, 1.0, z)
    lse = (top + z.log()).squeeze(-1)
    o = o.permute(0, 3, 1, 2, 4).reshape(seqs, -1, hq, d)[there]  # rows in their order
    lse = lse.permute(0, 3, 1, 2).reshape(seqs, -1, hq)[there]
    return [o.to(st["q"].dtype), lse]


# --------------------------------------------------------------- the calls
def _rotary_own(st):
    T = _T()
    layout = T.ROTARY_HALF if st["layout"] == "half" else T.ROTARY_INTERLEAVED
    freqs = st["freqs"]
    if st["fresh"]:
        factor, trained, low, high = SCALING[st["scaling"]]
        freqs = T.rotary_freqs(st["r"], st["theta"], st["scaling"], factor, trained, low, high)
    m = _attention_factor(st["scaling"])
    if st["op"] == "qk_norm":
        return list(T.qk_norm_rotary(st["q"], st["k"], st["q_weight"], st["k_weight"], 1e-6,
                                     st["positions"], freqs, layout, m))
    return list(T.rotary(st["q"], st["k"], st["positions"], freqs, layout, m)) + (
        [freqs] if st["fresh"] else [])


def _append_own(st):
    T = _T()
    cache = T.Kv8Cache(st["k_codes"], st["v_codes"], st["k_scale"], st["v_scale"])
    T.kv8_append(cache, st["k"], st["v"], st["q_start"], st["lengths"], st["page_table"])
    return [st["k_codes"], st["v_codes"], st["k_scale"], st["v_scale"]]


def _attention_own(st):
    T = _T()
    cache = T.Kv8Cache(st["k_codes"], st["v_codes"], st["k_scale"], st["v_scale"])
    return list(T.kv8_attention(cache, st["q"], st["q_start"], st["lengths"], st["page_table"],
                                max_q=st["max_q"], max_len=st["max_len"], window=st["window"],
                                return_lse=True))


def run(state):
    """One pass.  8-bit codes come back in their own 8-bit type, beside their scales: int8 codes
    are whole numbers that do not depend on how they are computed, because a quotient by a power
    of two is exact."""
    op = state["op"]
    if op in ("rotary", "qk_norm"):
        return _rotary_own(state) if own else _rotary_plain(state)
    if op == "append":
        return _append_own(state) if own else _append_plain(state)
    return _attention_own(state) if own else _attention_plain(state)


# ------------------------------------------------------ 64-bit definitions
def _exact_codes(x, fmt):
    """Values x in 64 bits to the nearest code, ties to the even one."""
    if fmt == "int8":
        return x.round()
    e = torch.frexp(x)[1].sub(1).clamp(min=-6)
    step = torch.ldexp(torch.ones_like(x), e - 3)
    return (x / step).round() * step


def _exact_rotary(st):
    r, h = st["r"], st["r"] // 2
    if st["layout"] == "half":
        first, second = torch.arange(h, device="cuda"), torch.arange(h, r, device="cuda")
    else:
        first = 2 * torch.arange(h, device="cuda")
        second = first + 1
    f = st["freqs"]
    turn = torch.polar(torch.full((st["rows"], 1, h), _attention_factor(st["scaling"]),
                                  device="cuda", dtype=torch.float64),
                       st["positions"].double()[:, None, None] * f)
    out = []
    for x, w in ((st["q"], st["q_weight"]), (st["k"], st["k_weight"])):
        x = x.double()
        if st["op"] == "qk_norm":
            x = x * w.double() * torch.rsqrt((x * x).sum(-1, keepdim=True) / st["d"] + 1e-6)
        z = torch.complex(x[..., first], x[..., second]) * turn
        y = x.clone()
        y[..., first], y[..., second] = z.real, z.imag
        out.append(y)
    return out + ([f] if st["fresh"] else [])


def _exact_append(st):
    page, fmt = st["page"], st["format"]
    out = {}
    start = st["q_start"].tolist()
    table = st["page_table"].tolist()
    for name in ("k", "v"):
        codes = st[name + "_codes"].double()
        scale = st[name + "_scale"].double()
        for i, total in enumerate(st["lengths"].tolist()):
            x = st[name][start[i]:start[i + 1]].double()
            pos = total - x.shape[0]
            while pos < total:
                end = min(total, (pos // page + 1) * page)
                at, slot = table[i][pos // page], pos % page
                part = x[pos - total + x.shape[0]:end - total + x.shape[0]].transpose(0, 1)
                amax = part.abs().amax((1, 2))
                s = torch.full_like(amax, LEAST_SCALE)
                need = torch.log2(amax / LARGEST_CODE[fmt]).round().clamp(min=-100)
                need = torch.exp2(need)
                need = torch.where(need * LARGEST_CODE[fmt] < amax, 2 * need, need)
                half = need / 2
                need = torch.where(half * LARGEST_CODE[fmt] >= amax, half, need)
                s = torch.maximum(s, need)
                if slot:
                    s = torch.maximum(s, scale[at])
                    old = codes[at, :, :slot] * (scale[at] / s)[:, None, None]
                    codes[at, :, :slot] = _exact_codes(old, fmt)
                codes[at, :, slot:slot + part.shape[1]] = _exact_codes(part / s[:, None, None], fmt)
                scale[at] = s
                pos = end
        out[name] = codes if fmt == "e4m3" else codes.to(torch.int8), scale
    return [out["k"][0], out["v"][0], out["k"][1], out["v"][1]]


def _exact_attention(st):
    hq, hkv, d = st["hq"], st["hkv"], st["d"]
    group = hq // hkv
    start = st["q_start"].tolist()
    o = torch.zeros(st["new"], hq, d, dtype=torch.float64, device="cuda")
    lse = torch.full((st["new"], hq), -math.inf, dtype=torch.float64, device="cuda")
    for i, total in enumerate(st["lengths"].tolist()):
        m = start[i + 1] - start[i]
        if not m or not total:
            continue
        pages = st["page_table"][i, :-(-total // st["page"])].long()
        hidden = (torch.arange(total, device="cuda")
                  > torch.arange(total - m, total, device="cuda")[:, None])
        if st["window"]:
            hidden |= (torch.arange(total, device="cuda")
                       <= torch.arange(total - m, total, device="cuda")[:, None] - st["window"])
        for h in range(hkv):
            k, v = (st[n + "_codes"][pages, h].double() * st[n + "_scale"][pages, h].double()[
                :, None, None] for n in ("k", "v"))
            k, v = k.reshape(-1, d)[:total], v.reshape(-1, d)[:total]
            q = st["q"][start[i]:start[i + 1], h * group:(h + 1) * group].double()
            s = torch.einsum("mgd,td->gmt", q, k) / math.sqrt(d)
            s[:, hidden] = -math.inf
            z = torch.logsumexp(s, -1)
            lse[start[i]:start[i + 1], h * group:(h + 1) * group] = z.T
            w = torch.exp(s - z[..., None])
            o[start[i]:start[i + 1], h * group:(h + 1) * group] = torch.einsum(
                "gmt,td->mgd", w, v)
    return [o, lse]


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] in ("rotary", "qk_norm"):
        return _exact_rotary(st)
    if case["op"] == "append":
        return _exact_append(st)
    if work(case)["flops"] > 3e11:
        return None
    return _exact_attention(st)
