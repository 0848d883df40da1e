"""Filtered sampling on the GPU against its definition in 64 bits.

The kernel's weights are whole numbers of 2^-40 of the largest or finer, the definition's are
doubles, so both draw the same token unless u times the sum, or top_p times it, lies within
about 2^-38 of a border.  Seeds are fixed; the chance that one of the some 20000 draws here
lies so near is below 20000 * 2000 borders * 2^-38 = 2^-12.8, where a border is hit at all."""
import numpy as np
import pytest
import torch

import mx_ref as R
import tb_b200 as T

pytestmark = pytest.mark.gpu

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def check(x, u, temperature=None, top_k=None, top_p=None, min_p=None, rows=None):
    """x [rows, vocab] on the GPU; settings numpy arrays or None."""
    def dev(a, dtype):
        return None if a is None else torch.from_numpy(np.asarray(a, dtype)).cuda()
    f, n = np.float32, x.shape[0]
    got = T.sample(x, dev(u, np.float64), dev(temperature, f), dev(top_k, np.int32),
                   dev(top_p, f), dev(min_p, f)).cpu().numpy()
    host = x.double().cpu().numpy()
    for i in range(n) if rows is None else rows:
        at = {k: float(np.asarray(a, f)[i]) for k, a in
              (("temperature", temperature), ("top_p", top_p), ("min_p", min_p)) if a is not None}
        if top_k is not None:
            at["top_k"] = int(top_k[i])
        assert got[i] == R.draw(host[i], u[i], **at), (i, at, u[i])
    return got


def settings(r, n):
    return dict(temperature=r.choice([0.0, 0.3, 0.7, 1.0, 1.5, 5.0], n),
                top_k=r.choice([0, 1, 2, 5, 40, 1000, 10 ** 6, -1], n),
                top_p=r.choice([0.0, 0.1, 0.5, 0.9, 0.95, 0.999, 1.0, 2.0], n),
                min_p=r.choice([0.0, 0.0, 0.01, 0.1, 0.5, 1.0, 1.5], n))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("std", [0.0, 0.5, 3.0, 30.0])
@pytest.mark.parametrize("rows,vocab", [(64, 1), (64, 2), (64, 31), (300, 100), (300, 1000),
                                        (100, 4099), (20, 32000), (6, 128256), (2, 300001)])
def test_all_settings(rows, vocab, std, dtype):
    r = np.random.default_rng(vocab * 100 + int(std * 10))
    x = torch.from_numpy(r.standard_normal((rows, vocab)) * std + 5).to(DTYPES[dtype]).cuda()
    check(x, r.random(rows), **settings(r, rows))


@pytest.mark.parametrize("name", ["temperature", "top_k", "top_p", "min_p", None])
def test_one_setting(name):
    r = np.random.default_rng(7)
    x = torch.from_numpy(r.standard_normal((200, 777)) * 2).float().cuda()
    s = settings(r, 200)
    check(x, r.random(200), **({name: s[name]} if name else {}))


def test_ties_go_to_the_first():
    r = np.random.default_rng(8)
    x = torch.from_numpy(r.integers(-3, 3, (400, 500))).float().cuda()
    x[:, 7] = -0.0  # equal to 0
    s = settings(r, 400)
    s["top_k"] = r.integers(1, 300, 400)
    check(x, r.random(400), **s)
    same = torch.zeros(8, 1000, device="cuda")
    u = np.array([0.0, 0.25, 0.5, 0.999, 0.0, 0.25, 0.5, 0.999])
    got = check(same, u, top_p=np.full(8, 0.5), top_k=np.array([0] * 4 + [100] * 4))
    assert got.tolist() == [0, 125, 250, 499, 0, 12, 25, 49]


def test_ends_of_u():
    x = torch.tensor([[0.0, 1.0, -np.inf, 2.0, -1.0]], device="cuda").repeat(3, 1)
    got = check(x, np.array([0.0, 1 - 2.0 ** -53, 5e-324]))
    assert got.tolist() == [0, 4, 0]


def test_rows_with_little_left():
    """Masks of -infinity and of the type's lowest value, NaN, infinities, alone and mixed."""
    low, inf, nan = float(np.finfo(np.float32).min), np.inf, np.nan
    base = np.random.default_rng(9).standard_normal(40)
    rows = [np.full(40, -inf), np.full(40, nan), np.where(np.arange(40) == 33, 1.0, -inf),
            np.where(np.arange(40) == 12, low, -inf), np.full(40, low),
            np.where(np.arange(40) % 3 == 0, nan, base), np.where(np.arange(40) < 20, inf, base),
            np.where(np.arange(40) == 39, inf, nan), np.where(np.arange(40) < 30, low, base),
            np.where(np.arange(40) < 39, -inf, nan), np.where(np.arange(40) > 5, -inf, base)]
    x = torch.from_numpy(np.stack(rows)).float().cuda()
    n = len(rows)
    r = np.random.default_rng(10)
    for _ in range(6):
        check(x, r.random(n), **settings(r, n))
    check(x, r.random(n))
    got = check(x, r.random(n), temperature=np.full(n, np.inf))
    assert got[0] == 0 and got[1] == 0 and got[2] == 33 and got[3] == 12


@pytest.mark.parametrize("temperature", [1e-45, 1e-30, 1e-6, 1e6, 3e38])
def test_ends_of_temperature(temperature):
    r = np.random.default_rng(11)
    x = torch.from_numpy(r.standard_normal((50, 300))).float().cuda()
    check(x, r.random(50), temperature=np.full(50, temperature))


def test_least_temperatures():
    """Equal logits, and ones a least number apart, either side of 2^-126."""
    x = torch.zeros(40, 300, device="cuda")
    x[:, 100:] = 2.0 ** -149
    x[:, 200:250] = 2.0 ** -130
    r = np.random.default_rng(19)
    t = np.tile([2.0 ** -126, 2.0 ** -127, 2.0 ** -149, 2.0 ** -125], 10)
    check(x, r.random(40), temperature=t)
    check(x, r.random(40), temperature=t, top_p=np.full(40, 0.7), min_p=np.full(40, 0.9))


def test_negative_top_p_keeps_one():
    r = np.random.default_rng(20)
    x = torch.from_numpy(r.standard_normal((12, 3000))).float().cuda()
    got = check(x, r.random(12), top_p=np.tile([-1.0, -np.inf, 0.0], 4))
    assert torch.equal(torch.from_numpy(got).long(), x.argmax(-1).cpu())


def test_nan_settings_are_off():
    r = np.random.default_rng(12)
    x = torch.from_numpy(r.standard_normal((30, 100))).float().cuda()
    u, nan = r.random(30), np.full(30, np.nan)
    off = check(x, u)
    dev = lambda a: torch.from_numpy(a.astype(np.float32)).cuda()  # noqa: E731
    got = T.sample(x, torch.from_numpy(u).cuda(), None, None, dev(nan), dev(nan))
    assert got.cpu().numpy().tolist() == off.tolist()
    got = T.sample(x, torch.from_numpy(u).cuda(), dev(nan))
    assert torch.equal(got.long(), x.argmax(-1))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("off,stride", [(0, 1000), (1, 1001), (3, 1010), (8, 1016)])
def test_strided_rows(off, stride, dtype):
    r = np.random.default_rng(13)
    big = torch.full((60, stride), np.inf, dtype=DTYPES[dtype], device="cuda")
    x = big[:, off:off + 990]
    x.copy_(torch.from_numpy(r.standard_normal((60, 990)) * 2))
    check(x, r.random(60), **settings(r, 60))


def test_distribution():
    """Draws at evenly spaced u follow the weights."""
    x = torch.tensor([[0.0, 1.0, 2.0, -1.0, 0.5]], device="cuda").repeat(10000, 1)
    u = (torch.arange(10000, dtype=torch.float64, device="cuda") + 0.5) / 10000
    got = torch.bincount(T.sample(x, u).long(), minlength=5).double().cpu() / 10000
    assert (got - torch.softmax(x[0].double().cpu(), 0)).abs().max() <= 1e-4


def test_same_settings_from_a_graph_and_another_stream():
    r = np.random.default_rng(14)
    x = torch.from_numpy(r.standard_normal((40, 5000)) * 2).float().cuda()
    u = torch.from_numpy(r.random(40)).cuda()
    s = settings(r, 40)
    dev = [torch.from_numpy(s["temperature"].astype(np.float32)).cuda(),
           torch.from_numpy(s["top_k"].astype(np.int32)).cuda(),
           torch.from_numpy(s["top_p"].astype(np.float32)).cuda(),
           torch.from_numpy(s["min_p"].astype(np.float32)).cuda()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        T.sample(x, u, *dev)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = T.sample(x, u, *dev)
    for seed in (15, 16):
        r = np.random.default_rng(seed)
        x.copy_(torch.from_numpy(r.standard_normal((40, 5000)) * 2))
        u.copy_(torch.from_numpy(r.random(40)))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        want = check(x, u.cpu().numpy(), **s)
        assert out.cpu().numpy().tolist() == want.tolist()


def test_head_and_sample():
    """Final norm -> head product -> a token, as a decode step ends."""
    g = torch.Generator("cuda").manual_seed(17)
    normal = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    x = normal(12, 512).bfloat16()
    head = T.mx_quantize(normal(3001, 512) * 512 ** -0.5 * 4, "e2m1")
    _, y = T.residual_rms_norm_mx(x, None, None, 1e-5)
    logits = T.mx_linear(y, head, dtype=torch.float32)
    r = np.random.default_rng(18)
    check(logits, r.random(12), **settings(r, 12))
    check(T.mx_linear(y, head), r.random(12), **settings(r, 12))
    assert T.sample(torch.empty(0, 5, device="cuda"),
                    torch.empty(0, dtype=torch.float64, device="cuda")).shape == (0,)
