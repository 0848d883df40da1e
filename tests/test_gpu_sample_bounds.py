"""How near to a border filtered sampling may draw either token, and that it draws one.

A weight is a whole number of 2^-shift of the largest, shift = 62 less the bits that hold
vocab - 1 (at most 50; 43 at the largest vocabulary), so it is off by half of that, 2^-44, and by
less than 2^-49 of double's and the table's roundings.  Roundings of equal weights have one sign:
a running sum is off by up to n times that, n its weights, and u times the whole sum by as much."""
import numpy as np
import pytest
import torch

import mx_ref as R
import tb_b200 as T
from test_gpu_sample_filters import check, settings

pytestmark = pytest.mark.gpu


def most_off(vocab):
    """Of a running sum, the largest weight being 1."""
    shift = min(50, 62 - max(0, int(vocab - 1).bit_length()))
    return vocab * (2.0 ** -(shift + 1) + 2.0 ** -49)


def sampled(x, u, **kw):
    out = torch.full((x.shape[0],), -1, dtype=torch.int32, device="cuda")
    return T.sample(x, torch.from_numpy(np.asarray(u)).cuda(), out=out, **kw).cpu().numpy()


def kept_of(x, top_k=0, top_p=1.0, min_p=0.0, temperature=1.0):
    """(indices kept, in their order, their weights in 64 bits of mantissa)."""
    w = np.exp((x.astype(np.longdouble) - x.max()) / temperature)
    order = np.argsort(-x, kind="stable")
    if 0 < top_k < len(x):
        order = order[:top_k]
    sums = np.cumsum(w[order])
    if top_p < 1:
        order = order[:1 + int((sums[:-1] < top_p * sums[-1]).sum())]
    kept = np.sort(order[w[order] >= min_p])
    return kept, w[kept]


def check_near(x, u, got, **settings):
    """got are draws by the definition, but for what the sums are off; settings are rows'."""
    host, off = x.double().cpu().numpy(), most_off(x.shape[1])
    for i in range(len(u)):
        kept, w = kept_of(host[i], **{k: v[i] for k, v in settings.items()})
        sums = np.cumsum(w)
        at = int(np.searchsorted(kept, got[i]))
        assert at < len(kept) and kept[at] == got[i], (i, u[i], got[i])
        goal = u[i] * sums[-1]
        assert sums[at] - w[at] - 2 * off <= goal < sums[at] + 2 * off, (i, u[i], got[i])


@pytest.mark.parametrize("vocab", [1000, 40001, 262144, 300001, 376832])
@pytest.mark.parametrize("tail", [42.3, 43.9, 44.1, 45.0, 47.0])
def test_many_equal_weights_next_to_a_unit(vocab, tail):
    """One logit and a tail whose weights, 2^-tail, are rounded up, down or away."""
    x = torch.full((1, vocab), -tail * np.log(2.0), dtype=torch.float32, device="cuda")
    x[0, vocab // 3] = 0.0
    mass = vocab * 2.0 ** -tail
    u = np.concatenate([[0.0, mass / 7, mass / 3.1, 0.5],
                        1 - mass * np.array([0.6, 0.5, 0.3, 0.1]), [1 - 2.0 ** -53]])
    x = x.expand(len(u), vocab).contiguous()
    check_near(x, u, sampled(x, u))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("std", [0.3, 3.0])
def test_largest_vocabulary(std, dtype):
    """(Unlike weights' roundings have no sign in common: sums are off by some 2^-36.)"""
    r = np.random.default_rng(21)
    x = torch.from_numpy(r.standard_normal((12, 376832)) * std).to(dtype).cuda()
    check(x, r.random(12))
    for _ in range(3):
        check(x, r.random(12), **settings(r, 12))


@pytest.mark.parametrize("filters", [dict(), dict(top_p=0.9), dict(top_k=700), dict(min_p=0.01),
                                     dict(top_k=900, top_p=0.97), dict(top_p=0.999, min_p=1e-5)])
@pytest.mark.parametrize("rows,vocab", [(400, 777), (200, 9001), (30, 128256)])
def test_the_last_unit_of_a_sum_is_drawn(rows, vocab, filters):
    """u next to 1 aims at the last unit of the whole sum: told sums and searched ones agree to it,
    or a row would be left without a token."""
    r = np.random.default_rng(vocab)
    x = torch.from_numpy(r.standard_normal((rows, vocab)) * 2).float().cuda()
    u = np.where(np.arange(rows) % 4, 1 - 2.0 ** -53, 1 - 2.0 ** -40 * r.random(rows))
    f = np.float32
    s = dict(temperature=r.uniform(0.3, 3.0, rows).astype(f))
    s.update({k: np.full(rows, v, np.int32 if k == "top_k" else f) for k, v in filters.items()})
    got = sampled(x, u, **{k: torch.from_numpy(v).cuda() for k, v in s.items()})
    assert ((got >= 0) & (got < vocab)).all()
    check_near(x, u, got, **{k: v.astype(np.float64) if k != "top_k" else v for k, v in s.items()})
