"""Rows so many that their pieces of work pass 32 bits."""
import numpy as np
import pytest
import torch

import mx_ref as R
import tb_b200 as T

pytestmark = pytest.mark.gpu

PERIOD = 1021  # rows, then they come again


@pytest.mark.parametrize("swiglu", [False, True])
def test_more_pieces_than_an_int_counts(swiglu, cuda):
    """2^28 and some f32 rows of one column: 16 pieces each; 20 GB."""
    rows = 2 ** 28 + 300
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < 40 * 2 ** 30:
        pytest.skip("needs 40 GB")
    table = torch.from_numpy(np.random.default_rng(1).standard_normal((PERIOD, 1))).float().cuda()
    x = table.repeat(-(-rows // PERIOD), 1)[:rows]
    if swiglu:
        t = T.swiglu_mx(x, x, "e2m1")
        few = T.swiglu_mx(table, table, "e2m1")
    else:
        t = T.mx_quantize(x, "e2m1")
        few = T.mx_quantize(table, "e2m1")
        want, _ = R.quantised(table.double().cpu().numpy(), "e2m1")
        assert np.array_equal(T.mx_dequantize(few).double().cpu().numpy(), want)
    del x
    codes = few.codes[:, 0].contiguous()
    scales = few.scales[torch.from_numpy(R.scale_places(PERIOD, 1)[:, 0]).cuda()]
    step = PERIOD * 128 * 200  # whole periods, whole tiles
    for at in range(0, rows, step):
        n = min(step, rows - at)
        r = torch.arange(n, device="cuda") % PERIOD
        part = t.codes[at:at + n]
        assert torch.equal(part[:, 0], codes[r])
        assert not part[:, 1:].any()
        tiles = t.scales[at * 4:(at + -(-n // 128) * 128) * 4].view(-1, 32, 4, 4)
        held = tiles.permute(0, 2, 1, 3).reshape(-1, 4)
        assert torch.equal(held[:n, 0], scales[r])
        assert not held[:n, 1:].any() and not held[n:].any()
    del t, part, tiles, held
    torch.cuda.empty_cache()
