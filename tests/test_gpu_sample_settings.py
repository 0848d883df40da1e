"""Settings of filtered sampling that change while rows are drawn: a row's CTAs decide by the same
values, whichever they are."""
import numpy as np
import pytest
import torch

import tb_b200 as T
from test_gpu_sample_filters import check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,vocab", [(300, 5000), (300, 40000), (100, 128256)])
def test_settings_that_another_stream_writes(rows, vocab):
    """Any token of the row while they change; by what they are, once they stand."""
    r = np.random.default_rng(vocab)
    x = torch.from_numpy(r.standard_normal((rows, vocab)) * 3).float().cuda()
    u = r.random(rows)
    uniforms = torch.from_numpy(u).cuda()
    kinds = [dict(temperature=0.0, top_k=0, top_p=1.0, min_p=0.0),
             dict(temperature=1.0, top_k=0, top_p=0.9, min_p=0.0),
             dict(temperature=0.7, top_k=50, top_p=1.0, min_p=0.2),
             dict(temperature=1.3, top_k=900, top_p=0.5, min_p=0.0)]
    sets = [{k: torch.full((rows,), v, dtype=torch.int32 if k == "top_k" else torch.float32,
                           device="cuda") for k, v in kind.items()} for kind in kinds]
    live = {k: v.clone() for k, v in sets[0].items()}
    outs = [torch.full((rows,), -1, dtype=torch.int32, device="cuda") for _ in range(20)]
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    for i, out in enumerate(outs):
        T.sample(x, uniforms, **live, out=out)
        with torch.cuda.stream(side):
            for j in range(12):
                for k, v in live.items():
                    v.copy_(sets[(i + j) % len(sets)][k])
    torch.cuda.synchronize()
    for out in outs:
        assert ((out >= 0) & (out < vocab)).all()
    check(x, u, **{k: v.cpu().numpy() for k, v in live.items()}, rows=range(0, rows, 7))
