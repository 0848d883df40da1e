"""Argument checks of the rotary and 8-bit cache entry points, on the CPU:
refused calls return their TbError before any device work, empty ones TB_OK."""
import ctypes as C

import pytest

import tb_b200 as T

OK, ARG, SHAPE, DTYPE = 0, 8, 9, 10
FAKE = 0x10000  # an address that is checked but never read


def rotary(**kw):
    f = dict(dtype=T.F32, rows=2, n_q_heads=2, n_kv_heads=1, head_dim=64, rotary_dim=64,
             layout=T.ROTARY_HALF, q=FAKE, q_stride=128, k=FAKE, k_stride=64, q_out=FAKE,
             q_out_stride=128, k_out=FAKE, k_out_stride=64, positions=FAKE, freqs=FAKE, scale=1.0)
    f.update(kw)
    return T.Rotary(**f)


@pytest.mark.parametrize("fn", ["tb_b200_rotary", "tb_b200_qk_norm_rotary"])
@pytest.mark.parametrize("change,want", [
    (dict(rows=-1), SHAPE), (dict(rows=2 ** 31), SHAPE), (dict(n_q_heads=-1), SHAPE),
    (dict(head_dim=0), SHAPE), (dict(head_dim=513), SHAPE), (dict(rotary_dim=63), SHAPE),
    (dict(rotary_dim=66), SHAPE), (dict(rotary_dim=-2), SHAPE), (dict(dtype=T.F16), DTYPE),
    (dict(layout=2), ARG), (dict(q_stride=127), SHAPE), (dict(k_stride=63), SHAPE),
    (dict(q_out_stride=127), SHAPE), (dict(k_out_stride=0), SHAPE), (dict(q=None), ARG),
    (dict(k_out=None), ARG), (dict(positions=None), ARG), (dict(freqs=None), ARG),
    (dict(q_out_stride=256), ARG),  # in place with another stride
    (dict(rows=0), OK), (dict(n_q_heads=0, n_kv_heads=0), OK)])
def test_rotary_refusals(fn, change, want):
    t = rotary(**change)
    assert getattr(T.lib(), fn)(C.byref(t), None) == want
    assert getattr(T.lib(), fn)(None, None) == ARG


@pytest.mark.parametrize("r,change,want", [
    (0, {}, SHAPE), (3, {}, SHAPE), (514, {}, SHAPE), (64, dict(kind=5), ARG),
    (64, dict(kind=-1), ARG), (64, dict(theta=0.0), ARG), (64, dict(theta=float("nan")), ARG),
    (64, dict(kind=1, factor=0.0), ARG), (2, dict(kind=2, factor=2.0), SHAPE),
    (64, dict(kind=3, factor=2.0, trained=0.0, low=1.0, high=4.0), ARG),
    (64, dict(kind=3, factor=2.0, trained=8.0, low=4.0, high=4.0), ARG),
    (64, dict(kind=4, factor=2.0, trained=8.0, low=0.0, high=4.0), ARG),
    (64, dict(kind=4, theta=1.0, factor=2.0, trained=8.0, low=1.0, high=4.0), ARG)])
def test_rotary_freqs_refusals(r, change, want):
    f = dict(kind=0, theta=1e4, factor=1.0)
    f.update(change)
    s = T.RotaryScaling(**f)
    assert T.lib().tb_b200_rotary_freqs(r, C.byref(s), FAKE, None) == want
    assert T.lib().tb_b200_rotary_freqs(64, None, FAKE, None) == ARG
    assert T.lib().tb_b200_rotary_freqs(64, C.byref(s), None, None) == ARG


def kv8(**kw):
    f = dict(format=T.KV_INT8, page=64, n_kv_heads=2, head_dim=64, n_pages=4, k=FAKE, v=FAKE,
             k_scale=FAKE, v_scale=FAKE)
    f.update(kw)
    return T.Kv8(**f)


def batch(**kw):
    f = dict(n_seqs=2, rows=3, row_start=FAKE, lengths=FAKE, page_table=FAKE, table_width=2,
             table_stride=2)
    f.update(kw)
    return T.Kv8Batch(**f)


def attention(**kw):
    f = dict(dtype=T.BF16, n_heads=4, q=FAKE, q_stride=256, out=2 * FAKE, out_stride=256,
             scale=0.125, max_rows=2, max_len=128, workspace=FAKE, workspace_bytes=1 << 40)
    f.update(kw)
    return T.Kv8Attention(**f)


CACHES = [(dict(format=4), DTYPE), (dict(page=48), SHAPE), (dict(page=256), SHAPE),
          (dict(page=0), SHAPE), (dict(n_kv_heads=0), SHAPE), (dict(head_dim=8), SHAPE),
          (dict(head_dim=72), SHAPE), (dict(head_dim=272), SHAPE), (dict(n_pages=-1), SHAPE),
          (dict(n_pages=0), SHAPE), (dict(n_pages=2 ** 31), SHAPE), (dict(k=None), ARG),
          (dict(v_scale=None), ARG), (dict(v=FAKE + 8), ARG)]
BATCHES = [(dict(n_seqs=-1), SHAPE), (dict(rows=-1), SHAPE), (dict(table_stride=1), SHAPE),
           (dict(table_width=-1), SHAPE), (dict(row_start=None), ARG), (dict(lengths=None), ARG),
           (dict(page_table=None), ARG), (dict(n_seqs=65536), SHAPE), (dict(rows=2 ** 31), SHAPE),
           (dict(rows=0), OK), (dict(n_seqs=0), OK)]


@pytest.mark.parametrize("c,want", CACHES)
def test_cache_refusals(c, want):
    L, k, b, a = T.lib(), kv8(**c), batch(), attention()
    assert L.tb_b200_kv8_append(C.byref(k), C.byref(b), T.F32, FAKE, 128, FAKE, 128, None) == want
    assert L.tb_b200_kv8_attention(C.byref(k), C.byref(b), C.byref(a), None) == want


@pytest.mark.parametrize("bt,want", BATCHES)
def test_batch_refusals(bt, want):
    L, k, b, a = T.lib(), kv8(), batch(**bt), attention()
    assert L.tb_b200_kv8_append(C.byref(k), C.byref(b), T.F32, FAKE, 128, FAKE, 128, None) == want
    assert L.tb_b200_kv8_attention(C.byref(k), C.byref(b), C.byref(a), None) == want


def test_append_refusals():
    L, k, b = T.lib(), kv8(), batch()

    def call(dtype=T.F32, kp=FAKE, ks=128, vp=FAKE, vs=128, c=k, bt=b):
        return L.tb_b200_kv8_append(c and C.byref(c), bt and C.byref(bt), dtype, kp, ks, vp, vs,
                                    None)
    assert call(dtype=T.F16) == DTYPE
    assert call(ks=127) == SHAPE and call(vs=0) == SHAPE
    assert call(kp=None) == ARG and call(vp=None) == ARG
    assert call(c=None) == ARG and call(bt=None) == ARG


@pytest.mark.parametrize("change,want", [
    (dict(dtype=T.F16), DTYPE), (dict(n_heads=0), SHAPE), (dict(n_heads=3), SHAPE),
    (dict(window=-1), SHAPE), (dict(max_rows=-1), SHAPE), (dict(max_len=-1), SHAPE),
    (dict(max_len=2 ** 30 + 1), SHAPE),
    (dict(q_stride=255), SHAPE), (dict(out_stride=255), SHAPE), (dict(q=None), ARG),
    (dict(out=None), ARG), (dict(out=FAKE), ARG)])
def test_attention_refusals(change, want):
    L, k, b, a = T.lib(), kv8(), batch(), attention(**change)
    assert L.tb_b200_kv8_attention(C.byref(k), C.byref(b), C.byref(a), None) == want
    assert L.tb_b200_kv8_attention(C.byref(k), C.byref(b), None, None) == ARG
    n = C.c_size_t()
    a = attention()
    assert L.tb_b200_kv8_attention_workspace(None, C.byref(b), C.byref(a), C.byref(n)) == ARG


def test_struct_sizes():
    assert C.sizeof(T.Rotary) == 152 and C.sizeof(T.RotaryScaling) == 48
    assert C.sizeof(T.Kv8) == 56 and C.sizeof(T.Kv8Batch) == 56
    assert C.sizeof(T.Kv8Attention) == 80


def test_python_refuses_host_tensors():
    import torch
    x = torch.zeros(2, 1, 64)
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError):
        T.rotary(x, x, i, torch.zeros(32, dtype=torch.float64))
    with pytest.raises(ValueError):
        T.Kv8Cache(torch.zeros(1, 1, 16, 64, dtype=torch.int8),
                   torch.zeros(1, 1, 16, 64, dtype=torch.int8), torch.zeros(1, 1),
                   torch.zeros(1, 1))


@pytest.mark.parametrize("hq,hkv", [(2 ** 30 - 1, 2 ** 30 - 1), (2 ** 30 - 1, 1), (1, 2 ** 30 - 1),
                                    (2 ** 31 - 1, 0), (2 ** 30, 0)])
def test_rotary_heads_that_an_index_does_not_hold(hq, hkv):
    """The kernel counts a row's heads, Q's and K's, in an int, a pass beyond the last."""
    t = rotary(n_q_heads=hq, n_kv_heads=hkv, head_dim=1, rotary_dim=0, rows=1)
    assert T.lib().tb_b200_rotary(C.byref(t), None) == SHAPE
    assert T.lib().tb_b200_qk_norm_rotary(C.byref(t), None) == SHAPE
