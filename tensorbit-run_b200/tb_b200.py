"""Python binding of libtb_b200.so over its C ABI (include/tb_b200.h,
include/tb_backend.h), for tests, benchmarks and Python hosts.

Device buffers are torch CUDA tensors (torch provides allocation, streams
and torch.distributed; the arithmetic is the library's sm_100a kernels).
Every call goes through ctypes to the C entry point of the same name and
raises ``TbError`` on a nonzero TbError code.  There is no fallback path:
if the library is missing, ``lib()`` raises.

Dtype codes follow TbDtype (F32 = 0, BF16 = 2).
"""
from __future__ import annotations

import ctypes as C
import os
import subprocess

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(HERE, "lib", "libtb_b200.so")

F32, F16, BF16, I32 = 0, 1, 2, 4
DEVICE_CPU, DEVICE_CUDA = 0, 1
FLAG_TOKEN_RANGE = 0x1
FLAG_WAIT_TIMEOUT = 0x2

# TbOpType values (include/tb_backend.h)
OP = dict(SPARSE_LINEAR=0, DENSE_LINEAR=1, RMS_NORM=2, LAYER_NORM=3, GELU=4, SILU=5, SOFTMAX=6,
          ATTENTION_QKV=7, SCALED_DOT_PRODUCT=8, ROPE=9, RESIDUAL_ADD=10, EMBEDDING=11, CONV2D=12,
          RESIDUAL_RMS_NORM=13, SWIGLU=14, ARGMAX=15, ROPE_ROWS=16, LAYER_CHAIN=17, COUNT=18)

ERRORS = {0: "ok", 7: "out of memory", 8: "invalid argument", 9: "invalid shape",
          10: "unsupported dtype", 14: "backend not found", 16: "device error"}


class TbError(RuntimeError):
    def __init__(self, code: int, what: str, detail: str = ""):
        self.code = code
        msg = f"{what}: TbError {code} ({ERRORS.get(code, 'error')})"
        super().__init__(msg + (f": {detail}" if detail else ""))


class TbTensor(C.Structure):
    """ABI image of TbTensor (include/tb_types.h)."""
    _fields_ = [("data", C.c_void_p), ("shape", C.c_size_t * 8), ("rank", C.c_uint8),
                ("dtype", C.c_int), ("device", C.c_int), ("owns_data", C.c_bool)]


class LayerChain(C.Structure):
    """ABI image of TbB200LayerChain (include/tb_b200.h)."""
    _fields_ = [("dtype", C.c_int), ("rows", C.c_int64),
                ("hidden", C.c_int64), ("x", C.c_void_p), ("residual", C.c_void_p),
                ("norm_weight", C.c_void_p), ("h_out", C.c_void_p), ("y", C.c_void_p),
                ("eps", C.c_float),
                ("n_q_heads", C.c_int), ("n_kv_heads", C.c_int), ("head_dim", C.c_int),
                ("q", C.c_void_p), ("k", C.c_void_p), ("positions", C.c_void_p),
                ("theta", C.c_float), ("rope_table", C.c_void_p),
                ("rope_table_positions", C.c_int),
                ("intermediate", C.c_int64), ("gate", C.c_void_p), ("up", C.c_void_p),
                ("act_out", C.c_void_p)]


class RopeRowsParams(C.Structure):
    _fields_ = [("positions", C.c_void_p), ("theta", C.c_float), ("head_dim", C.c_int),
                ("max_position", C.c_int)]


class LayerChainParams(C.Structure):
    _fields_ = [("eps", C.c_float), ("positions", C.c_void_p), ("theta", C.c_float),
                ("head_dim", C.c_int), ("max_position", C.c_int)]


_lib = None
vp, i64, i32, f32 = C.c_void_p, C.c_int64, C.c_int, C.c_float
P = C.POINTER

INT8, INT4 = 7, 8  # TbDtype codes of quantized weights
ATTN_REFERENCE, ATTN_STANDARD = 0, 1
FLAG_POSITION_RANGE = 0x4
FLAG_PAGE_RANGE = 0x8
FLAG_NONFINITE = 0x10
ROTARY_INTERLEAVED, ROTARY_HALF = 0, 1
ROTARY_SCALING = {"none": 0, "linear": 1, "ntk": 2, "bands": 3, "yarn": 4}
KV_INT8, KV_E4M3 = 7, 0x43
MX_FORMATS = {"e4m3": 0x43, "e2m1": 0x21}
PROJECTIONS = ("q", "k", "v", "o", "gate", "up", "down")


class Weight(C.Structure):  # TbB200Weight
    _fields_ = [("data", vp), ("dtype", i32), ("rows", i64), ("cols", i64), ("mask", vp),
                ("scales", vp), ("n_scales", i64), ("group_size", C.c_uint32)]


class RunnerLayer(C.Structure):  # TbB200RunnerLayer
    _fields_ = [(n, Weight) for n in PROJECTIONS] + [("input_norm", vp), ("post_norm", vp)]


class RunnerDesc(C.Structure):  # TbB200RunnerDesc
    _fields_ = [(n, i32) for n in ("hidden", "n_heads", "n_kv_heads", "head_dim", "intermediate",
                                   "vocab", "max_seq", "layers")] + [
        ("norm_eps", f32), ("rope_theta", f32), ("attention", i32), ("use_graph", i32),
        ("embed", Weight), ("final_norm", vp), ("lm_head", Weight), ("layer", P(RunnerLayer))]

class TbmConfig(C.Structure):  # TbB200TbmConfig
    _fields_ = [("architecture", C.c_char * 64)] + [
        (n, i32) for n in ("hidden_size", "num_heads", "num_kv_heads", "intermediate_size",
                           "vocab_size", "max_seq_len", "num_layers")] + [
        ("norm_eps", f32), ("rope_theta", f32), ("head_dim", i32)]


class TbmTensor(C.Structure):  # TbB200TbmTensor
    _fields_ = [("name", C.c_char * 128), ("shape", i64 * 2), ("dtype", i32),
                ("nm_n", C.c_uint32), ("nm_m", C.c_uint32), ("num_weights", i64),
                ("num_mask_bytes", i64), ("scale_count", i64), ("group_size", C.c_uint32),
                ("weights", vp), ("mask", vp), ("scales", vp), ("weight_bytes", i64)]


class Rotary(C.Structure):  # TbB200Rotary
    _fields_ = [("dtype", i32), ("rows", i64), ("n_q_heads", i32), ("n_kv_heads", i32),
                ("head_dim", i32), ("rotary_dim", i32), ("layout", i32), ("q", vp),
                ("q_stride", i64), ("k", vp), ("k_stride", i64), ("q_out", vp),
                ("q_out_stride", i64), ("k_out", vp), ("k_out_stride", i64), ("positions", vp),
                ("freqs", vp), ("scale", f32), ("q_weight", vp), ("k_weight", vp), ("eps", f32)]


class RotaryScaling(C.Structure):  # TbB200RotaryScaling
    _fields_ = [("kind", i32)] + [(n, C.c_double) for n in ("theta", "factor", "trained", "low",
                                                            "high")]


class Kv8(C.Structure):  # TbB200Kv8
    _fields_ = [("format", i32), ("page", i32), ("n_kv_heads", i32), ("head_dim", i32),
                ("n_pages", i64), ("k", vp), ("v", vp), ("k_scale", vp), ("v_scale", vp)]


class Kv8Batch(C.Structure):  # TbB200Kv8Batch
    _fields_ = [("n_seqs", i32), ("rows", i64), ("row_start", vp), ("lengths", vp),
                ("page_table", vp), ("table_width", i32), ("table_stride", i64)]


class Kv8Attention(C.Structure):  # TbB200Kv8Attention
    _fields_ = [("dtype", i32), ("n_heads", i32), ("q", vp), ("q_stride", i64), ("out", vp),
                ("out_stride", i64), ("lse", vp), ("scale", f32), ("window", i32),
                ("max_rows", i32), ("max_len", i32), ("workspace", vp),
                ("workspace_bytes", C.c_size_t)]


class Mx(C.Structure):  # TbB200Mx
    _fields_ = [("format", i32), ("rows", i64), ("cols", i64), ("codes", vp), ("scales", vp)]


class Sample(C.Structure):  # TbB200Sample
    _fields_ = [("dtype", i32), ("rows", i64), ("vocab", i64), ("logits", vp), ("stride", i64),
                ("temperature", vp), ("top_k", vp), ("top_p", vp), ("min_p", vp),
                ("uniforms", vp), ("out", vp)]


# name -> (restype, argtypes); every entry point of include/tb_b200.h and tb_backend.h.
SIGNATURES = {
    "tb_b200_version": (i32, []),
    "tb_b200_last_error": (C.c_char_p, []),
    "tb_b200_launch_count": (C.c_ulonglong, []),
    "tb_b200_device_count": (i32, [P(i32)]),
    "tb_b200_set_device": (i32, [i32]),
    "tb_b200_get_device": (i32, [P(i32)]),
    "tb_b200_malloc": (i32, [P(vp), C.c_size_t]),
    "tb_b200_free": (i32, [vp]),
    "tb_b200_malloc_host": (i32, [P(vp), C.c_size_t]),
    "tb_b200_free_host": (i32, [vp]),
    "tb_b200_memcpy_h2d": (i32, [vp, vp, C.c_size_t, vp]),
    "tb_b200_memcpy_d2h": (i32, [vp, vp, C.c_size_t, vp]),
    "tb_b200_memcpy_d2d": (i32, [vp, vp, C.c_size_t, vp]),
    "tb_b200_memset": (i32, [vp, i32, C.c_size_t, vp]),
    "tb_b200_set_stream": (i32, [vp]),
    "tb_b200_get_stream": (vp, []),
    "tb_b200_stream_sync": (i32, [vp]),
    "tb_b200_sync": (i32, []),
    "tb_b200_stage_h2d": (i32, [vp, C.c_size_t, P(vp), vp]),
    "tb_b200_stage_release": (i32, [vp, vp]),
    "tb_b200_is_device_ptr": (i32, [vp, P(i32)]),
    "tb_b200_check_status": (i32, [vp, P(C.c_uint)]),
    "tb_b200_residual_rms_norm": (i32, [i32, i64, i64, vp, vp, vp, vp, vp, f32, vp]),
    "tb_b200_rms_norm": (i32, [i32, i64, i64, vp, vp, vp, f32, vp]),
    "tb_b200_residual_add": (i32, [i32, i64, vp, vp, vp, vp]),
    "tb_b200_silu": (i32, [i32, i64, vp, vp, vp]),
    "tb_b200_gelu": (i32, [i32, i64, vp, vp, vp]),
    "tb_b200_swiglu": (i32, [i32, i64, vp, vp, vp, vp]),
    "tb_b200_rope_table": (i32, [f32, i32, i32, vp, vp]),
    "tb_b200_rope_rows": (i32, [i32, i64, i32, i32, i32, vp, vp, vp, f32, vp, i32, vp]),
    "tb_b200_rope": (i32, [i32, i32, i32, i32, vp, vp, i32, f32, vp]),
    "tb_b200_softmax": (i32, [i32, i64, i64, vp, vp, vp, vp]),
    "tb_b200_sample_temperature": (i32, [i64, i64, vp, f32, vp, vp, vp]),
    "tb_b200_dequant": (i32, [i32, i64, vp, vp, i64, C.c_uint32, i32, vp, vp]),
    "tb_b200_sparse_linear": (i32, [i64, i64, vp, vp, vp, vp, vp, i32, i32, vp]),
    "tb_b200_dense_linear": (i32, [i64, i64, vp, vp, vp, vp, vp]),
    "tb_b200_argmax": (i32, [i32, i64, i64, vp, vp, vp]),
    "tb_b200_embedding": (i32, [i32, i64, i64, i64, vp, vp, vp, vp]),
    "tb_b200_embedding_host_ids": (i32, [i32, i64, i64, i64, vp, vp, vp, vp]),
    "tb_b200_embedding_host_ids_static": (i32, [i32, i64, i64, i64, vp, vp, vp, vp]),
    "tb_b200_layer_chain": (i32, [P(LayerChain), vp]),
    "tb_b200_sparse24_pack": (i32, [i64, i64, vp, vp, vp, vp, vp, vp]),
    "tb_b200_sparse24_linear": (i32, [i64, i64, vp, vp, vp, vp, vp, vp]),
    "tb_b200_decode_attention": (i32, [i32, i32, i32, i32, i32, vp, vp, vp, vp, vp, vp, vp, vp]),
    "tb_b200_rotary_freqs": (i32, [i32, P(RotaryScaling), vp, vp]),
    "tb_b200_rotary": (i32, [P(Rotary), vp]),
    "tb_b200_qk_norm_rotary": (i32, [P(Rotary), vp]),
    "tb_b200_kv8_append": (i32, [P(Kv8), P(Kv8Batch), i32, vp, i64, vp, i64, vp]),
    "tb_b200_kv8_attention": (i32, [P(Kv8), P(Kv8Batch), P(Kv8Attention), vp]),
    "tb_b200_kv8_attention_workspace": (i32, [P(Kv8), P(Kv8Batch), P(Kv8Attention),
                                              P(C.c_size_t)]),
    "tb_b200_mx_bytes": (i32, [i32, i64, i64, P(C.c_size_t), P(C.c_size_t)]),
    "tb_b200_mx_quantize": (i32, [i32, vp, i64, P(Mx), vp]),
    "tb_b200_mx_dequantize": (i32, [P(Mx), i32, vp, i64, vp]),
    "tb_b200_residual_rms_norm_mx": (i32, [i32, vp, vp, vp, vp, P(Mx), f32, vp]),
    "tb_b200_swiglu_mx": (i32, [i32, vp, i64, vp, i64, P(Mx), vp]),
    "tb_b200_mx_linear": (i32, [P(Mx), P(Mx), vp, i32, vp, i64, vp]),
    "tb_b200_sample": (i32, [P(Sample), vp]),
    "tb_b200_runner_create": (i32, [P(RunnerDesc), P(vp)]),
    "tb_b200_runner_forward": (i32, [vp, C.c_int32, P(vp)]),
    "tb_b200_runner_logits": (i32, [vp, vp]),
    "tb_b200_runner_reset": (i32, [vp]),
    "tb_b200_runner_position": (i32, [vp, P(i32)]),
    "tb_b200_runner_stream": (i32, [vp, P(vp)]),
    "tb_b200_runner_launches_per_token": (i32, [vp, P(i32)]),
    "tb_b200_runner_destroy": (i32, [vp]),
    "tb_b200_tbm_load": (i32, [C.c_char_p, vp, P(vp)]),
    "tb_b200_tbm_config": (i32, [vp, P(TbmConfig)]),
    "tb_b200_tbm_count": (i32, [vp, P(i32)]),
    "tb_b200_tbm_find": (i32, [vp, C.c_char_p, P(i32)]),
    "tb_b200_tbm_tensor": (i32, [vp, i32, P(TbmTensor)]),
    "tb_b200_tbm_runner_desc": (i32, [vp, i32, i32, P(RunnerDesc), P(RunnerLayer), i32]),
    "tb_b200_tbm_free": (i32, [vp]),
    "tb_b200_partition": (i32, [i64, i32, i32, P(i64), P(i64)]),
    "tb_b200_shard_plan": (i32, [i64, i64, i32, i32, vp, vp, vp, vp, vp, vp, vp, P(i64)]),
    "tb_b200_comm_unique_id": (i32, [vp]),
    "tb_b200_comm_init": (i32, [i32, i32, vp, i32]),
    "tb_b200_comm_destroy": (i32, []),
    "tb_b200_comm_info": (i32, [P(i32), P(i32)]),
    "tb_b200_comm_wait": (i32, [vp]),
    "tb_b200_selftest_wait": (i32, [i32, C.c_uint32, vp]),
    "tb_b200_comm_window_alloc": (i32, [C.c_size_t, P(vp)]),
    "tb_b200_comm_window_free": (i32, [vp]),
    "tb_b200_embedding_sharded_window": (i32, [i32, i64, i64, i64, vp, vp, vp, vp]),
    "tb_b200_embedding_sharded": (i32, [i32, i64, i64, i64, vp, vp, vp, vp]),
    "tb_b200_embedding_sharded_p2p": (i32, [i32, i64, i64, i64, vp, P(vp), i32, vp, vp]),
    "tb_b200_p2p_export": (i32, [vp, vp, P(i64)]),
    "tb_b200_p2p_import": (i32, [vp, i64, P(vp)]),
    "tb_b200_p2p_close": (i32, [vp, i64]),
    # registry (include/tb_backend.h)
    "tb_backend_register": (i32, [vp]),
    "tb_backend_register_device": (i32, [vp, i32]),
    "tb_backend_get_best": (vp, [i32]),
    "tb_backend_get_best_device": (vp, [i32, i32]),
    "tb_backend_count": (i32, []),
    "tb_backend_get": (vp, [i32]),
    "tb_backend_reset": (None, []),
    "tb_backend_b200_init": (i32, []),
    "tb_dispatch_sparse_linear": (i32, [vp, vp, vp, vp, vp]),
    "tb_dispatch_dense_linear": (i32, [vp, vp, vp, vp]),
    "tb_dispatch_rms_norm": (i32, [vp, vp, vp, f32]),
    "tb_dispatch_layer_norm": (i32, [vp, vp, vp, vp, f32]),
    "tb_dispatch_gelu": (i32, [vp, vp]),
    "tb_dispatch_silu": (i32, [vp, vp]),
    "tb_dispatch_softmax": (i32, [vp, vp, vp]),
    "tb_dispatch_attention_qkv": (i32, [vp] * 10 + [i32, i32, i32]),
    "tb_dispatch_scaled_dot_product": (i32, [vp, vp, vp, vp, vp, f32, C.c_bool]),
    "tb_dispatch_rope": (i32, [vp, vp, i32, f32, i32]),
    "tb_dispatch_residual_add": (i32, [vp, vp, vp]),
    "tb_dispatch_embedding": (i32, [vp, vp, i32, vp]),
    "tb_dispatch_conv2d": (i32, [vp, vp, vp, vp, i32, i32]),
    "tb_dispatch_residual_rms_norm": (i32, [vp, vp, vp, vp, vp, f32]),
    "tb_dispatch_swiglu": (i32, [vp, vp, vp]),
    "tb_dispatch_argmax": (i32, [vp, vp]),
    "tb_dispatch_rope_rows": (i32, [vp, vp, vp, f32, i32, i32]),
    "tb_dispatch_layer_chain": (i32, [vp] * 10 + [P(LayerChainParams)]),
}


def build() -> None:
    """Compile lib/libtb_b200.so (nvcc, sm_100a)."""
    out = subprocess.run(["make", "-C", HERE, "-j8"], capture_output=True, text=True)
    if out.returncode != 0:
        raise RuntimeError("libtb_b200 build failed:\n" + out.stdout[-4000:] + out.stderr[-4000:])


def lib() -> C.CDLL:
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise RuntimeError(f"{LIB_PATH} is not built (run __graft_entry__.build())")
        L = C.CDLL(LIB_PATH)
        for name, (res, args) in SIGNATURES.items():
            fn = getattr(L, name)
            fn.restype = res
            fn.argtypes = args
        _lib = L
    return _lib


def last_error() -> str:
    s = lib().tb_b200_last_error()
    return s.decode() if s else ""


def check(rc: int, what: str) -> None:
    if rc != 0:
        raise TbError(rc, what, last_error())


# ------------------------------------------------------------- torch glue
def _torch():
    import torch
    return torch


def dtype_code(t) -> int:
    torch = _torch()
    if t.dtype == torch.float32:
        return F32
    if t.dtype == torch.bfloat16:
        return BF16
    if t.dtype == torch.int32:
        return I32
    raise TypeError(f"unsupported dtype {t.dtype}")


def ptr(t):
    return None if t is None else C.c_void_p(t.data_ptr())


def cur_stream():
    torch = _torch()
    return C.c_void_p(torch.cuda.current_stream().cuda_stream)


def _dev(*ts):
    for t in ts:
        if t is not None and not (t.is_cuda and t.is_contiguous()):
            raise ValueError("expected contiguous CUDA tensors")


def residual_rms_norm(x, residual, weight, eps, h_out=None, y=None, stream=None):
    torch = _torch()
    y = torch.empty_like(x) if y is None else y
    _dev(x, residual, weight, h_out, y)
    rows, cols = (x.numel() // x.shape[-1], x.shape[-1]) if x.dim() else (1, 1)
    check(lib().tb_b200_residual_rms_norm(dtype_code(x), rows, cols, ptr(x), ptr(residual),
                                          ptr(weight), ptr(h_out), ptr(y), eps,
                                          stream or cur_stream()), "residual_rms_norm")
    return h_out, y


def rms_norm(x, weight, eps, y=None, stream=None):
    torch = _torch()
    y = torch.empty_like(x) if y is None else y
    _dev(x, weight, y)
    rows, cols = x.numel() // x.shape[-1], x.shape[-1]
    check(lib().tb_b200_rms_norm(dtype_code(x), rows, cols, ptr(x), ptr(weight), ptr(y), eps,
                                 stream or cur_stream()), "rms_norm")
    return y


def residual_add(x, residual, y=None, stream=None):
    torch = _torch()
    y = torch.empty_like(x) if y is None else y
    _dev(x, residual, y)
    check(lib().tb_b200_residual_add(dtype_code(x), x.numel(), ptr(x), ptr(residual), ptr(y),
                                     stream or cur_stream()), "residual_add")
    return y


def silu(x, y=None, stream=None):
    torch = _torch()
    y = torch.empty_like(x) if y is None else y
    _dev(x, y)
    check(lib().tb_b200_silu(dtype_code(x), x.numel(), ptr(x), ptr(y), stream or cur_stream()),
          "silu")
    return y


def gelu(x, y=None, stream=None):
    torch = _torch()
    y = torch.empty_like(x) if y is None else y
    _dev(x, y)
    check(lib().tb_b200_gelu(dtype_code(x), x.numel(), ptr(x), ptr(y), stream or cur_stream()),
          "gelu")
    return y


def swiglu(gate, up, out=None, stream=None):
    torch = _torch()
    out = torch.empty_like(gate) if out is None else out
    _dev(gate, up, out)
    check(lib().tb_b200_swiglu(dtype_code(gate), gate.numel(), ptr(gate), ptr(up), ptr(out),
                               stream or cur_stream()), "swiglu")
    return out


def rope_table(theta, head_dim, n_positions, device=None):
    torch = _torch()
    t = torch.empty((n_positions, head_dim), dtype=torch.float32,
                    device=device or torch.cuda.current_device())
    check(lib().tb_b200_rope_table(theta, head_dim, n_positions, ptr(t), cur_stream()),
          "rope_table")
    return t


def rope_rows(q, k, positions, theta, table=None, stream=None):
    """In place on q [R, Hq, d] and k [R, Hkv, d]; positions int32 [R] on the device."""
    _dev(q, k, positions, table)
    rows, hq, d = q.shape
    hkv = k.shape[1]
    check(lib().tb_b200_rope_rows(dtype_code(q), rows, hq, hkv, d, ptr(q), ptr(k), ptr(positions),
                                  theta, ptr(table), 0 if table is None else table.shape[0],
                                  stream or cur_stream()), "rope_rows")
    return q, k


def rope(q, k, position, theta, stream=None):
    """Single token: q [Hq, d], k [Hkv, d], in place."""
    _dev(q, k)
    check(lib().tb_b200_rope(dtype_code(q), q.shape[0], k.shape[0], q.shape[-1], ptr(q), ptr(k),
                             position, theta, stream or cur_stream()), "rope")
    return q, k


def softmax(x, mask=None, y=None, stream=None):
    torch = _torch()
    y = torch.empty_like(x) if y is None else y
    _dev(x, mask, y)
    rows, cols = x.numel() // x.shape[-1], x.shape[-1]
    check(lib().tb_b200_softmax(dtype_code(x), rows, cols, ptr(x), ptr(mask), ptr(y),
                                stream or cur_stream()), "softmax")
    return y


def argmax(x, out=None, stream=None):
    torch = _torch()
    rows, cols = x.numel() // x.shape[-1], x.shape[-1]
    out = torch.empty(rows, dtype=torch.int32, device=x.device) if out is None else out
    _dev(x, out)
    check(lib().tb_b200_argmax(dtype_code(x), rows, cols, ptr(x), ptr(out),
                               stream or cur_stream()), "argmax")
    return out


def sample_temperature(logits, temperature, uniforms, out=None, stream=None):
    """Index drawn per row of f32 logits at the given uniform (float64 device
    tensor, one per row), as the reference's sample_temperature draws it."""
    torch = _torch()
    rows, cols = logits.numel() // logits.shape[-1], logits.shape[-1]
    out = torch.empty(rows, dtype=torch.int32, device=logits.device) if out is None else out
    _dev(logits, out)
    u = None if uniforms is None else ptr(uniforms)
    check(lib().tb_b200_sample_temperature(rows, cols, ptr(logits), temperature, u, ptr(out),
                                           stream or cur_stream()), "sample_temperature")
    return out


def dequant(src_dtype, n, q, scales, group_size, out_dtype=F32, out=None, stream=None):
    """n INT4 (src_dtype 8) / INT8 (7) weights in the uint8 device tensor q
    to f32 or bf16 with per-group f32 scales (Model::get_weight_fp32)."""
    torch = _torch()
    if out is None:
        dt = torch.float32 if out_dtype == F32 else torch.bfloat16
        out = torch.empty(n, dtype=dt, device=q.device)
    _dev(q, out)
    check(lib().tb_b200_dequant(src_dtype, n, ptr(q), ptr(scales) if scales is not None else None,
                                0 if scales is None else scales.numel(), group_size, out_dtype,
                                ptr(out), stream or cur_stream()), "dequant")
    return out


def linear(x, w, mask=None, bias=None, nm_n=2, nm_m=4, y=None, stream=None):
    """y = W x (+ bias) for an f32 vector x: N:M-masked when `mask` (uint8,
    one byte per M-group of a row) is given, else dense."""
    torch = _torch()
    out_f, in_f = w.shape
    y = torch.empty(out_f, dtype=torch.float32, device=w.device) if y is None else y
    _dev(x, w, y)
    b = ptr(bias) if bias is not None else None
    if mask is not None:
        rc = lib().tb_b200_sparse_linear(out_f, in_f, ptr(x), ptr(w), ptr(mask), b, ptr(y), nm_n,
                                         nm_m, stream or cur_stream())
    else:
        rc = lib().tb_b200_dense_linear(out_f, in_f, ptr(x), ptr(w), b, ptr(y),
                                        stream or cur_stream())
    check(rc, "linear")
    return y


def sparse24_pack(w, mask, stream=None):
    """Pack a 2:4-masked f32 [out, in] weight: (vals float32 [out, P, 4],
    idx uint8 [out, S], packable) with P = ceil((in / 4) / 2) and S = P
    rounded up to a multiple of 128."""
    torch = _torch()
    out_f, in_f = w.shape
    pairs = (in_f // 4 + 1) // 2
    vals = torch.empty((out_f, pairs, 4), dtype=torch.float32, device=w.device)
    idx = torch.empty((out_f, (pairs + 127) // 128 * 128), dtype=torch.uint8, device=w.device)
    flag = torch.zeros(1, dtype=torch.int32, device=w.device)
    _dev(w, mask)
    check(lib().tb_b200_sparse24_pack(out_f, in_f, ptr(w), ptr(mask), ptr(vals), ptr(idx),
                                      ptr(flag), stream or cur_stream()), "sparse24_pack")
    return vals, idx, int(flag.item()) == 0


def sparse24_linear(x, vals, idx, in_features, bias=None, y=None, stream=None):
    torch = _torch()
    out_f = vals.shape[0]
    y = torch.empty(out_f, dtype=torch.float32, device=x.device) if y is None else y
    _dev(x, vals, idx, y)
    check(lib().tb_b200_sparse24_linear(out_f, in_features, ptr(x), ptr(vals), ptr(idx),
                                        ptr(bias) if bias is not None else None, ptr(y),
                                        stream or cur_stream()), "sparse24_linear")
    return y


def embedding(ids, table, y=None, stream=None):
    torch = _torch()
    n = ids.numel()
    y = torch.empty((n, table.shape[1]), dtype=table.dtype, device=table.device) if y is None else y
    _dev(ids, table, y)
    check(lib().tb_b200_embedding(dtype_code(table), n, table.shape[1], table.shape[0], ptr(ids),
                                  ptr(table), ptr(y), stream or cur_stream()), "embedding")
    return y


def check_status(stream=None):
    flags = C.c_uint(0)
    rc = lib().tb_b200_check_status(stream or cur_stream(), C.byref(flags))
    return rc, flags.value


def layer_chain(chain: LayerChain, stream=None):
    check(lib().tb_b200_layer_chain(C.byref(chain), stream or cur_stream()), "layer_chain")


def make_chain(x=None, residual=None, norm_weight=None, h_out=None, y=None, eps=1e-5, q=None,
               k=None, positions=None, theta=10000.0, table=None, gate=None, up=None,
               act_out=None) -> LayerChain:
    c = LayerChain()
    ref = next(t for t in (x, q, gate) if t is not None)
    c.dtype = dtype_code(ref)
    c.rows = ref.shape[0]
    if x is not None:
        c.hidden, c.x, c.residual = x.shape[-1], ptr(x), ptr(residual)
        c.norm_weight, c.h_out, c.y, c.eps = ptr(norm_weight), ptr(h_out), ptr(y), eps
    if q is not None:
        c.n_q_heads, c.n_kv_heads, c.head_dim = q.shape[1], k.shape[1], q.shape[2]
        c.q, c.k, c.positions, c.theta = ptr(q), ptr(k), ptr(positions), theta
        c.rope_table = ptr(table)
        c.rope_table_positions = 0 if table is None else table.shape[0]
    if gate is not None:
        c.intermediate, c.gate, c.up, c.act_out = gate.shape[-1], ptr(gate), ptr(up), ptr(act_out)
    return c


def tensor(t, device=None) -> TbTensor:
    """TbTensor view of a torch tensor (no copy, owns_data = false)."""
    d = TbTensor()
    d.data = t.data_ptr()
    for i, s in enumerate(t.shape):
        d.shape[i] = s
    d.rank = t.dim()
    d.dtype = dtype_code(t)
    d.device = (DEVICE_CUDA if t.is_cuda else DEVICE_CPU) if device is None else device
    d.owns_data = False
    return d


# ------------------------------------------------------------ multi-GPU
def partition(total: int, parts: int, part: int):
    """[lo, hi) of part `part` when `total` items are split into `parts`."""
    lo, hi = C.c_int64(), C.c_int64()
    check(lib().tb_b200_partition(total, parts, part, C.byref(lo), C.byref(hi)), "partition")
    return lo.value, hi.value


def shard_plan(ids, vocab: int, nranks: int, rank: int):
    """The exchange plan of tb_b200_embedding_sharded for `rank` (host only):
    (send_counts, recv_counts, send_rows, recv_rows, local_dst, local_src) as
    numpy arrays, trimmed to their counts."""
    import numpy as np
    ids = np.ascontiguousarray(ids, np.int32)
    n = len(ids)
    sc = np.zeros(nranks, np.int64)
    rc = np.zeros(nranks, np.int64)
    bufs = [np.zeros(n + 1, np.int32) for _ in range(4)]
    nl = C.c_int64()
    check(lib().tb_b200_shard_plan(n, vocab, nranks, rank, ids.ctypes.data, sc.ctypes.data,
                                   rc.ctypes.data, *[b.ctypes.data for b in bufs], C.byref(nl)),
          "shard_plan")
    s, r, ld, ls = bufs
    return sc, rc, s[:sc.sum()], r[:rc.sum()], ld[:nl.value], ls[:nl.value]


def comm_unique_id() -> bytes:
    buf = C.create_string_buffer(128)
    check(lib().tb_b200_comm_unique_id(buf), "comm_unique_id")
    return buf.raw


def comm_init(nranks: int, rank: int, unique_id: bytes, device: int) -> None:
    buf = C.create_string_buffer(bytes(unique_id), 128)
    check(lib().tb_b200_comm_init(nranks, rank, buf, device), "comm_init")


def comm_destroy() -> None:
    check(lib().tb_b200_comm_destroy(), "comm_destroy")


def comm_wait(stream=None) -> int:
    """Bounded wait for the stream's queued work, exchanges included
    (tb_b200_comm_wait): TB_OK, or TB_ERR_DEVICE after aborting the
    communicator on an error or a timeout.  Returns the code."""
    return lib().tb_b200_comm_wait(stream or cur_stream())


def comm_window_alloc(nbytes: int) -> int:
    """Device address of `nbytes` of the communicator's symmetric memory
    (collective: every rank, same size, same order)."""
    p = vp()
    check(lib().tb_b200_comm_window_alloc(nbytes, C.byref(p)), "comm_window_alloc")
    return p.value


def comm_window_free(addr: int) -> None:
    check(lib().tb_b200_comm_window_free(vp(addr)), "comm_window_free")


def embedding_sharded_window(ids, shard_addr: int, vocab: int, dim: int, dtype, y=None,
                             stream=None):
    """Rows of `ids` (int32 CUDA tensor) from the vocab shards held in the
    communicator's symmetric memory (tb_b200_embedding_sharded_window)."""
    torch = _torch()
    _dev(ids)
    if y is None:
        y = torch.empty((ids.numel(), dim), dtype=dtype, device=ids.device)
    check(lib().tb_b200_embedding_sharded_window(dtype_code(y), ids.numel(), dim, vocab, ptr(ids),
                                                 vp(shard_addr), ptr(y), stream or cur_stream()),
          "embedding_sharded_window")
    return y


def comm_info():
    """(rank, nranks) of this process's communicator; (0, 0) without one."""
    rank, nranks = C.c_int(), C.c_int()
    check(lib().tb_b200_comm_info(C.byref(rank), C.byref(nranks)), "comm_info")
    return rank.value, nranks.value


def embedding_sharded(ids_host, table_shard, vocab: int, y_local=None, stream=None):
    """This rank's token part of the full-table gather, from its vocab shard
    (tb_b200_embedding_sharded).  ids_host: int32 numpy array of all tokens."""
    import numpy as np
    torch = _torch()
    rank, nranks = C.c_int(), C.c_int()
    check(lib().tb_b200_comm_info(C.byref(rank), C.byref(nranks)), "comm_info")
    ids = np.ascontiguousarray(ids_host, np.int32)
    lo, hi = partition(len(ids), nranks.value, rank.value)
    if y_local is None:
        y_local = torch.empty((hi - lo, table_shard.shape[1]), dtype=table_shard.dtype,
                              device=table_shard.device)
    check(lib().tb_b200_embedding_sharded(dtype_code(table_shard), len(ids), table_shard.shape[1],
                                          vocab, ids.ctypes.data, ptr(table_shard), ptr(y_local),
                                          stream or cur_stream()), "embedding_sharded")
    return y_local


P2P_HANDLE_BYTES = 64


def p2p_export(t):
    """(handle bytes, offset) of CUDA tensor t's allocation, for the other
    processes of the box to import (tb_b200_p2p_export)."""
    _dev(t)
    h = C.create_string_buffer(P2P_HANDLE_BYTES)
    off = C.c_int64()
    check(lib().tb_b200_p2p_export(ptr(t), h, C.byref(off)), "p2p_export")
    return h.raw, off.value


def p2p_import(handle: bytes, offset: int) -> int:
    """Device address, in this process, of a buffer another process exported."""
    p = vp()
    check(lib().tb_b200_p2p_import(C.create_string_buffer(bytes(handle), P2P_HANDLE_BYTES),
                                   offset, C.byref(p)), "p2p_import")
    return p.value


def p2p_close(addr: int, offset: int) -> None:
    check(lib().tb_b200_p2p_close(vp(addr), offset), "p2p_close")


def embedding_sharded_p2p(ids, shard_addrs, vocab: int, dim: int, dtype, y=None, stream=None):
    """The rows of `ids` (int32 CUDA tensor) gathered in one kernel from the
    vocab shards at `shard_addrs` (device addresses, rank order)
    (tb_b200_embedding_sharded_p2p)."""
    torch = _torch()
    _dev(ids)
    if ids.dtype != torch.int32:
        raise TypeError("ids must be int32")
    if y is None:
        y = torch.empty((ids.numel(), dim), dtype=dtype, device=ids.device)
    _dev(y)
    arr = (vp * len(shard_addrs))(*shard_addrs)
    check(lib().tb_b200_embedding_sharded_p2p(dtype_code(y), ids.numel(), dim, vocab, ptr(ids),
                                              arr, len(shard_addrs), ptr(y),
                                              stream or cur_stream()), "embedding_sharded_p2p")
    return y


# ------------------------- rotary positions, head norms, the 8-bit KV cache
# These calls are a few microseconds of GPU work in a decode step, so their
# checks are written to cost little: one look at each tensor's device, strides
# and dtype.
def _here():
    """(torch, index of the current device), where a launch goes."""
    torch = _torch()
    if not torch.cuda.is_initialized():
        if not torch.cuda.is_available():
            return torch, None  # no tensor is there
        torch.cuda.init()
    return torch, torch._C._cuda_getDevice()


def _stream(torch, dev, stream):
    """(The stream that a call given `stream` runs on, as an integer: torch's current one
    without, and where that is the default stream the one that the library takes for it
    (tb_b200_set_stream); it as torch's, None where it is the current one.)"""
    if dev is None:
        return 0, None  # no device: the tensors are refused
    here = torch._C._cuda_getCurrentRawStream(dev)
    there = here if stream is None else getattr(stream, "value", stream)
    there = there or lib().tb_b200_get_stream() or 0
    return there, None if there == here else torch.cuda.ExternalStream(there)


def _new(other, make, *args, **kw):
    """make(...), an uninitialised tensor for a call on stream `other` (of _stream): from
    that stream's pool, so that the memory's earlier uses are ordered before the call and
    its later ones after it."""
    if other is None:
        return make(*args, **kw)
    with _torch().cuda.stream(other):
        return make(*args, **kw)


def _c_int(n):
    """n as the C int that says the same to the library, which refuses what is below 0 and
    has bounds of its own; ctypes would take the low 32 bits."""
    return max(-1, min(n, 0x7fffffff))


def _device_is(t, dev):
    if t.get_device() != dev:
        raise ValueError(f"expected a tensor on the current device cuda:{dev}, got {t.device}")


def _heads(t, dtype, shape, dev, what):
    """Row stride of a [rows, heads, head_dim] tensor whose heads are dense
    within a row."""
    _device_is(t, dev)
    if t.dtype is not dtype:
        raise TypeError(f"{what} must be {dtype}, got {t.dtype}")
    if t.shape != shape:
        raise ValueError(f"{what} must be {tuple(shape)}, got {tuple(t.shape)}")
    s0, s1, s2 = t.stride()
    if (s2 != 1 and shape[2] > 1) or (s1 != shape[2] and shape[1] > 1):
        raise ValueError(f"{what} must have its heads dense in a row")
    return s0


def _flat(t, dtype, n, dev, what):
    """Address of a contiguous tensor of n elements."""
    _device_is(t, dev)
    if t.dtype is not dtype:
        raise TypeError(f"{what} must be {dtype}, got {t.dtype}")
    if t.numel() != n or not t.is_contiguous():
        raise ValueError(f"{what} must have {n} contiguous elements")
    return t.data_ptr()


def _heads_dtype(t):
    code = dtype_code(t)
    if code == I32 or t.dim() != 3:
        raise ValueError("expected [rows, heads, head_dim] of float32 or bfloat16")
    return code


def rotary_freqs(rotary_dim, theta, scaling="none", factor=1.0, trained=0.0, low=0.0, high=0.0,
                 out=None, stream=None):
    """Angle per position of each of rotary_dim / 2 pairs (float64, on the
    device), stretched by `scaling`: "none", "linear", "ntk", "bands" or
    "yarn" (tb_b200_rotary_freqs)."""
    torch, dev = _here()
    stream, other = _stream(torch, dev, stream)
    n = rotary_dim // 2
    if out is None:
        out = _new(other, torch.empty, n, dtype=torch.float64, device="cuda")
    at = _flat(out, torch.float64, n, dev, "out")
    sc = RotaryScaling(ROTARY_SCALING[scaling], theta, factor, trained, low, high)
    check(lib().tb_b200_rotary_freqs(_c_int(rotary_dim), sc, at, stream), "rotary_freqs")
    return out


def _rotary(fn, q, k, q_weight, k_weight, eps, positions, freqs, layout, scale, q_out, k_out,
            stream):
    torch, dev = _here()
    stream, other = _stream(torch, dev, stream)
    dtype, code = q.dtype, _heads_dtype(q)
    q_shape, k_shape = q.shape, k.shape
    rows, hq, d = q_shape
    if len(k_shape) != 3 or k_shape[0] != rows or k_shape[2] != d:
        raise ValueError("q and k must agree in rows and head_dim")
    hkv = k_shape[1]
    qs = _heads(q, dtype, q_shape, dev, "q")
    ks = _heads(k, dtype, k_shape, dev, "k")
    dense = torch.contiguous_format
    if q_out is None:
        q_out, qos = _new(other, torch.empty_like, q, memory_format=dense), hq * d
    else:
        qos = _heads(q_out, dtype, q_shape, dev, "q_out")
    if k_out is None:
        k_out, kos = _new(other, torch.empty_like, k, memory_format=dense), hkv * d
    else:
        kos = _heads(k_out, dtype, k_shape, dev, "k_out")
    r, at, fr = 0, None, None
    if freqs is not None:
        if positions is None:
            raise ValueError("freqs without positions")
        r = 2 * freqs.numel()
        at = _flat(positions, torch.int32, rows, dev, "positions")
        fr = _flat(freqs, torch.float64, r // 2, dev, "freqs")
    qw = None if q_weight is None else _flat(q_weight, dtype, d, dev, "q_weight")
    kw = None if k_weight is None else _flat(k_weight, dtype, d, dev, "k_weight")
    t = Rotary(code, rows, hq, hkv, d, r, _c_int(layout), q.data_ptr(), qs, k.data_ptr(), ks,
               q_out.data_ptr(), qos, k_out.data_ptr(), kos, at, fr, scale, qw, kw, eps)
    check(fn(t, stream), "rotary")
    return q_out, k_out


def rotary(q, k, positions, freqs, layout=ROTARY_HALF, scale=1.0, q_out=None, k_out=None,
           stream=None):
    """Rotary positions of q [R, Hq, d] and k [R, Hkv, d], whose rows may be
    strided (slices of a packed QKV): the first 2 * freqs.numel() elements of
    each head, at int32 positions [R] (tb_b200_rotary).  New tensors unless
    q_out and k_out are given; those may be q and k themselves."""
    return _rotary(lib().tb_b200_rotary, q, k, None, None, 0.0, positions, freqs, layout, scale,
                   q_out, k_out, stream)


def qk_norm_rotary(q, k, q_weight, k_weight, eps, positions=None, freqs=None,
                   layout=ROTARY_HALF, scale=1.0, q_out=None, k_out=None, stream=None):
    """RMSNorm of each head of q and k (weights [d] or None), then rotary
    positions, in one pass (tb_b200_qk_norm_rotary); without freqs the norm
    alone."""
    return _rotary(lib().tb_b200_qk_norm_rotary, q, k, q_weight, k_weight, eps, positions, freqs,
                   layout, scale, q_out, k_out, stream)


class Kv8Cache:
    """A paged 8-bit KV cache over the caller's tensors: codes k and v
    [n_pages, n_kv_heads, page, head_dim], int8 or float8_e4m3fn, and float32
    k_scale and v_scale [n_pages, n_kv_heads] (TbB200Kv8).  A scale is a power
    of two, as kv8_append writes it, or 0 in a page that nobody wrote, whose
    codes are 0: values take a scale's exponent alone, so any other one gives
    wrong results."""

    def __init__(self, k, v, k_scale, v_scale):
        torch = _torch()
        dtype, shape, dev = k.dtype, k.shape, k.get_device()
        if dtype is not torch.int8 and dtype is not torch.float8_e4m3fn:
            raise TypeError(f"codes must be int8 or float8_e4m3fn, got {dtype}")
        if dev < 0 or len(shape) != 4:
            raise ValueError("codes are CUDA tensors [n_pages, n_kv_heads, page, head_dim]")
        pages, heads, page, d = shape
        n, ns = pages * heads * page * d, pages * heads
        if v.shape != shape:
            raise ValueError("k and v must have the same shape")
        self.k, self.v, self.k_scale, self.v_scale, self.device = k, v, k_scale, v_scale, dev
        self.c = Kv8(KV_INT8 if dtype is torch.int8 else KV_E4M3, page, heads, d, pages,
                     _flat(k, dtype, n, dev, "k"), _flat(v, dtype, n, dev, "v"),
                     _flat(k_scale, torch.float32, ns, dev, "k_scale"),
                     _flat(v_scale, torch.float32, ns, dev, "v_scale"))

    @classmethod
    def empty(cls, n_pages, n_kv_heads, page, head_dim, dtype, device=None):
        """A cache of its own memory; dtype torch.int8 or torch.float8_e4m3fn."""
        torch = _torch()
        device = torch.cuda.current_device() if device is None else device
        codes = [torch.zeros((n_pages, n_kv_heads, page, head_dim), dtype=torch.uint8,
                             device=device).view(dtype) for _ in range(2)]
        scales = [torch.zeros((n_pages, n_kv_heads), dtype=torch.float32, device=device)
                  for _ in range(2)]
        return cls(*codes, *scales)


def _kv8_batch(torch, cache, dev, rows, row_start, lengths, page_table):
    i32_ = torch.int32
    if cache.device != dev:
        raise ValueError(f"the cache is on cuda:{cache.device}, the current device is cuda:{dev}")
    _device_is(page_table, dev)
    if page_table.dtype is not i32_:
        raise TypeError(f"page_table must be int32, got {page_table.dtype}")
    n, width = page_table.shape
    s0, s1 = page_table.stride()
    if s1 != 1 and width > 1:
        raise ValueError("page_table must be [n_seqs, pages], dense in a row")
    return Kv8Batch(n, rows, _flat(row_start, i32_, n + 1, dev, "row_start"),
                    _flat(lengths, i32_, n, dev, "lengths"), page_table.data_ptr(), width,
                    s0 if n > 1 else width)


def kv8_append(cache, k, v, row_start, lengths, page_table, stream=None):
    """Store K and V rows [R, n_kv_heads, head_dim] (rows may be strided) as
    the last tokens of the sequences of a ragged batch (tb_b200_kv8_append):
    rows row_start[i] : row_start[i + 1] end sequence i at lengths[i] tokens."""
    torch, dev = _here()
    dtype, code, shape = k.dtype, _heads_dtype(k), k.shape
    if shape[1] != cache.c.n_kv_heads or shape[2] != cache.c.head_dim:
        raise ValueError("k and v must be [rows, n_kv_heads, head_dim] of the cache")
    ks, vs = _heads(k, dtype, shape, dev, "k"), _heads(v, dtype, shape, dev, "v")
    b = _kv8_batch(torch, cache, dev, shape[0], row_start, lengths, page_table)
    check(lib().tb_b200_kv8_append(cache.c, b, code, k.data_ptr(), ks, v.data_ptr(), vs,
                                   _stream(torch, dev, stream)[0]), "kv8_append")


def kv8_attention(cache, q, row_start, lengths, page_table, max_q=None, max_len=None, scale=None,
                  window=0, out=None, lse=None, return_lse=False, workspace=None, stream=None):
    """Causal attention of q rows [R, n_heads, head_dim] over the cache
    (tb_b200_kv8_attention).  max_q and max_len bound the rows and the tokens
    of one sequence (as many as q and page_table hold without them); scale is
    1 / sqrt(head_dim) unless given; window > 0 attends that many last keys.
    Returns out, or (out, lse) with return_lse or lse."""
    torch, dev = _here()
    stream, other = _stream(torch, dev, stream)
    dtype, code, shape = q.dtype, _heads_dtype(q), q.shape
    rows, heads, d = shape
    if d != cache.c.head_dim:
        raise ValueError("q must be [rows, n_heads, head_dim] of the cache")
    qs = _heads(q, dtype, shape, dev, "q")
    dense = torch.contiguous_format
    if out is None:
        out, os_ = _new(other, torch.empty_like, q, memory_format=dense), heads * d
    else:
        os_ = _heads(out, dtype, shape, dev, "out")
    ls = None
    if lse is not None:
        if lse.shape != shape[:2]:
            raise ValueError("lse must be [rows, n_heads]")
        ls = _flat(lse, torch.float32, rows * heads, dev, "lse")
    elif return_lse:
        lse = _new(other, q.new_empty, (rows, heads), dtype=torch.float32)
        ls = lse.data_ptr()
    b = _kv8_batch(torch, cache, dev, rows, row_start, lengths, page_table)
    a = Kv8Attention(code, heads, q.data_ptr(), qs, out.data_ptr(), os_, ls,
                     d ** -0.5 if scale is None else scale, _c_int(window),
                     _c_int(rows if max_q is None else max_q),
                     min(b.table_width * cache.c.page, 1 << 30) if max_len is None
                     else _c_int(max_len), None, 0)
    L, need = lib(), C.c_size_t()
    if workspace is None:
        check(L.tb_b200_kv8_attention_workspace(cache.c, b, a, need), "kv8_attention_workspace")
        if need.value:
            workspace = _new(other, q.new_empty, need.value, dtype=torch.uint8)
    else:
        _device_is(workspace, dev)
        if not workspace.is_contiguous():
            raise ValueError("workspace must be contiguous")
    if workspace is not None:
        a.workspace = workspace.data_ptr()
        a.workspace_bytes = workspace.numel() * workspace.element_size()
    check(L.tb_b200_kv8_attention(cache.c, b, a, stream), "kv8_attention")
    return out if lse is None else (out, lse)


# ------------------------- microscaled formats, their product, filtered sampling
class MxTensor:
    """[rows, cols] in a microscaled format ("e4m3" or "e2m1") over the caller's uint8
    tensors: codes [rows, bytes of a row], whose columns are filled up to a multiple of 128,
    and the tiled scales (TbB200Mx)."""

    def __init__(self, codes, scales, cols, format):
        torch = _torch()
        dev = codes.get_device()
        if dev < 0 or codes.dim() != 2:
            raise ValueError("codes are a CUDA tensor [rows, bytes of a row]")
        rows = codes.shape[0]
        tiles = -(-cols // 128)
        pitch = tiles * (64 if format == "e2m1" else 128)
        self.c = Mx(MX_FORMATS[format], rows, cols,
                    _flat(codes, torch.uint8, rows * pitch, dev, "codes"),
                    _flat(scales, torch.uint8, -(-rows // 128) * tiles * 512, dev, "scales"))
        self.codes, self.scales, self.format, self.device = codes, scales, format, dev
        self.rows, self.cols = rows, cols

    @classmethod
    def empty(cls, rows, cols, format="e4m3", device=None):
        """A tensor of its own, uninitialised memory."""
        torch = _torch()
        device = torch.cuda.current_device() if device is None else device
        return cls._like(torch.empty(0, dtype=torch.uint8, device=device), rows, cols, format)

    @classmethod
    def _like(cls, t, rows, cols, format):
        """empty() on tensor t's device, past the checks of the caller's tensors."""
        if cols < 1:
            raise ValueError("an MxTensor has columns")
        u8 = _torch().uint8
        tiles = -(-cols // 128)
        self = cls.__new__(cls)
        self.codes = codes = t.new_empty((rows, tiles * (64 if format == "e2m1" else 128)),
                                         dtype=u8)
        self.scales = scales = t.new_empty(-(-rows // 128) * tiles * 512, dtype=u8)
        self.c = Mx(MX_FORMATS[format], rows, cols, codes.data_ptr(), scales.data_ptr())
        self.format, self.device, self.rows, self.cols = format, t.get_device(), rows, cols
        return self


def _mx(t, dev, what):
    if t.device != dev:
        raise ValueError(f"{what} is on cuda:{t.device}, the current device is cuda:{dev}")
    return t.c


def _mx_out(other, dev, out, like, rows, cols, format):
    if out is None:
        return _new(other, MxTensor._like, like, rows, cols, format or "e4m3")
    if (out.rows, out.cols) != (rows, cols):
        raise ValueError(f"out must be [{rows}, {cols}]")
    if format is not None and format != out.format:
        raise TypeError(f"out must be in {format}, got {out.format}")
    _mx(out, dev, "out")
    return out


def _rows(t, dev, what, dtype=None):
    """(dtype code, row stride) of a [rows, cols] tensor of f32 or bf16 that is dense in a
    row."""
    _device_is(t, dev)
    code = dtype_code(t)
    if code == I32 or t.dim() != 2:
        raise ValueError(f"{what} must be [rows, cols] of float32 or bfloat16")
    if dtype is not None and t.dtype is not dtype:
        raise TypeError(f"{what} must be {dtype}, got {t.dtype}")
    s0, s1 = t.stride()
    if s1 != 1 and t.shape[1] > 1:
        raise ValueError(f"{what} must be dense in a row")
    return code, s0


def mx_quantize(x, format=None, out=None, stream=None):
    """x [rows, cols], whose rows may be strided, in a microscaled format (`format`, or out's;
    e4m3 without both) (tb_b200_mx_quantize)."""
    torch, dev = _here()
    stream, other = _stream(torch, dev, stream)
    code, stride = _rows(x, dev, "x")
    out = _mx_out(other, dev, out, x, x.shape[0], x.shape[1], format)
    check(lib().tb_b200_mx_quantize(code, x.data_ptr(), stride, out.c, stream), "mx_quantize")
    return out


def mx_dequantize(t, dtype=None, out=None, stream=None):
    """The values of an MxTensor, [rows, cols] of float32 or bfloat16 (`dtype`, or out's)
    (tb_b200_mx_dequantize)."""
    torch, dev = _here()
    stream, other = _stream(torch, dev, stream)
    c = _mx(t, dev, "t")
    if out is None:
        out = _new(other, t.codes.new_empty, (t.rows, t.cols),
                   dtype=torch.float32 if dtype is None else dtype)
    elif out.shape != (t.rows, t.cols):
        raise ValueError(f"out must be [{t.rows}, {t.cols}]")
    code, stride = _rows(out, dev, "out", dtype)
    check(lib().tb_b200_mx_dequantize(c, code, out.data_ptr(), stride, stream), "mx_dequantize")
    return out


def residual_rms_norm_mx(x, residual, weight, eps, h_out=None, format=None, out=None,
                         stream=None):
    """(h, y): residual_rms_norm of [rows, cols] with y in a microscaled format (`format`, or
    out's; e4m3 without both) (tb_b200_residual_rms_norm_mx): h / sqrt((eps + sum h^2) / cols),
    so a model whose norm has mean(h^2) + eps gives cols * eps.  residual None: the norm of x,
    with no h; h is a new tensor unless h_out is given (x or residual may be)."""
    torch, dev = _here()
    stream, other = _stream(torch, dev, stream)
    code, _ = _rows(x, dev, "x")
    (rows, cols), dtype = x.shape, x.dtype
    n = rows * cols
    at = [_flat(x, dtype, n, dev, "x"),
          None if residual is None else _flat(residual, dtype, n, dev, "residual"),
          None if weight is None else _flat(weight, dtype, cols, dev, "weight")]
    if h_out is None and residual is not None:
        h_out = _new(other, torch.empty_like, x)
    h = None if h_out is None else _flat(h_out, dtype, n, dev, "h_out")
    out = _mx_out(other, dev, out, x, rows, cols, format)
    check(lib().tb_b200_residual_rms_norm_mx(code, *at, h, out.c, eps, stream),
          "residual_rms_norm_mx")
    return h_out, out


def swiglu_mx(gate, up, format=None, out=None, stream=None):
    """silu(gate) * up of [rows, cols], whose rows may be strided, in a microscaled format
    (`format`, or out's; e4m3 without both) (tb_b200_swiglu_mx)."""
    torch, dev = _here()
    stream, other = _stream(torch, dev, stream)
    code, gs = _rows(gate, dev, "gate")
    _, us = _rows(up, dev, "up", gate.dtype)
    if up.shape != gate.shape:
        raise ValueError("gate and up must have the same shape")
    out = _mx_out(other, dev, out, gate, gate.shape[0], gate.shape[1], format)
    check(lib().tb_b200_swiglu_mx(code, gate.data_ptr(), gs, up.data_ptr(), us, out.c, stream),
          "swiglu_mx")
    return out


def mx_linear(x, w, bias=None, dtype=None, y=None, stream=None):
    """y = x w^T (+ bias) of MxTensors x [rows, cols] and w [outs, cols]: [rows, outs] of
    float32 or bfloat16 (`dtype`, or y's; bfloat16 without both), bias float32 [outs]
    (tb_b200_mx_linear)."""
    torch, dev = _here()
    stream, other = _stream(torch, dev, stream)
    xc, wc = _mx(x, dev, "x"), _mx(w, dev, "w")
    if y is None:
        y = _new(other, x.codes.new_empty, (x.rows, w.rows),
                 dtype=torch.bfloat16 if dtype is None else dtype)
    elif y.shape != (x.rows, w.rows):
        raise ValueError(f"y must be [{x.rows}, {w.rows}]")
    code, stride = _rows(y, dev, "y", dtype)
    b = None if bias is None else _flat(bias, torch.float32, w.rows, dev, "bias")
    check(lib().tb_b200_mx_linear(xc, wc, b, code, y.data_ptr(), stride, stream), "mx_linear")
    return y


def sample(logits, uniforms, temperature=None, top_k=None, top_p=None, min_p=None, out=None,
           stream=None):
    """A token of each row of logits [rows, vocab] (rows may be strided), drawn by its
    uniform (float64 in [0, 1)) after its temperature, top_k (int32), top_p and min_p
    (float32), device tensors [rows] or None for off (tb_b200_sample).  int32 [rows]."""
    torch, dev = _here()
    stream, other = _stream(torch, dev, stream)
    code, stride = _rows(logits, dev, "logits")
    rows, vocab = logits.shape
    f = torch.float32

    def setting(t, dtype, what):
        return None if t is None else _flat(t, dtype, rows, dev, what)

    if out is None:
        out = _new(other, logits.new_empty, rows, dtype=torch.int32)
    t = Sample(code, rows, vocab, logits.data_ptr(), stride,
               setting(temperature, f, "temperature"), setting(top_k, torch.int32, "top_k"),
               setting(top_p, f, "top_p"), setting(min_p, f, "min_p"),
               _flat(uniforms, torch.float64, rows, dev, "uniforms"),
               _flat(out, torch.int32, rows, dev, "out"))
    check(lib().tb_b200_sample(t, stream), "sample")
    return out


# ------------------------------------------------ decoder forward (runner)
def decode_attention(q, k, v, k_cache, v_cache, position, n_heads, n_kv_heads,
                     mode=ATTN_REFERENCE, out=None, stream=None):
    """Single-token attention over one layer's f32 KV cache
    [max_seq, n_kv_heads * head_dim]; `position` a 1-element int32 device
    tensor.  Also writes k and v into cache row `position`."""
    torch = _torch()
    head_dim = q.numel() // n_heads
    out = torch.empty(n_heads * head_dim, dtype=torch.float32, device=q.device) if out is None else out
    _dev(q, k, v, k_cache, v_cache, position, out)
    check(lib().tb_b200_decode_attention(mode, n_heads, n_kv_heads, head_dim, k_cache.shape[0],
                                         ptr(position), ptr(q), ptr(k), ptr(v), ptr(k_cache),
                                         ptr(v_cache), ptr(out), stream or cur_stream()),
          "decode_attention")
    return out


class QuantWeight:
    """An INT4 (dtype INT4, two weights per byte, low nibble first) or INT8
    weight tensor [rows, cols] with per-group f32 scales, as a .tbm layer
    stores it."""

    def __init__(self, data, dtype, rows, cols, scales, group_size):
        self.data, self.dtype, self.rows, self.cols = data, dtype, rows, cols
        self.scales, self.group_size = scales, group_size


class Runner:
    """TransformerRunner (include/tensorbit/run/ops.hpp:33-288) on the device.

    cfg: dict with hidden, n_heads, n_kv_heads, head_dim, intermediate,
    vocab, max_seq, layers, norm_eps, rope_theta.  model: {"embed": W,
    "final_norm": v, "lm_head": W or None, "layers": [{"q": (W, mask), ...,
    "in_norm": v, "post_norm": v}]}, where W is an f32 numpy array (copied
    to the device), an f32 CUDA tensor (borrowed) or a QuantWeight, and a
    mask is uint8 2:4 group bytes or None (dense)."""

    def __init__(self, cfg, model, attention=ATTN_REFERENCE, use_graph=True):
        import numpy as np
        self._keep = []
        self.vocab = int(cfg["vocab"])

        def addr(a, dt=None):
            if a is None:
                return None
            if hasattr(a, "data_ptr"):
                self._keep.append(a)
                return a.data_ptr()
            a = np.ascontiguousarray(a, dtype=dt)
            self._keep.append(a)
            return a.ctypes.data

        def weight(w, mask=None):
            if w is None:
                return Weight()
            if isinstance(w, QuantWeight):
                sc = w.scales
                n_sc = 0 if sc is None else int(sc.numel() if hasattr(sc, "numel") else np.size(sc))
                return Weight(addr(w.data, np.uint8), w.dtype, w.rows, w.cols, addr(mask, np.uint8),
                              addr(sc, np.float32), n_sc, w.group_size)
            return Weight(addr(w, np.float32), F32, w.shape[0], w.shape[1], addr(mask, np.uint8),
                          None, 0, 0)

        n_layers = int(cfg["layers"])
        layers = (RunnerLayer * max(1, n_layers))()
        for i, ly in enumerate(model["layers"][:n_layers]):
            for n in PROJECTIONS:
                wm = ly.get(n)
                if wm is not None:
                    setattr(layers[i], n, weight(wm[0], wm[1] if len(wm) > 1 else None))
            layers[i].input_norm = addr(ly.get("in_norm"), np.float32)
            layers[i].post_norm = addr(ly.get("post_norm"), np.float32)
        d = RunnerDesc(*[int(cfg[n]) for n in ("hidden", "n_heads", "n_kv_heads", "head_dim",
                                               "intermediate", "vocab", "max_seq", "layers")],
                       float(cfg.get("norm_eps", 1e-5)), float(cfg.get("rope_theta", 10000.0)),
                       attention, 1 if use_graph else 0, weight(model["embed"]),
                       addr(model.get("final_norm"), np.float32), weight(model.get("lm_head")),
                       layers)
        h = vp()
        check(lib().tb_b200_runner_create(C.byref(d), C.byref(h)), "runner_create")
        self._h = h
        # host arrays were copied during create; device tensors stay borrowed
        self._keep = [a for a in self._keep if hasattr(a, "data_ptr")]

    @classmethod
    def from_desc(cls, desc, vocab, keep=()):
        """A runner from a filled RunnerDesc (e.g. tb_b200_tbm_runner_desc);
        `keep` holds whatever the descriptor points into."""
        self = cls.__new__(cls)
        self._keep = list(keep)
        self.vocab = int(vocab)
        h = vp()
        check(lib().tb_b200_runner_create(C.byref(desc), C.byref(h)), "runner_create")
        self._h = h
        return self

    def forward(self, token):
        """Run one token; returns the device logits address (valid until the
        next forward)."""
        out = vp()
        check(lib().tb_b200_runner_forward(self._h, int(token), C.byref(out)), "runner_forward")
        return out.value

    def logits(self):
        import numpy as np
        out = np.empty(self.vocab, dtype=np.float32)
        check(lib().tb_b200_runner_logits(self._h, out.ctypes.data), "runner_logits")
        return out

    def reset(self):
        check(lib().tb_b200_runner_reset(self._h), "runner_reset")

    @property
    def position(self):
        p = i32()
        check(lib().tb_b200_runner_position(self._h, C.byref(p)), "runner_position")
        return p.value

    @property
    def stream(self):
        s = vp()
        check(lib().tb_b200_runner_stream(self._h, C.byref(s)), "runner_stream")
        return s

    @property
    def launches_per_token(self):
        n = i32()
        check(lib().tb_b200_runner_launches_per_token(self._h, C.byref(n)), "runner_launches")
        return n.value

    def close(self):
        if getattr(self, "_h", None):
            lib().tb_b200_runner_destroy(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class TbmModel:
    """A .tbm container read into device memory (tb_b200_tbm_load)."""

    def __init__(self, path, stream=None):
        h = vp()
        check(lib().tb_b200_tbm_load(str(path).encode(), stream or cur_stream(), C.byref(h)),
              "tbm_load")
        self._h = h

    def config(self) -> TbmConfig:
        c = TbmConfig()
        check(lib().tb_b200_tbm_config(self._h, C.byref(c)), "tbm_config")
        return c

    def __len__(self):
        n = i32()
        check(lib().tb_b200_tbm_count(self._h, C.byref(n)), "tbm_count")
        return n.value

    def tensor(self, i):
        """(return code, TbmTensor) of tensor i: TB_OK, or TB_ERR_BAD_MAGIC
        for a tensor whose .tb header is not one."""
        t = TbmTensor()
        rc = lib().tb_b200_tbm_tensor(self._h, i, C.byref(t))
        return rc, t

    def find(self, name):
        i = i32()
        rc = lib().tb_b200_tbm_find(self._h, name.encode(), C.byref(i))
        return i.value if rc == 0 else -1

    def runner(self, attention=ATTN_REFERENCE, use_graph=True, max_layers=512):
        """A device runner over this model's tensors (borrowed: the model
        must stay open while the runner lives)."""
        layers = (RunnerLayer * max_layers)()
        d = RunnerDesc()
        check(lib().tb_b200_tbm_runner_desc(self._h, attention, 1 if use_graph else 0,
                                            C.byref(d), layers, max_layers), "tbm_runner_desc")
        return Runner.from_desc(d, d.vocab, keep=(layers, self))

    def close(self):
        if getattr(self, "_h", None):
            check(lib().tb_b200_tbm_free(self._h), "tbm_free")
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass
