"""Python binding of libq4k_gemv.so (the C ABI in include/q4k_gemv.h,
include/q4k_batch.h, include/q4k_step.h and include/q4k_gguf.h).

The product is the C ABI; this module is plumbing for tests and the
benchmark: it passes torch device tensors and torch's current HIP stream to
the library and turns status codes into exceptions.  It never computes on the
CPU: if the library is missing, loading it raises.

torch is imported before the library is loaded so that the library binds to
the HIP runtime torch already loaded (one runtime per process).
"""
from __future__ import annotations

import ctypes
import os

import numpy as np

PKG_DIR = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(PKG_DIR, "libq4k_gemv.so")

Q4K_OK, Q4K_EUNSUPPORTED, Q4K_EINVAL, Q4K_EHIP, Q4K_ENOMEM, Q4K_EIO, Q4K_EFORMAT, Q4K_ESCRATCH = 0, 1, 2, 3, 4, 5, 6, 7
NOALLOC_SCRATCH_BYTES = 1 << 20
GGML_TYPE_F32, GGML_TYPE_Q8_1, GGML_TYPE_Q4_K, GGML_TYPE_Q6_K = 0, 9, 12, 14
GGML_TYPE_F16, GGML_TYPE_BF16 = 1, 30
QK_K = 256
BLOCK_Q4_K_BYTES = 144
BLOCK_Q6_K_BYTES = 210
BLOCK_Q8_1_BYTES = 36
MATRIX_ROW_PADDING = 512

class q4k_gguf_tensor_info(ctypes.Structure):
    """A GGUF tensor directory entry (include/q4k_gguf.h)."""
    _fields_ = [("name", ctypes.c_char_p), ("type", ctypes.c_int32), ("n_dims", ctypes.c_int32),
                ("ne", ctypes.c_int64 * 4), ("offset", ctypes.c_uint64), ("nbytes", ctypes.c_uint64),
                ("data", ctypes.c_void_p)]


_P = ctypes.c_void_p
_I64 = ctypes.c_int64
_I = ctypes.c_int


class q4k_lora(ctypes.Structure):
    """The adapters of one projection (include/q4k_batch.h)."""
    _fields_ = [("type", ctypes.c_int32), ("rank", ctypes.c_int32), ("n_adapters", _I64),
                ("a", _P), ("nb_a", _I64), ("nb_a_adapter", _I64),
                ("b", _P), ("nb_b", _I64), ("nb_b_adapter", _I64),
                ("scale", _P), ("ranks", _P)]


class q4k_kv_pages(ctypes.Structure):
    """Keys and values in pages (include/q4k_batch.h)."""
    _fields_ = [("k", _P), ("v", _P), ("n_pages", _I64), ("page_size", _I64),
                ("nb_k_page", _I64), ("nb_k_token", _I64), ("nb_k_head", _I64),
                ("nb_v_page", _I64), ("nb_v_token", _I64), ("nb_v_head", _I64),
                ("table", _P), ("table_stride", _I64), ("table_len", _I64)]


class q4k_prefix_attn_args(ctypes.Structure):
    """Arguments of q4k_prefix_attn (include/q4k_batch.h)."""
    _fields_ = [("q_type", ctypes.c_int32), ("kv_type", ctypes.c_int32), ("n_head", ctypes.c_int32),
                ("n_head_kv", ctypes.c_int32), ("head_dim", ctypes.c_int32), ("scale", ctypes.c_float),
                ("n_tokens", _I64), ("n_requests", _I64), ("n_q", _I64), ("q_start", _P),
                ("q", _P), ("nb_q_token", _I64), ("nb_q_head", _I64),
                ("prefix", ctypes.POINTER(q4k_kv_pages)), ("n_prefix", _I64),
                ("suffix", ctypes.POINTER(q4k_kv_pages)), ("suffix_len", _P), ("max_suffix", _I64),
                ("dst", _P), ("nb_dst_token", _I64), ("nb_dst_head", _I64), ("lse", _P)]


class q4k_logits_rules(ctypes.Structure):
    """What changes the logits of each row (include/q4k_batch.h)."""
    _fields_ = [("repeat", _P), ("frequency", _P), ("presence", _P),
                ("history", _P), ("history_start", _P), ("n_history", _I64),
                ("bias_ids", _P), ("bias", _P), ("bias_start", _P), ("n_bias", _I64),
                ("mask", _P), ("n_masks", _I64), ("nb_mask", _I64), ("mask_rows", _P)]


class q4k_rope_rows(ctypes.Structure):
    """Rows of queries or keys (include/q4k_step.h)."""
    _fields_ = [("src", _P), ("dst", _P), ("src_type", ctypes.c_int32), ("dst_type", ctypes.c_int32), ("n_head", _I64),
                ("nb_src_token", _I64), ("nb_src_head", _I64), ("nb_dst_token", _I64), ("nb_dst_head", _I64), ("norm", _P)]


class q4k_rope_args(ctypes.Structure):
    """Arguments of q4k_rope (include/q4k_step.h)."""
    _fields_ = [("head_dim", ctypes.c_int32), ("n_rot", ctypes.c_int32), ("mode", ctypes.c_int32), ("eps", ctypes.c_float),
                ("freq_base", ctypes.c_float), ("freq_scale", ctypes.c_float), ("ext_factor", ctypes.c_float),
                ("attn_factor", ctypes.c_float), ("beta_fast", ctypes.c_float), ("beta_slow", ctypes.c_float),
                ("n_ctx_orig", _I64), ("freq_factors", _P), ("n_tokens", _I64), ("pos", _P),
                ("q", ctypes.POINTER(q4k_rope_rows)), ("k", ctypes.POINTER(q4k_rope_rows))]


class q4k_kv8_pages(ctypes.Structure):
    """Keys and values in pages of 8 bits (include/q4k_step.h)."""
    _fields_ = [("type", ctypes.c_int32), ("n_head_kv", ctypes.c_int32), ("head_dim", ctypes.c_int32), ("block", ctypes.c_int32),
                ("k", _P), ("v", _P), ("n_pages", _I64), ("page_size", _I64),
                ("nb_k_page", _I64), ("nb_k_token", _I64), ("nb_k_head", _I64),
                ("nb_v_page", _I64), ("nb_v_token", _I64), ("nb_v_head", _I64),
                ("k_scale", _P), ("v_scale", _P), ("nb_s_page", _I64), ("nb_s_block", _I64), ("nb_s_head", _I64),
                ("table", _P), ("table_stride", _I64), ("table_len", _I64)]


class q4k_kv8_rows(ctypes.Structure):
    """The last tokens of each request (include/q4k_step.h)."""
    _fields_ = [("pages", ctypes.POINTER(q4k_kv8_pages)), ("type", ctypes.c_int32), ("n_tokens", _I64), ("n_requests", _I64),
                ("n_q", _I64), ("q_start", _P), ("len", _P), ("max_len", _I64), ("k", _P), ("v", _P),
                ("nb_k_token", _I64), ("nb_k_head", _I64), ("nb_v_token", _I64), ("nb_v_head", _I64)]


class q4k_kv8_attn_args(ctypes.Structure):
    """Arguments of q4k_kv8_attn (include/q4k_step.h)."""
    _fields_ = [("pages", ctypes.POINTER(q4k_kv8_pages)), ("q_type", ctypes.c_int32), ("n_head", ctypes.c_int32), ("scale", ctypes.c_float),
                ("n_tokens", _I64), ("n_requests", _I64), ("n_q", _I64), ("q_start", _P), ("len", _P), ("max_len", _I64),
                ("q", _P), ("nb_q_token", _I64), ("nb_q_head", _I64), ("dst", _P), ("nb_dst_token", _I64), ("nb_dst_head", _I64), ("lse", _P)]


class q4k_sample_rules(ctypes.Structure):
    """How the next token of each row is drawn (include/q4k_step.h)."""
    _fields_ = [("temperature", _P), ("top_k", _P), ("top_p", _P), ("min_p", _P), ("uniform", _P)]


# Every symbol the headers of include/ declare: (restype, argtypes)
SIGNATURES = {
    "q4k_version": (ctypes.c_int32, []),
    "q4k_strerror": (ctypes.c_char_p, [_I]),
    "q4k_last_hip_error": (ctypes.c_int32, []),
    "q4k_q8_1_bytes": (ctypes.c_size_t, [_I64, _I64]),
    "q4k_quantize_row_q8_1": (_I, [_P, _P, _I64, _I64, _I64, _I64, _P]),
    "q4k_mul_mat_vec_q": (_I, [_P, _I64, _I64, _I64, _P, _I64, _I64, _P, _I64, _P, ctypes.c_size_t, _P]),
    "q4k_mul_mat_vec_q_noalloc": (_I, [_P, _I64, _I64, _I64, _P, _I64, _I64, _P, _I64, _P]),
    "q4k_mul_mat_vec_q_sums": (_I, [_P, _I64, _I64, _I64, _P, _I64, _I64, _P, _I64, _P, ctypes.c_size_t,
                                    _P, _P, _P]),
    "q6k_mul_mat_vec_q_sums": (_I, [_P, _I64, _I64, _I64, _P, _I64, _I64, _P, _I64, _P, ctypes.c_size_t,
                                    _P, _P]),
    "q4k_op_mul_mat_vec_q": (_I, [_P, _I64, _I64, _I64, _P, _I64, _I64, _P, _I64, _P]),
    "q4k_ggml_mul_mat_vec_q": (_I, [_P, _P, _P, _P, _P, _P, ctypes.c_size_t, _P]),
    "q4k_subblock_sums": (_I, [_P, _I64, _I64, _I64, _P, _I64, _I64, _P, _P, _P]),
    "q4k_gemv_geometry": (_I, [_I64, _I64, _I64, _P]),
    "q4k_gemv_geometry_q8_1": (_I, [_I64, _I64, _I64, _P]),
    "q4k_gemv_geometry_fused": (_I, [_I64, _I64, ctypes.c_int32, _P]),
    "q6k_gemv_geometry_fused": (_I, [_I64, _I64, ctypes.c_int32, _P]),
    "q4k_set_geometry_override": (_I, [ctypes.c_int32] * 4),
    "q4k_set_pipeline_override": (_I, [ctypes.c_int32] * 2),
    "q4k_read_probe": (_I, [_P, ctypes.c_size_t, ctypes.c_int32, ctypes.c_int32, ctypes.c_int32, ctypes.c_int32,
                            _P, _P]),
    "q4k_mul_mat_vec_q_fused": (_I, [ctypes.c_int32, _P, _I64, _I64, _I64, _P, _P, _P, _P]),
    "q4k_quantize_rows_q4_K": (_I, [_P, _P, _I64, _I64, _I]),
    "q6k_mul_mat_vec_q": (_I, [_P, _I64, _I64, _I64, _P, _I64, _I64, _P, _I64, _P, ctypes.c_size_t, _P]),
    "q6k_op_mul_mat_vec_q": (_I, [_P, _I64, _I64, _I64, _P, _I64, _I64, _P, _I64, _P]),
    "q6k_group_sums": (_I, [_P, _I64, _I64, _I64, _P, _I64, _I64, _P, _P]),
    "q6k_gemv_geometry": (_I, [_I64, _I64, _I64, _P]),
    "q6k_gemv_geometry_q8_1": (_I, [_I64, _I64, _I64, _P]),
    "q4k_quantize_rows_q6_K": (_I, [_P, _P, _I64, _I64, _I]),
    # include/q4k_batch.h
    "q4k_lora_workspace_bytes": (ctypes.c_size_t, [_P, _I64, _I64, _I64]),
    "q4k_lora_add": (_I, [_P, _I64, _I64, _P, _I64, _I64, _P, _P, _I64, _P, _I64, _P, ctypes.c_size_t, _P]),
    "q4k_prefix_attn_workspace_bytes": (ctypes.c_size_t, [_P]),
    "q4k_prefix_attn": (_I, [_P, _P, ctypes.c_size_t, _P]),
    "q4k_logits_adjust": (_I, [_P, _I64, _I64, _I64, _P, _P, _I64, _P]),
    # include/q4k_step.h
    "q4k_rope": (_I, [_P, _P]),
    "q4k_kv8_store": (_I, [_P, _P]),
    "q4k_kv8_load": (_I, [_P, _P]),
    "q4k_kv8_attn_workspace_bytes": (ctypes.c_size_t, [_P]),
    "q4k_kv8_attn": (_I, [_P, _P, ctypes.c_size_t, _P]),
    "q4k_sample_workspace_bytes": (ctypes.c_size_t, [_I64, _I64]),
    "q4k_sample": (_I, [_P, _I64, _I64, _I64, _P, _P, _P, _P, ctypes.c_size_t, _P]),
    # include/q4k_gguf.h
    "q4k_gguf_open": (_I, [ctypes.c_char_p, ctypes.POINTER(_P)]),
    "q4k_gguf_close": (None, [_P]),
    "q4k_gguf_version": (ctypes.c_uint32, [_P]),
    "q4k_gguf_alignment": (ctypes.c_uint64, [_P]),
    "q4k_gguf_data_offset": (ctypes.c_uint64, [_P]),
    "q4k_gguf_tensor_count": (_I64, [_P]),
    "q4k_gguf_find_tensor": (_I64, [_P, ctypes.c_char_p]),
    "q4k_gguf_get_tensor": (_I, [_P, _I64, ctypes.POINTER(q4k_gguf_tensor_info)]),
    "q4k_ggml_row_size": (ctypes.c_uint64, [ctypes.c_int32, _I64]),
    "q4k_gguf_kv_count": (_I64, [_P]),
    "q4k_gguf_find_key": (_I64, [_P, ctypes.c_char_p]),
    "q4k_gguf_key": (ctypes.c_char_p, [_P, _I64]),
    "q4k_gguf_kv_type": (ctypes.c_int32, [_P, _I64]),
    "q4k_gguf_get_int": (_I, [_P, _I64, ctypes.POINTER(_I64)]),
    "q4k_gguf_get_float": (_I, [_P, _I64, ctypes.POINTER(ctypes.c_double)]),
    "q4k_gguf_get_str": (_I, [_P, _I64, ctypes.POINTER(ctypes.c_char_p)]),
    "q4k_gguf_get_arr": (_I, [_P, _I64, ctypes.POINTER(ctypes.c_int32), ctypes.POINTER(_I64),
                              ctypes.POINTER(_P)]),
    "q4k_gguf_get_arr_str": (_I, [_P, _I64, _I64, ctypes.POINTER(ctypes.c_char_p)]),
}


class q4k_tensor(ctypes.Structure):
    """The ggml_tensor subset of include/q4k_gemv.h."""
    _fields_ = [("type", ctypes.c_int32), ("ne", ctypes.c_int64 * 4), ("nb", ctypes.c_size_t * 4),
                ("data", ctypes.c_void_p)]


class q4k_fusion(ctypes.Structure):
    """Fused epilogue, device pointers (include/q4k_gemv.h)."""
    _fields_ = [("x_bias", ctypes.c_void_p), ("gate", ctypes.c_void_p), ("gate_bias", ctypes.c_void_p),
                ("glu_op", ctypes.c_int32)]


class q4k_fusion_args(ctypes.Structure):
    """Fused epilogue, tensor descriptors (ggml_cuda_mm_fusion_args_host)."""
    _fields_ = [("x_bias", ctypes.POINTER(q4k_tensor)), ("gate", ctypes.POINTER(q4k_tensor)),
                ("gate_bias", ctypes.POINTER(q4k_tensor)), ("glu_op", ctypes.c_int32)]


GLU_OP_GEGLU, GLU_OP_SWIGLU, GLU_OP_SWIGLU_OAI = 1, 2, 3


class Q4KError(RuntimeError):
    def __init__(self, status: int, where: str):
        self.status = status
        msg = f"{where}: {lib().q4k_strerror(status).decode()} (status {status}"
        if status == Q4K_EHIP:
            msg += f", hipError {lib().q4k_last_hip_error()}"
        super().__init__(msg + ")")


_lib = None


def lib():
    """Loads libq4k_gemv.so (raises if it has not been built)."""
    global _lib
    if _lib is None:
        import torch  # noqa: F401  -- bind to torch's HIP runtime
        if not os.path.exists(LIB_PATH):
            raise RuntimeError(f"{LIB_PATH} is missing: build it with gemv-q4_k-optimization_amd/build.py")
        L = ctypes.CDLL(LIB_PATH)
        for name, (res, args) in SIGNATURES.items():
            f = getattr(L, name)
            f.restype = res
            f.argtypes = args
        _lib = L
    return _lib


def _check(status: int, where: str):
    if status != Q4K_OK:
        raise Q4KError(status, where)


def _stream(stream=None):
    """torch's current HIP stream (or `stream`); the null stream when no GPU
    is visible, where only the host-side argument checks can run."""
    import torch
    if stream is None:
        if not torch.cuda.is_available():
            return None
        stream = torch.cuda.current_stream()
    return ctypes.c_void_p(stream.cuda_stream)


def _ptr(t) -> ctypes.c_void_p:
    return ctypes.c_void_p(t.data_ptr()) if t is not None else None


def pad_k(K: int) -> int:
    return (K + MATRIX_ROW_PADDING - 1) // MATRIX_ROW_PADDING * MATRIX_ROW_PADDING


def q8_1_bytes(K: int, ncols: int) -> int:
    return int(lib().q4k_q8_1_bytes(K, ncols))


# ------------------------------------------------------------------ host ----
def quantize_rows_q4_K(w: np.ndarray, nthreads: int = 8) -> np.ndarray:
    """Host F32 [M, K] -> Q4_K bytes [M, K/256*144]."""
    w = np.ascontiguousarray(w, dtype=np.float32)
    M, K = w.shape
    out = np.empty((M, K // QK_K * BLOCK_Q4_K_BYTES), dtype=np.uint8)
    _check(lib().q4k_quantize_rows_q4_K(w.ctypes.data_as(_P), out.ctypes.data_as(_P), M, K, nthreads),
           "q4k_quantize_rows_q4_K")
    return out


def quantize_rows_q6_K(w: np.ndarray, nthreads: int = 8) -> np.ndarray:
    """Host F32 [M, K] -> Q6_K bytes [M, K/256*210]."""
    w = np.ascontiguousarray(w, dtype=np.float32)
    M, K = w.shape
    out = np.empty((M, K // QK_K * BLOCK_Q6_K_BYTES), dtype=np.uint8)
    _check(lib().q4k_quantize_rows_q6_K(w.ctypes.data_as(_P), out.ctypes.data_as(_P), M, K, nthreads),
           "q4k_quantize_rows_q6_K")
    return out


# ---------------------------------------------------------------- device ----
def quantize_row_q8_1(x, K: int | None = None, out=None, stream=None):
    """x: float32 cuda [N, K] (row = one activation column) -> uint8 cuda
    [N, pad(K)/32*36] block_q8_1."""
    import torch
    N, Kx = x.shape
    K = Kx if K is None else K
    kp = pad_k(K)
    if out is None:
        out = torch.empty((N, kp // 32 * BLOCK_Q8_1_BYTES), dtype=torch.uint8, device=x.device)
    _check(lib().q4k_quantize_row_q8_1(_ptr(x), _ptr(out), K, x.stride(0), kp, N, _stream(stream)),
           "q4k_quantize_row_q8_1")
    return out


def _entry(wtype: int, q4k_name: str, q6k_name: str):
    if wtype == GGML_TYPE_Q4_K:
        return q4k_name, getattr(lib(), q4k_name)
    if wtype == GGML_TYPE_Q6_K:
        return q6k_name, getattr(lib(), q6k_name)
    raise ValueError(f"weight type {wtype} has no GEMV here")


def mul_mat_vec_q(w_q, K: int, x, out=None, workspace=None, stream=None, wtype: int = GGML_TYPE_Q4_K):
    """ggml_cuda_mul_mat_vec_q: Q4_K [M, K/256*144] or (wtype GGML_TYPE_Q6_K)
    Q6_K [M, K/256*210] (uint8 cuda) x F32 [N, K] -> F32 [N, M] (row c of the
    result = column c of ggml's dst)."""
    import torch
    M = w_q.shape[0]
    N = x.shape[0]
    if out is None:
        out = torch.empty((N, M), dtype=torch.float32, device=x.device)
    ws_bytes = workspace.numel() * workspace.element_size() if workspace is not None else 0
    name, fn = _entry(wtype, "q4k_mul_mat_vec_q", "q6k_mul_mat_vec_q")
    _check(fn(_ptr(w_q), K, M, w_q.stride(0), _ptr(x), N, x.stride(0) * 4, _ptr(out), out.stride(0) * 4,
              _ptr(workspace), ws_bytes, _stream(stream)), name)
    return out


def mul_mat_vec_q_sums(w_q, K: int, x, workspace=None, stream=None, wtype: int = GGML_TYPE_Q4_K):
    """The parity form of mul_mat_vec_q: the production launch's SUMS
    variant.  Returns (dst F32 [N, M], sums int32, sq int32 or None): Q4_K
    sums [N, M, K/32] of q4*q8 per sub-block and sq [N, K/32] of q8; Q6_K
    sums [N, M, K/16] of (q - 32)*q8 per 16-weight group."""
    import torch
    M = w_q.shape[0]
    N = x.shape[0]
    dev = x.device
    out = torch.empty((N, M), dtype=torch.float32, device=dev)
    ws_bytes = workspace.numel() * workspace.element_size() if workspace is not None else 0
    args = (_ptr(w_q), K, M, w_q.stride(0), _ptr(x), N, x.stride(0) * 4, _ptr(out), out.stride(0) * 4,
            _ptr(workspace), ws_bytes)
    if wtype == GGML_TYPE_Q4_K:
        sums = torch.empty((N, M, K // 32), dtype=torch.int32, device=dev)
        sq = torch.empty((N, K // 32), dtype=torch.int32, device=dev)
        _check(lib().q4k_mul_mat_vec_q_sums(*args, _ptr(sums), _ptr(sq), _stream(stream)), "q4k_mul_mat_vec_q_sums")
        return out, sums, sq
    if wtype == GGML_TYPE_Q6_K:
        sums = torch.empty((N, M, K // 16), dtype=torch.int32, device=dev)
        _check(lib().q6k_mul_mat_vec_q_sums(*args, _ptr(sums), _stream(stream)), "q6k_mul_mat_vec_q_sums")
        return out, sums, None
    raise ValueError(f"weight type {wtype} has no GEMV here")


def mul_mat_vec_q_fused(w_q, K: int, x, gate=None, x_bias=None, gate_bias=None, glu_op: int = GLU_OP_SWIGLU,
                        out=None, stream=None, wtype: int = GGML_TYPE_Q4_K):
    """One column with the fused epilogue: dst = x_bias + w_q . x, or with a
    gate weight glu(w_q . x + x_bias, gate . x + gate_bias) -> F32 [1, M]."""
    import torch
    M = w_q.shape[0]
    if out is None:
        out = torch.empty((1, M), dtype=torch.float32, device=x.device)
    f = q4k_fusion(_ptr(x_bias), _ptr(gate), _ptr(gate_bias), glu_op)
    _check(lib().q4k_mul_mat_vec_q_fused(wtype, _ptr(w_q), K, M, w_q.stride(0), _ptr(x), ctypes.byref(f),
                                         _ptr(out), _stream(stream)), "q4k_mul_mat_vec_q_fused")
    return out


def op_mul_mat_vec_q(w_q, K: int, q8, ncols: int, row_low: int = 0, row_high: int | None = None,
                     out=None, nrows_dst: int | None = None, stream=None, wtype: int = GGML_TYPE_Q4_K):
    """ggml_cuda_op_mul_mat_vec_q: rows [row_low, row_high) of a contiguous
    Q4_K (or Q6_K) weight (w_q holds exactly those rows) x pre-quantised Q8_1
    columns."""
    import torch
    if row_high is None:
        row_high = row_low + w_q.shape[0]
    rows = row_high - row_low
    nrows_dst = rows if nrows_dst is None else nrows_dst
    if out is None:
        out = torch.empty((ncols, nrows_dst), dtype=torch.float32, device=q8.device)
    padded = q8.shape[1] // BLOCK_Q8_1_BYTES * 32
    name, fn = _entry(wtype, "q4k_op_mul_mat_vec_q", "q6k_op_mul_mat_vec_q")
    _check(fn(_ptr(w_q), K, row_low, row_high, _ptr(q8), ncols, padded, _ptr(out), nrows_dst,
              _stream(stream)), name)
    return out


def make_tensor(type_id: int, ne, nb, data_ptr: int) -> q4k_tensor:
    t = q4k_tensor()
    t.type = type_id
    for i in range(4):
        t.ne[i] = ne[i] if i < len(ne) else 1
    last = nb[-1] * (ne[len(nb) - 1] if len(nb) else 1)
    for i in range(4):
        t.nb[i] = nb[i] if i < len(nb) else last
    t.data = data_ptr
    return t


def ggml_mul_mat_vec_q(src0: q4k_tensor, src1: q4k_tensor, dst: q4k_tensor, ids=None, fusion=None,
                       workspace=None, stream=None) -> int:
    """Descriptor form; returns the status (Q4K_EUNSUPPORTED means: fall back)."""
    ws_bytes = workspace.numel() * workspace.element_size() if workspace is not None else 0
    return int(lib().q4k_ggml_mul_mat_vec_q(ctypes.byref(src0), ctypes.byref(src1),
                                            ctypes.byref(ids) if ids is not None else None,
                                            ctypes.byref(dst),
                                            ctypes.byref(fusion) if fusion is not None else None,
                                            _ptr(workspace), ws_bytes, _stream(stream)))


def subblock_sums(w_q, K: int, q8, ncols: int, stream=None):
    """Returns (sqq int32 [N, M, K/32], sq int32 [N, K/32]) on the device."""
    import torch
    M = w_q.shape[0]
    sqq = torch.empty((ncols, M, K // 32), dtype=torch.int32, device=q8.device)
    sq = torch.empty((ncols, K // 32), dtype=torch.int32, device=q8.device)
    _check(lib().q4k_subblock_sums(_ptr(w_q), K, M, w_q.stride(0), _ptr(q8), ncols,
                                   q8.shape[1] // BLOCK_Q8_1_BYTES, _ptr(sqq), _ptr(sq),
                                   _stream(stream)), "q4k_subblock_sums")
    return sqq, sq


def group_sums_q6_K(w_q, K: int, q8, ncols: int, stream=None):
    """Q6_K parity probe: int32 [N, M, K/16] sums of (q - 32) * q8 per
    16-weight scale group, on the device."""
    import torch
    M = w_q.shape[0]
    s16 = torch.empty((ncols, M, K // 16), dtype=torch.int32, device=q8.device)
    _check(lib().q6k_group_sums(_ptr(w_q), K, M, w_q.stride(0), _ptr(q8), ncols,
                                q8.shape[1] // BLOCK_Q8_1_BYTES, _ptr(s16), _stream(stream)),
           "q6k_group_sums")
    return s16


def set_geometry_override(rows_per_tile: int = 0, waves_per_wg: int = 0, workgroups: int = 0,
                          kernel: int = 0):
    _check(lib().q4k_set_geometry_override(rows_per_tile, waves_per_wg, workgroups, kernel),
           "q4k_set_geometry_override")


def set_pipeline_override(slots: int = 0, prologue: int = -1):
    _check(lib().q4k_set_pipeline_override(slots, prologue), "q4k_set_pipeline_override")


def geometry(K: int, M: int, N: int, wtype: int = GGML_TYPE_Q4_K, route: str = "f32") -> dict:
    """The launch of an (M x K) x (K x N) product: route "f32" quantises
    the F32 activation inside the GEMV launch, "q8_1" runs on a Q8_1
    activation (op_mul_mat_vec_q, or mul_mat_vec_q with a workspace where
    it quantises separately), "gate" / "bias" the one-column launch with
    that fused epilogue (mul_mat_vec_q_fused)."""
    out = (ctypes.c_int32 * 8)()
    if route in ("gate", "bias"):
        if N != 1:
            raise ValueError("fused geometry: one column")
        name, fn = _entry(wtype, "q4k_gemv_geometry_fused", "q6k_gemv_geometry_fused")
        _check(fn(K, M, 1 if route == "gate" else 0, ctypes.cast(out, _P)), name)
    elif route == "q8_1":
        name, fn = _entry(wtype, "q4k_gemv_geometry_q8_1", "q6k_gemv_geometry_q8_1")
    else:
        name, fn = _entry(wtype, "q4k_gemv_geometry", "q6k_gemv_geometry")
    if route not in ("gate", "bias"):
        _check(fn(K, M, N, ctypes.cast(out, _P)), name)
    keys = ("rows_per_tile", "waves_per_wg", "workgroups", "lds_bytes", "cols_per_launch", "fused",
            "kernel", "rows_per_step")
    return dict(zip(keys, list(out)))


# ----------------------------------------------------- operators of a batch ----
def _new(shape, dtype, device, stream):
    """An uninitialised tensor that the allocator ties to the stream of the call."""
    import torch
    if stream is None:
        return torch.empty(shape, dtype=dtype, device=device)
    with torch.cuda.stream(stream):
        return torch.empty(shape, dtype=dtype, device=device)


def _need(ok, what):
    """The binding's own checks: what the C ABI cannot see of a tensor."""
    if not ok:
        raise ValueError(what)


def _stream_of(stream, device):
    """The stream of a call on `device`: torch's current one unless given.
    (Without torch.cuda.current_stream, which costs as much as a launch.)"""
    if stream is not None:
        return stream.cuda_stream
    import torch
    return torch._C._cuda_getCurrentRawStream(device)


def _rows(t, dtype, shape, device, what):
    """The row stride of t, checked to be of dtype and shape (n, m) on device (its number) with contiguous rows."""
    strides = t.stride()
    if t.dtype is not dtype or t.shape != shape or t.get_device() != device or (strides[1] != 1 and shape[1] > 1):
        raise ValueError(f"{what}: {dtype} {list(shape)} with contiguous rows on device {device} expected")
    return strides[0]


def _type16(t):
    import torch
    if t.dtype == torch.float16:
        return GGML_TYPE_F16
    if t.dtype == torch.bfloat16:
        return GGML_TYPE_BF16
    raise ValueError(f"{t.dtype}: float16 or bfloat16 expected")


def _vector(t, dtype, shape, device, what):
    """The address of a contiguous device vector of shape (n,) (None: any n), or None for None."""
    if t is None:
        return None
    if t.dtype is not dtype or (t.dim() != 1 if shape is None else t.shape != shape) or t.get_device() != device or not t.is_contiguous():
        raise ValueError(f"{what}: contiguous {dtype} {'vector' if shape is None else list(shape)} on device {device} expected")
    return t.data_ptr()


def _ws(workspace, device):
    if workspace is None:
        return None, 0
    if workspace.get_device() != device or not workspace.is_contiguous():
        raise ValueError(f"workspace: contiguous on device {device} expected")
    return workspace.data_ptr(), workspace.nbytes


class LoraAdapters:
    """The low-rank adapters of one projection: a [adapters, rank, K] and
    b [adapters, M, rank] of float16 or bfloat16 (rows contiguous), scale F32
    [adapters] or None (1), ranks int32 [adapters] or None (all of rank).
    Described once, used by every lora_add; the tensors are kept alive."""

    def __init__(self, a, b, scale=None, ranks=None):
        import torch
        _need(a.is_cuda, "a, b: device tensors expected")
        _need(a.dim() == 3 and b.dim() == 3 and a.dtype == b.dtype and a.device == b.device and
              a.shape[0] == b.shape[0] and a.shape[1] == b.shape[2], "a [adapters, rank, K], b [adapters, M, rank] of one type")
        _need(a.numel() == 0 or (a.stride(2) == 1 or a.shape[2] == 1), "rows of a are not contiguous")
        _need(b.numel() == 0 or (b.stride(2) == 1 or b.shape[2] == 1), "rows of b are not contiguous")
        n = a.shape[0]
        self.tensors = (a, b, scale, ranks)
        self.K, self.M, self.rank, self.device, self.index = a.shape[2], b.shape[1], a.shape[1], a.device, a.get_device()
        self.desc = q4k_lora(_type16(a), self.rank, n, a.data_ptr(), a.stride(1) * 2, a.stride(0) * 2, b.data_ptr(),
                             b.stride(1) * 2, b.stride(0) * 2, _vector(scale, torch.float32, (n,), a.get_device(), "scale"),
                             _vector(ranks, torch.int32, (n,), a.get_device(), "ranks"))
        self._ref = ctypes.byref(self.desc)


def lora_workspace(adapters: LoraAdapters, n_tokens: int):
    """A workspace for lora_add of up to n_tokens tokens."""
    import torch
    n = int(lib().q4k_lora_workspace_bytes(adapters._ref, adapters.K, adapters.M, n_tokens))
    return torch.empty(max(n, 16), dtype=torch.uint8, device=adapters.device)


def lora_add(adapters: LoraAdapters, x, ids, base=None, out=None, workspace=None, stream=None):
    """base + the tokens' adapters' products: F32 x [N, K], int32 ids [N]
    (outside [0, adapters): none), base F32 [N, M] or None (zeros) -> F32
    [N, M].  out may be base: the shared projection's result is then added to
    in place."""
    import torch
    f32, dev, K, M, N = torch.float32, adapters.index, adapters.K, adapters.M, x.shape[0]
    shape = (N, M)
    ldx = _rows(x, f32, (N, K), dev, "x")
    if out is None:
        out = _new(shape, f32, adapters.device, stream)
    ldo = _rows(out, f32, shape, dev, "out")
    bp, ldb = (base.data_ptr(), _rows(base, f32, shape, dev, "base")) if base is not None else (None, 0)
    ws, ws_bytes = _ws(workspace, dev)
    st = lib().q4k_lora_add(adapters._ref, K, M, x.data_ptr(), N, ldx * 4, _vector(ids, torch.int32, (N,), dev, "ids"), bp, ldb * 4,
                            out.data_ptr(), ldo * 4, ws, ws_bytes, _stream_of(stream, dev))
    if st != Q4K_OK:
        raise Q4KError(st, "q4k_lora_add")
    return out


class KVPages:
    """Keys and values k, v [pages, page_size, heads_kv, head_dim] of float16 or
    bfloat16 (any strides, the last dimension contiguous) and the page numbers:
    table int32 [requests, pages per request] (a prefix: [pages of it] or None
    for the pages in order).  A contiguous prefix [tokens, heads_kv, head_dim] is
    k[None], v[None].  The tensors are kept alive; their contents and the table's
    may change between calls."""

    def __init__(self, k, v, table=None):
        import torch
        _need(k.is_cuda, "k, v: device tensors expected")
        _need(k.dim() == 4 and k.shape == v.shape and k.dtype == v.dtype and k.device == v.device and k.numel() > 0,
              "k, v: [pages, page_size, heads_kv, head_dim] of one type and shape expected")
        _need(k.stride(3) == 1 and v.stride(3) == 1, "head_dim of k, v is not contiguous")
        self.tensors = (k, v, table)
        self.type, self.heads, self.dim, self.device = _type16(k), k.shape[2], k.shape[3], k.get_device()
        self.rows, stride, length = None, 0, k.shape[0]
        if table is not None:
            _need(table.dtype == torch.int32 and table.dim() in (1, 2) and table.device == k.device and
                  (table.stride(-1) == 1 or table.shape[-1] <= 1), "table: int32 with contiguous rows expected")
            length = table.shape[-1]
            if table.dim() == 2:
                self.rows, stride = table.shape[0], table.stride(0)
        self.desc = q4k_kv_pages(k.data_ptr(), v.data_ptr(), k.shape[0], k.shape[1], *(k.stride(i) * 2 for i in range(3)),
                                 *(v.stride(i) * 2 for i in range(3)), table.data_ptr() if table is not None else None,
                                 stride, length)
        self._p = ctypes.pointer(self.desc)


def _prefix_attn_args(q, prefix, n_prefix, suffix, suffix_len, max_suffix, n_q, q_start, scale, out, lse):
    import torch
    n, heads, dim = q.shape
    dev, dtype = q.get_device(), q.dtype
    cache = suffix if prefix is None else prefix
    if cache is None or cache.dim != dim or cache.device != dev or (q.stride(2) != 1 and dim > 1):
        raise ValueError("q: [tokens, heads, head_dim] with contiguous dimensions, of the caches' head_dim and device expected")
    if suffix is not None and cache is not suffix and (suffix.heads, suffix.dim, suffix.type, suffix.device) != (cache.heads, dim, cache.type, dev):
        raise ValueError("prefix, suffix: one type, number of heads, head_dim and device expected")
    qt, es = (GGML_TYPE_F32, 4) if dtype is torch.float32 else (_type16(q), 2)
    start = None
    if n_q is None:  # one token a request; as many as there are where q_start tells
        n_q = 1 if q_start is None else n
    if q_start is not None:
        start = _vector(q_start, torch.int32, None, dev, "q_start")
        requests = q_start.shape[0] - 1
        _need(requests >= 0, "q_start: requests + 1 entries expected")
    else:
        requests = n // n_q if n_q else 0
    lens = own = None
    if max_suffix:
        _need(suffix is not None and suffix_len is not None, "max_suffix without suffix and suffix_len")
        lens = _vector(suffix_len, torch.int32, (requests,), dev, "suffix_len")
        own = suffix._p
        if suffix.tensors[2] is None:
            if requests:  # the call's own description: pages in order, as many for each request
                own = ctypes.pointer(q4k_kv_pages.from_buffer_copy(suffix.desc))
                own.contents.table_len = suffix.desc.n_pages // requests
        elif suffix.rows != requests and (requests != 1 or suffix.rows == 0):
            raise ValueError("suffix: a table row for each request expected")
    if n_prefix and (prefix is None or prefix.rows not in (None, 1)):
        raise ValueError("n_prefix without a prefix of one table row")
    if out is None:
        out = q
    elif out.shape != q.shape or out.dtype is not dtype or out.get_device() != dev or (out.stride(2) != 1 and dim > 1):
        raise ValueError("out: shape, type and device of q with contiguous dimensions expected")
    if lse is not None:
        if lse.shape != (n, heads) or lse.dtype is not torch.float32 or lse.get_device() != dev or not lse.is_contiguous():
            raise ValueError("lse: contiguous float32 [tokens, heads] expected")
        lse = lse.data_ptr()
    return q4k_prefix_attn_args(
        qt, cache.type, heads, cache.heads, dim, dim ** -0.5 if scale is None else scale, n, requests, n_q,
        start, q.data_ptr(), q.stride(0) * es, q.stride(1) * es, prefix._p if n_prefix else None, n_prefix,
        own, lens, max_suffix, out.data_ptr(), out.stride(0) * es, out.stride(1) * es, lse)


def prefix_attention_workspace(q, prefix, n_prefix, suffix=None, suffix_len=None, max_suffix=0, n_q=None, q_start=None):
    """A workspace for prefix_attention calls of these sizes."""
    import torch
    args = _prefix_attn_args(q, prefix, n_prefix, suffix, suffix_len, max_suffix, n_q, q_start, None, None, None)
    n = int(lib().q4k_prefix_attn_workspace_bytes(ctypes.byref(args)))
    return torch.empty(max(n, 16), dtype=torch.uint8, device=q.device)


def prefix_attention(q, prefix, n_prefix, suffix=None, suffix_len=None, max_suffix=0, n_q=None, q_start=None, scale=None,
                     out=None, lse=None, workspace=None, stream=None):
    """Attention of a batch over n_prefix tokens that all requests share
    (prefix, read once for all) and each request's own suffix_len[r] <=
    max_suffix tokens (suffix), the last of which are the queries' own.
    q [tokens, heads, head_dim], float32 or the caches' type: n_q tokens a
    request (1), or q_start int32 [requests + 1] with at most n_q each (all tokens;
    a bound near the longest request runs faster, tokens past it are left out).
    Returns out of q's type; lse F32 [tokens, heads] receives the rows' log-sum-exp."""
    if out is None:
        out = _new(q.shape, q.dtype, q.device, stream)
    args = _prefix_attn_args(q, prefix, n_prefix, suffix, suffix_len, max_suffix, n_q, q_start, scale, out, lse)
    dev = q.get_device()
    ws, ws_bytes = _ws(workspace, dev)
    st = lib().q4k_prefix_attn(ctypes.byref(args), ws, ws_bytes, _stream_of(stream, dev))
    if st != Q4K_OK:
        raise Q4KError(st, "q4k_prefix_attn")
    return out


def logits_adjust(logits, repeat=None, frequency=None, presence=None, history=None, history_start=None, bias_ids=None,
                  bias=None, bias_start=None, mask=None, mask_rows=None, out=None, stream=None):
    """Penalties for repeated tokens, biases and grammar masks on F32 logits
    [N, V] (q4k_logits_adjust).  repeat, frequency, presence F32 [N]; history
    int32 with history_start int64 [N + 1]; bias_ids int32 and bias F32 with
    bias_start int64 [N + 1]; mask int32 [masks, ceil(V / 32)] with mask_rows
    int32 [N] (outside [0, masks): none).  out may be logits."""
    import torch
    f32, i32, i64 = torch.float32, torch.int32, torch.int64
    _need(logits.is_cuda, "logits: a device tensor expected")
    N, V = logits.shape
    dev = logits.get_device()
    shape, per_row, starts = (N, V), (N,), (N + 1,)
    ldx = _rows(logits, f32, shape, dev, "logits")
    if out is None:
        out = _new(shape, f32, logits.device, stream)
    ldo = _rows(out, f32, shape, dev, "out")
    if (history is None) != (history_start is None):
        raise ValueError("history without history_start")
    if (bias_ids is None) != (bias is None) or (bias_ids is None) != (bias_start is None):
        raise ValueError("bias_ids, bias and bias_start go together")
    h = hs = bi = bv = bs = m = mr = None
    nh = nb = masks = nbm = 0
    if history is not None:
        h, hs, nh = _vector(history, i32, None, dev, "history"), _vector(history_start, i64, starts, dev, "history_start"), history.shape[0]
        if nh == 0:
            h = hs = None
    if bias_ids is not None:
        nb = bias_ids.shape[0]
        bi, bv = _vector(bias_ids, i32, None, dev, "bias_ids"), _vector(bias, f32, (nb,), dev, "bias")
        bs = _vector(bias_start, i64, starts, dev, "bias_start")
        if nb == 0:
            bi = bv = bs = None
    if mask is not None:
        masks, words = mask.shape
        ldm = _rows(mask, i32, (masks, words), dev, "mask")
        if words < -(-V // 32):
            raise ValueError(f"mask: int32 [masks, {-(-V // 32)}] expected")
        if mask_rows is None and masks < N:
            raise ValueError("mask: a row for each row of logits, or mask_rows, expected")
        mr = _vector(mask_rows, i32, per_row, dev, "mask_rows")
        if masks:
            m, nbm = mask.data_ptr(), ldm * 4
        else:
            mr = None
    elif mask_rows is not None:
        raise ValueError("mask_rows without mask")
    r = q4k_logits_rules(_vector(repeat, f32, per_row, dev, "repeat"), _vector(frequency, f32, per_row, dev, "frequency"),
                         _vector(presence, f32, per_row, dev, "presence"), h, hs, nh, bi, bv, bs, nb, m, masks, nbm, mr)
    st = lib().q4k_logits_adjust(logits.data_ptr(), V, N, ldx * 4, ctypes.byref(r), out.data_ptr(), ldo * 4, _stream_of(stream, dev))
    if st != Q4K_OK:
        raise Q4KError(st, "q4k_logits_adjust")
    return out


# ------------------------------------------------- operators of a decode step ----
ROPE_NORMAL, ROPE_NEOX = 0, 2


def _types():
    """The ggml type and bytes of a value of the float types that rows may have."""
    import torch
    return {torch.float32: (GGML_TYPE_F32, 4), torch.float16: (GGML_TYPE_F16, 2), torch.bfloat16: (GGML_TYPE_BF16, 2)}


_TYPES = {}


def _float_type(t, what):
    if not _TYPES:
        _TYPES.update(_types())
    got = _TYPES.get(t.dtype)
    if got is None:
        raise ValueError(f"{what}: float32, float16 or bfloat16 expected, not {t.dtype}")
    return got


def _on_device(name, device, *args):
    """Calls the library with `device` (its number) as the current one."""
    import torch
    f = getattr(lib(), name)
    if torch._C._cuda_getDevice() == device:
        st = f(*args)
    else:
        with torch.cuda.device(device):
            st = f(*args)
    if st != Q4K_OK:
        raise Q4KError(st, name)


class Rope:
    """The norms and position rotation of a model's heads, described once for
    every rope call (include/q4k_step.h): n_rot of head_dim dimensions (all)
    are rotated, mode "normal" (pairs of neighbours) or "neox" (of halves);
    freq_factors F32 [n_rot / 2]; YaRN with ext_factor not 0 and n_ctx_orig;
    q_norm, k_norm F32 [head_dim], eps of the norms.  The tensors are kept alive."""

    def __init__(self, head_dim, n_rot=None, mode="normal", freq_base=10000.0, freq_scale=1.0, ext_factor=0.0, attn_factor=1.0,
                 beta_fast=32.0, beta_slow=1.0, n_ctx_orig=0, freq_factors=None, q_norm=None, k_norm=None, eps=1e-6):
        import torch
        _need(mode in ("normal", "neox"), 'mode: "normal" or "neox" expected')
        n_rot = head_dim if n_rot is None else n_rot
        self.head_dim, self.device = head_dim, None
        self.tensors = (freq_factors, q_norm, k_norm)
        for t in self.tensors:
            if t is not None:
                _need(t.is_cuda, "freq_factors, q_norm, k_norm: device tensors expected")
                _need(self.device in (None, t.get_device()), "freq_factors, q_norm, k_norm: one device expected")
                self.device = t.get_device()
        dev, f32 = self.device, torch.float32
        self.q_norm, self.k_norm = _vector(q_norm, f32, (head_dim,), dev, "q_norm"), _vector(k_norm, f32, (head_dim,), dev, "k_norm")
        self.desc = q4k_rope_args(head_dim, n_rot, ROPE_NORMAL if mode == "normal" else ROPE_NEOX, eps, freq_base, freq_scale, ext_factor,
                                  attn_factor, beta_fast, beta_slow, n_ctx_orig, _vector(freq_factors, f32, (n_rot // 2,), dev, "freq_factors"))
        # (what the library refuses of it, here already: a call without tokens checks the description alone)
        st = lib().q4k_rope(ctypes.byref(self.desc), None)
        if st != Q4K_OK:
            raise Q4KError(st, "q4k_rope")


def _rope_rows(x, out, norm, tokens, dim, device, what):
    st, es = _float_type(x, what)
    dt, ds = (st, es) if out.dtype is x.dtype else _float_type(out, what)
    shape, strides, to = x.shape, x.stride(), out.stride()
    if len(shape) != 3 or shape[0] != tokens or shape[2] != dim or x.get_device() != device or (strides[2] != 1 and dim > 1):
        raise ValueError(f"{what}: [{tokens}, heads, {dim}] with contiguous dimensions on device {device} expected")
    if out.shape != shape or out.get_device() != device or (to[2] != 1 and dim > 1):
        raise ValueError(f"{what}_out: shape and device of {what} with contiguous dimensions expected")
    return ctypes.pointer(q4k_rope_rows(x.data_ptr(), out.data_ptr(), st, dt, shape[1], strides[0] * es, strides[1] * es, to[0] * ds,
                                        to[1] * ds, norm))


def rope(r: Rope, q, k, pos, q_out=None, k_out=None, stream=None):
    """The norms and rotation r of queries q [tokens, heads, head_dim] and keys k
    (either may be None) at int32 positions pos [tokens]; float32, float16 or
    bfloat16, results of the same type in new tensors, or in q_out, k_out, which
    may be q, k themselves or, of float32 rows, of 16 bits.  Returns (q_out, k_out)."""
    import torch
    some = q if q is not None else k
    if some is None:
        raise ValueError("q or k expected")
    dev, n = some.get_device(), some.shape[0]
    if dev < 0 or r.device not in (None, dev):
        raise ValueError("q, k: tensors on the description's device expected")
    args = q4k_rope_args.from_buffer_copy(r.desc)
    args.n_tokens, args.pos = n, _vector(pos, torch.int32, (n,), dev, "pos")
    if q is not None:
        if q_out is None:
            q_out = _new(q.shape, q.dtype, q.device, stream)
        args.q = _rope_rows(q, q_out, r.q_norm, n, r.head_dim, dev, "q")
    if k is not None:
        if k_out is None:
            k_out = _new(k.shape, k.dtype, k.device, stream)
        args.k = _rope_rows(k, k_out, r.k_norm, n, r.head_dim, dev, "k")
    _on_device("q4k_rope", dev, ctypes.byref(args), _stream_of(stream, dev))
    return q_out, k_out


TYPE_I8, TYPE_E4M3 = 24, 1000


class KV8Pages:
    """Keys and values in 8 bits: k, v [pages, page_size, heads_kv, head_dim] of
    int8 or float8_e4m3fn (any strides of multiples of 16, the last dimension
    contiguous), their scales F32 [pages, page_size / block, heads_kv] (of both
    with the same strides) and the page numbers: table int32 [requests, pages per request],
    or None for the pages in order, as many for each request.  The tensors are kept
    alive; their contents and the table's may change between calls."""

    def __init__(self, k, v, k_scale, v_scale, table=None):
        import torch
        _need(k.is_cuda, "k, v: device tensors expected")
        _need(k.dim() == 4 and k.shape == v.shape and k.dtype == v.dtype and k.device == v.device and k.numel() > 0,
              "k, v: [pages, page_size, heads_kv, head_dim] of one type and shape expected")
        _need(k.dtype in (torch.int8, torch.float8_e4m3fn), "k, v: int8 or float8_e4m3fn expected")
        _need(k.stride(3) == 1 and v.stride(3) == 1, "head_dim of k, v is not contiguous")
        pages, page, heads, dim = k.shape
        for s in (k_scale, v_scale):
            _need(s.dtype == torch.float32 and s.device == k.device and s.dim() == 3 and s.shape == k_scale.shape and
                  s.stride() == k_scale.stride() and s.shape[0] == pages and s.shape[2] == heads and s.shape[1] > 0 and page % s.shape[1] == 0,
                  "k_scale, v_scale: float32 [pages, page_size / block, heads_kv] of one layout expected")
        self.tensors = (k, v, k_scale, v_scale, table)
        self.heads, self.dim, self.device, self.rows, stride, length = heads, dim, k.get_device(), None, 0, pages
        if table is not None:
            _need(table.dtype == torch.int32 and table.dim() == 2 and table.device == k.device and
                  (table.stride(1) == 1 or table.shape[1] <= 1), "table: int32 [requests, pages] with contiguous rows expected")
            self.rows, length = table.shape
            stride = table.stride(0)
        self.desc = q4k_kv8_pages(TYPE_I8 if k.dtype == torch.int8 else TYPE_E4M3, heads, dim, page // k_scale.shape[1], k.data_ptr(), v.data_ptr(),
                                  pages, page, *(k.stride(i) for i in range(3)), *(v.stride(i) for i in range(3)), k_scale.data_ptr(),
                                  v_scale.data_ptr(), *(k_scale.stride(i) * 4 for i in range(3)),
                                  table.data_ptr() if table is not None else None, stride, length)
        self._p = ctypes.pointer(self.desc)

    def _of(self, requests):
        """The description for a call of so many requests."""
        if self.rows is None:
            if not requests:
                return self._p
            own = q4k_kv8_pages.from_buffer_copy(self.desc)  # pages in order, as many for each request
            own.table_len = self.desc.n_pages // requests
            return ctypes.pointer(own)
        _need(self.rows == requests or (requests == 1 and self.rows > 0) or not requests, "table: a row for each request expected")
        return self._p


def _kv8_requests(n, n_q, q_start, lens, device):
    """Requests, the most tokens of one, and the addresses of q_start and lens."""
    import torch
    start = None
    if n_q is None:  # one token a request; as many as there are where q_start tells
        n_q = 1 if q_start is None else n
    if q_start is not None:
        start = _vector(q_start, torch.int32, None, device, "q_start")
        requests = q_start.shape[0] - 1
        _need(requests >= 0, "q_start: requests + 1 entries expected")
    else:
        requests = n // n_q if n_q else 0
    return requests, n_q, start, _vector(lens, torch.int32, (requests,), device, "lens")


def _kv8_rows(name, pages, k, v, lens, max_len, n_q, q_start, stream):
    some = k if k is not None else v
    _need(some is not None, "k or v expected")
    t, es = _float_type(some, "k, v")
    dev, n, shape = pages.device, some.shape[0], (some.shape[0], pages.heads, pages.dim)
    requests, n_q, start, lens = _kv8_requests(n, n_q, q_start, lens, dev)
    at = []
    for x in (k, v):
        if x is None:
            at.append((None, 0, 0))
            continue
        strides = x.stride()
        if x.shape != shape or x.dtype is not some.dtype or x.get_device() != dev or strides[2] != 1:
            raise ValueError(f"k, v: {some.dtype} {list(shape)} with contiguous dimensions on device {dev} expected")
        at.append((x.data_ptr(), strides[0] * es, strides[1] * es))
    (kp, kt, kh), (vp, vt, vh) = at
    args = q4k_kv8_rows(pages._of(requests), t, n, requests, n_q, start, lens, max_len, kp, vp, kt, kh, vt, vh)
    _on_device(name, dev, ctypes.byref(args), _stream_of(stream, dev))


def kv8_store(pages: KV8Pages, k, v, lens, max_len, n_q=None, q_start=None, stream=None):
    """Writes the requests' new keys and values k, v [tokens, heads_kv, head_dim]
    (float32, float16 or bfloat16) into their pages: the last of each request's lens[r]
    <= max_len tokens (int32, with the new ones), n_q each (1), or those that q_start
    int32 [requests + 1] names, at most n_q each (all tokens)."""
    _need(k is not None and v is not None, "k and v expected")
    _kv8_rows("q4k_kv8_store", pages, k, v, lens, max_len, n_q, q_start, stream)


def kv8_load(pages: KV8Pages, k, v, lens, max_len, n_q=None, q_start=None, stream=None):
    """Reads each request's last tokens into k, v (either may be None), as the
    values that the pages' bytes stand for; requests and tokens as in kv8_store."""
    _kv8_rows("q4k_kv8_load", pages, k, v, lens, max_len, n_q, q_start, stream)
    return k, v


def _kv8_attn_args(q, pages, lens, max_len, n_q, q_start, scale, out, lse):
    dev = pages.device
    shape, strides = q.shape, q.stride()
    if len(shape) != 3 or shape[2] != pages.dim or q.get_device() != dev or (strides[2] != 1 and pages.dim > 1):
        raise ValueError("q: [tokens, heads, head_dim] with contiguous dimensions, of the cache's head_dim and device expected")
    n, heads, dim = shape
    t, es = _float_type(q, "q")
    requests, n_q, start, lens = _kv8_requests(n, n_q, q_start, lens, dev)
    if out is None:
        out = q
    to = out.stride()
    if out.shape != shape or out.dtype is not q.dtype or out.get_device() != dev or (to[2] != 1 and dim > 1):
        raise ValueError("out: shape, type and device of q with contiguous dimensions expected")
    if lse is not None:
        lse = _lse(lse, n, heads, dev)
    return q4k_kv8_attn_args(pages._of(requests), t, heads, dim ** -0.5 if scale is None else scale, n, requests, n_q, start, lens, max_len,
                             q.data_ptr(), strides[0] * es, strides[1] * es, out.data_ptr(), to[0] * es, to[1] * es, lse)


def _lse(lse, n, heads, device):
    import torch
    if lse.shape != (n, heads) or lse.dtype is not torch.float32 or lse.get_device() != device or not lse.is_contiguous():
        raise ValueError("lse: contiguous float32 [tokens, heads] expected")
    return lse.data_ptr()


def kv8_attention_workspace(q, pages: KV8Pages, lens, max_len, n_q=None, q_start=None):
    """A workspace for kv8_attention calls of these sizes."""
    import torch
    args = _kv8_attn_args(q, pages, lens, max_len, n_q, q_start, None, None, None)
    with torch.cuda.device(pages.device):
        n = int(lib().q4k_kv8_attn_workspace_bytes(ctypes.byref(args)))
    return torch.empty(max(n, 16), dtype=torch.uint8, device=q.device)


def kv8_attention(q, pages: KV8Pages, lens, max_len, n_q=None, q_start=None, scale=None, out=None, lse=None, workspace=None, stream=None):
    """Attention of a batch over its caches of 8 bits: q [tokens, heads, head_dim]
    (float32, float16 or bfloat16) are the last of each request's lens[r] <= max_len
    tokens (int32), n_q each (1), or those that q_start int32 [requests + 1] names, at
    most n_q each (all tokens; a bound near the longest request runs faster).  Returns
    out of q's type; lse F32 [tokens, heads] receives the rows' log-sum-exp."""
    if out is None:
        out = _new(q.shape, q.dtype, q.device, stream)
    args = _kv8_attn_args(q, pages, lens, max_len, n_q, q_start, scale, out, lse)
    dev = pages.device
    ws, ws_bytes = _ws(workspace, dev)
    _on_device("q4k_kv8_attn", dev, ctypes.byref(args), ws, ws_bytes, _stream_of(stream, dev))
    return out


def sample_workspace(logits):
    """A workspace for sample calls of up to these rows of logits [N, V]."""
    import torch
    N, V = logits.shape
    with torch.cuda.device(logits.device):
        n = int(lib().q4k_sample_workspace_bytes(V, N))
    return torch.empty(max(n, 16), dtype=torch.uint8, device=logits.device)


def sample(logits, uniform=None, temperature=None, top_k=None, top_p=None, min_p=None, out=None, logprob=None, workspace=None, stream=None):
    """The next token of each row of F32 logits [N, V]: temperature (1; 0: the
    largest), then top_k int32 (0: all), top_p (1: all) and min_p (0: all), F32 [N] each,
    drawn by uniform F32 [N] in [0, 1) (None: the largest logit).  Returns (tokens
    int32 [N], logprob F32 [N] or None): the logarithm of the token's share of what
    the cuts kept goes to logprob where one is given."""
    import torch
    f32 = torch.float32
    _need(logits.is_cuda, "logits: a device tensor expected")
    N, V = logits.shape
    dev, n = logits.get_device(), (N,)
    ldx = _rows(logits, f32, (N, V), dev, "logits")
    if out is None:
        out = _new(n, torch.int32, logits.device, stream)
    r = q4k_sample_rules(_vector(temperature, f32, n, dev, "temperature"), _vector(top_k, torch.int32, n, dev, "top_k"),
                         _vector(top_p, f32, n, dev, "top_p"), _vector(min_p, f32, n, dev, "min_p"), _vector(uniform, f32, n, dev, "uniform"))
    ws, ws_bytes = _ws(workspace, dev)
    _on_device("q4k_sample", dev, logits.data_ptr(), V, N, ldx * 4, ctypes.byref(r), _vector(out, torch.int32, n, dev, "out"),
               _vector(logprob, f32, n, dev, "logprob"), ws, ws_bytes, _stream_of(stream, dev))
    return out, logprob


# ------------------------------------------------------------------ GGUF ----
GGUF_ARRAY, GGUF_STRING = 9, 8
_GGUF_NP = {0: np.uint8, 1: np.int8, 2: np.uint16, 3: np.int16, 4: np.uint32, 5: np.int32, 6: np.float32,
            7: np.bool_, 10: np.uint64, 11: np.int64, 12: np.float64}


class GGUFFile:
    """A GGUF file opened with the library's reader (q4k_gguf_open).
    tensors: {name: dict(type, ne, offset, nbytes)}; tensor_bytes(name) is a
    zero-copy uint8 view of the mapped data, valid until close()."""

    def __init__(self, path: str):
        self._h = ctypes.c_void_p()
        _check(lib().q4k_gguf_open(os.fsencode(path), ctypes.byref(self._h)), f"q4k_gguf_open({path})")
        L = lib()
        self.version = int(L.q4k_gguf_version(self._h))
        self.alignment = int(L.q4k_gguf_alignment(self._h))
        self.data_offset = int(L.q4k_gguf_data_offset(self._h))
        self.tensors = {}
        for i in range(L.q4k_gguf_tensor_count(self._h)):
            ti = q4k_gguf_tensor_info()
            _check(L.q4k_gguf_get_tensor(self._h, i, ctypes.byref(ti)), "q4k_gguf_get_tensor")
            self.tensors[ti.name.decode()] = {"index": i, "type": ti.type, "ne": list(ti.ne)[:ti.n_dims],
                                              "offset": int(ti.offset), "nbytes": int(ti.nbytes),
                                              "data": ti.data}

    def metadata(self) -> dict:
        L = lib()
        out = {}
        for i in range(L.q4k_gguf_kv_count(self._h)):
            key = L.q4k_gguf_key(self._h, i).decode()
            t = L.q4k_gguf_kv_type(self._h, i)
            if t == GGUF_STRING:
                sp = ctypes.c_char_p()
                _check(L.q4k_gguf_get_str(self._h, i, ctypes.byref(sp)), key)
                out[key] = sp.value.decode()
            elif t == GGUF_ARRAY:
                et, n, dp = ctypes.c_int32(), ctypes.c_int64(), ctypes.c_void_p()
                _check(L.q4k_gguf_get_arr(self._h, i, ctypes.byref(et), ctypes.byref(n), ctypes.byref(dp)), key)
                if et.value == GGUF_STRING:
                    vals = []
                    for j in range(n.value):
                        sp = ctypes.c_char_p()
                        _check(L.q4k_gguf_get_arr_str(self._h, i, j, ctypes.byref(sp)), key)
                        vals.append(sp.value.decode())
                    out[key] = vals
                else:
                    dt = np.dtype(_GGUF_NP[et.value])
                    buf = (ctypes.c_uint8 * (n.value * dt.itemsize)).from_address(dp.value) if n.value else b""
                    out[key] = np.frombuffer(bytes(buf), dtype=dt).tolist()
            elif t in (6, 12):
                v = ctypes.c_double()
                _check(L.q4k_gguf_get_float(self._h, i, ctypes.byref(v)), key)
                out[key] = v.value
            else:
                v = ctypes.c_int64()
                _check(L.q4k_gguf_get_int(self._h, i, ctypes.byref(v)), key)
                out[key] = bool(v.value) if t == 7 else v.value
        return out

    def tensor_bytes(self, name: str) -> np.ndarray:
        t = self.tensors[name]
        if not t["nbytes"]:
            raise ValueError(f"{name}: block size of ggml type {t['type']} unknown")
        buf = (ctypes.c_uint8 * t["nbytes"]).from_address(t["data"])
        return np.frombuffer(buf, dtype=np.uint8)

    def weight_rows(self, name: str) -> np.ndarray:
        """A 2-D quantised weight as [rows, row bytes] (zero-copy view)."""
        t = self.tensors[name]
        rb = int(lib().q4k_ggml_row_size(t["type"], t["ne"][0]))
        return self.tensor_bytes(name).reshape(-1, rb)

    def close(self):
        if self._h:
            lib().q4k_gguf_close(self._h)
            self._h = ctypes.c_void_p()

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.close()
