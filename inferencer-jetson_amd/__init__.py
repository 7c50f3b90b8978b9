"""MI355X (gfx950) Q4_K / Q6_K dequant-GEMV: Python host mirror of the C ABI.

libqk.so (built from csrc/ by the Makefile) exports the C ABI declared in
include/qk.h.  This module binds it with ctypes and mirrors the reference's
host-side interface for the path (inferencer.cu:178-186 Tensor,
1101-1180 FastGPU, 1265-1278 batch_matvec): the same names, argument meaning
and error behaviour -- a failing call raises QKError("where: message") like
cuda_check (inferencer.cu:126-128).

Device buffers are passed as raw pointers; torch tensors (or anything with
data_ptr()) are accepted for convenience, torch being only the allocator and
stream provider.  There is no CPU fallback: if libqk.so is missing, loading
raises ImportError.
"""
from __future__ import annotations

import ctypes
import pathlib
from dataclasses import dataclass
from typing import Sequence

_HERE = pathlib.Path(__file__).resolve().parent
LIB_PATH = _HERE / "libqk.so"

F32, F16, Q4_K, Q6_K = 0, 1, 12, 14
Q6_K_SPLIT = 114   # Q6_K in the split row layout of qk_q6k_split (16-byte aligned fields)
BLOCK_BYTES = {Q4_K: 144, Q6_K: 210, Q6_K_SPLIT: 210}
QUANT_TYPES = (Q4_K, Q6_K, Q6_K_SPLIT)
STORAGE_NAMES = {F32: "FP32", F16: "FP16", Q4_K: "Q4_K", Q6_K: "Q6_K", Q6_K_SPLIT: "Q6_K (split)"}
MAX_FUSED = 8
# Types of paged cache rows, besides F16.
I8, F8_E4M3, I4 = 24, 120, 121
ROPE_SCALING = {"none": 0, "linear": 1, "llama3": 2, "yarn": 3}

QK_OK = 0
QK_ERR_INVALID_ARG = 1
QK_ERR_SHAPE = 2
QK_ERR_TYPE = 3
QK_ERR_ALIGN = 4
QK_ERR_DEVICE = 5
QK_ERR_LIMIT = 6
QK_ERR_FORMAT = 7
QK_ERR_IO = 8


class QKError(RuntimeError):
    """A non-zero qk status; .status holds the code."""

    def __init__(self, where: str, status: int, detail: str):
        super().__init__(f"{where}: {detail}")
        self.status = status


class qk_matrix(ctypes.Structure):
    _fields_ = [("type", ctypes.c_int), ("rows", ctypes.c_int),
                ("w", ctypes.c_void_p), ("y", ctypes.c_void_p)]


class qk_batch_token(ctypes.Structure):
    """One token of a ragged decode batch (include/qk.h)."""
    _fields_ = [("pos", ctypes.c_int32), ("seq", ctypes.c_int32), ("kv_row", ctypes.c_int64)]


class qk_llama_config(ctypes.Structure):
    _fields_ = [(n, ctypes.c_int) for n in ("dim", "layers", "heads", "kv_heads", "hidden", "vocab", "context")] + \
               [("eps", ctypes.c_float), ("rope_theta", ctypes.c_float)]


class qk_llama_layer(ctypes.Structure):
    _fields_ = [(n, ctypes.c_int) for n in ("q_type", "k_type", "v_type", "o_type", "gate_type", "up_type",
                                             "down_type")] + \
               [(n, ctypes.c_void_p) for n in ("q", "k", "v", "o", "gate", "up", "down", "attn_norm", "ffn_norm")]


class qk_llama_weights(ctypes.Structure):
    _fields_ = [("embd_type", ctypes.c_int), ("token_embd", ctypes.c_void_p), ("output_type", ctypes.c_int),
                ("output", ctypes.c_void_p), ("output_norm", ctypes.c_void_p),
                ("layers", ctypes.POINTER(qk_llama_layer))]


class qk_llama_memory(ctypes.Structure):
    _fields_ = [("weight_copies", ctypes.c_uint64), ("kv_cache", ctypes.c_uint64), ("buffers", ctypes.c_uint64)]


class qk_gguf_tensor(ctypes.Structure):
    """One tensor-table entry of a GGUF file (include/qk.h)."""
    _fields_ = [("name", ctypes.c_char_p), ("type", ctypes.c_int), ("n_dims", ctypes.c_int),
                ("dims", ctypes.c_int64 * 4), ("offset", ctypes.c_uint64), ("bytes", ctypes.c_uint64),
                ("host", ctypes.c_void_p), ("device", ctypes.c_void_p)]


class qk_paged_kv(ctypes.Structure):
    """One layer's paged cache (include/qk.h)."""
    _fields_ = [(n, ctypes.c_int) for n in ("type", "kv_heads", "head_dim", "page_rows")] + \
               [("pages", ctypes.c_int64)] + [(n, ctypes.c_void_p) for n in ("key", "value", "key_scale", "value_scale")]


class qk_paged_seq(ctypes.Structure):
    """One sequence of a call over a paged cache (include/qk.h)."""
    _fields_ = [(n, ctypes.c_int32) for n in ("first", "count", "pos", "table")]


class qk_paged_batch(ctypes.Structure):
    """The sequences of a call over a paged cache (include/qk.h)."""
    _fields_ = [("page_table", ctypes.c_void_p), ("table_rows", ctypes.c_int), ("table_stride", ctypes.c_int),
                ("seqs", ctypes.c_void_p)] + \
               [(n, ctypes.c_int) for n in ("n_seqs", "n_tokens", "max_count", "max_rows")]


class qk_attention_terms(ctypes.Structure):
    """What attention adds to its scores and which rows tokens see (include/qk.h)."""
    _fields_ = [("cap", ctypes.c_float), ("window", ctypes.c_int), ("slopes", ctypes.c_void_p),
                ("prefix", ctypes.c_void_p)]


class qk_page_pool(ctypes.Structure):
    """A pool of pages and the table of those that hold them (include/qk.h)."""
    _fields_ = [("page_table", ctypes.c_void_p), ("table_rows", ctypes.c_int), ("table_stride", ctypes.c_int),
                ("refs", ctypes.c_void_p), ("pages", ctypes.c_int64), ("page_rows", ctypes.c_int),
                ("layers", ctypes.POINTER(qk_paged_kv)), ("n_layers", ctypes.c_int)]


class qk_rope_scaling(ctypes.Structure):
    """Scaling of rotary frequencies (include/qk.h)."""
    _fields_ = [("type", ctypes.c_int)] + \
               [(n, ctypes.c_float) for n in ("factor", "low_freq_factor", "high_freq_factor", "original_context",
                                              "beta_fast", "beta_slow", "attention_factor")]


_i, _vp, _f = ctypes.c_int, ctypes.c_void_p, ctypes.c_float
# name -> (restype, argtypes), exactly the declarations of include/qk.h.
SIGNATURES = {
    "qk_status_string": (ctypes.c_char_p, [_i]),
    "qk_last_error": (ctypes.c_char_p, []),
    "qk_block_bytes": (_i, [_i]),
    "qk_tensor_bytes": (ctypes.c_int64, [_i, ctypes.c_int64, ctypes.c_int64]),
    "qk_gemv_f32": (_i, [_i, _vp, _vp, _vp, _i, _i, _vp]),
    "qk_gemv_multi_f32": (_i, [ctypes.POINTER(qk_matrix), _i, _vp, _i, _vp]),
    "qk_gemv_batched_workspace_bytes": (ctypes.c_size_t, [_i, _i, _i]),
    "qk_gemv_batched_f32": (_i, [_i, _vp, _vp, _i, _vp, _i, _i, _i, _i, _vp, ctypes.c_size_t, _vp]),
    "qk_gemv_multi_batched_f32": (_i, [ctypes.POINTER(qk_matrix), _i, _vp, _i, _i, _i, _vp, ctypes.c_size_t, _vp]),
    "qk_dequant_rows": (_i, [_i, _vp, _vp, _i, _i, _i, _vp]),
    "qk_embedding": (_i, [_i, _vp, _vp, _i, _vp, _i, _i, _vp]),
    "qk_q6k_split": (_i, [_vp, _vp, _i, _i, _vp]),
    "qk_gemv_argmax_workspace_bytes": (ctypes.c_size_t, []),
    "qk_gemv_argmax_f32": (_i, [_i, _vp, _vp, _vp, _i, _i, _vp, _vp, _vp]),
    "qk_gemv_argmax_f32_noalloc": (_i, [_i, _vp, _vp, _vp, _i, _i, _vp, _vp]),
    "qk_quantize_x32": (_i, [_vp, _i, _vp, _i, _vp, _i, _i, _i, _vp]),
    "qk_gemv_multi_i8": (_i, [ctypes.POINTER(qk_matrix), _i, _vp, _vp, _i, _vp]),
    "qk_llama_set_int8": (_i, [_vp, _i, _i]),
    "qk_rmsnorm_quantize_x32": (_i, [_vp, _i, _vp, _vp, _i, _vp, _i, _vp, _i, _i, _i, ctypes.c_float, _vp]),
    "qk_gemv_i8": (_i, [_i, _vp, _vp, _i, _vp, _i, _vp, _i, _i, _i, _i, _vp]),
    "qk_gemv_batched_i8": (_i, [_i, _vp, _vp, _i, _vp, _i, _vp, _i, _i, _i, _i, _vp, ctypes.c_size_t, _vp]),
    "qk_gemv_batched_i8_workspace_bytes": (ctypes.c_size_t, [_i, _i, _i]),
    "qk_gemv_multi_batched_i8": (_i, [ctypes.POINTER(qk_matrix), _i, _vp, _i, _vp, _i, _i, _i, _vp, ctypes.c_size_t,
                                      _vp]),
    "qk_ffn_batched_i8_workspace_bytes": (ctypes.c_size_t, [_i, _i, _i]),
    "qk_ffn_batched_i8": (_i, [_i, _vp, _i, _vp, _i, _vp, _vp, _i, _vp, _i, _vp, _i, _i, _i, _i, _i, _vp,
                               ctypes.c_size_t, _vp]),
    "qk_rmsnorm_f32": (_i, [_vp, _vp, _vp, _i, _i, _f, _vp]),
    "qk_rope_kv_write": (_i, [_vp, _vp, _vp, _vp, _vp, _vp, _vp, _i, _i, _i, _i, _i, _i, _vp]),
    "qk_attention_f32": (_i, [_vp, _vp, _vp, _vp, _i, _i, _i, _i, _i, _i, _vp]),
    "qk_add_f32": (_i, [_vp, _vp, _i, _vp]),
    "qk_silu_mul_f32": (_i, [_vp, _vp, _i, _vp]),
    "qk_argmax_workspace_bytes": (ctypes.c_size_t, [_i]),
    "qk_argmax_f32": (_i, [_vp, _i, _vp, _vp, _vp]),
    "qk_rope_tables_f32": (_i, [_f, _i, ctypes.POINTER(qk_rope_scaling), _vp, _i, _i, _vp, _vp, _vp]),
    "qk_rope_paged_write": (_i, [ctypes.POINTER(qk_paged_kv), ctypes.POINTER(qk_paged_batch), _vp, _i, _vp, _i, _vp,
                                 _i, _vp, _i, _i, _vp, _vp, _i, _i, _i, _vp]),
    "qk_paged_read_f32": (_i, [ctypes.POINTER(qk_paged_kv), ctypes.POINTER(qk_paged_batch), _vp, _i, _vp, _i, _vp]),
    "qk_paged_attention_workspace_bytes": (ctypes.c_size_t, [ctypes.POINTER(qk_paged_batch), _i, _i, _i]),
    "qk_paged_attention_f32": (_i, [ctypes.POINTER(qk_paged_kv), ctypes.POINTER(qk_paged_batch), _vp, _i, _vp, _i, _i,
                                    _f, _vp, ctypes.c_size_t, _vp]),
    "qk_paged_attention_terms_workspace_bytes": (ctypes.c_size_t, [ctypes.POINTER(qk_paged_batch), _i, _i, _i, _i]),
    "qk_paged_attention_terms_f32": (_i, [ctypes.POINTER(qk_paged_kv), ctypes.POINTER(qk_paged_batch), _vp, _i, _vp, _i,
                                          _i, _f, ctypes.POINTER(qk_attention_terms), _vp, ctypes.c_size_t, _vp]),
    "qk_pages_workspace_bytes": (ctypes.c_size_t, [ctypes.POINTER(qk_page_pool)]),
    "qk_pages_resize": (_i, [ctypes.POINTER(qk_page_pool), _vp, _vp, _vp, _vp, ctypes.c_size_t, _vp]),
    "qk_pages_fork": (_i, [ctypes.POINTER(qk_page_pool), _vp, _vp, _vp, _vp, ctypes.c_size_t, _vp]),
    "qk_pages_compact": (_i, [ctypes.POINTER(qk_page_pool), _vp, _vp, ctypes.c_size_t, _vp]),
    "qk_pages_copy": (_i, [ctypes.POINTER(qk_paged_kv), _i, _vp, _vp, _i, _vp]),
    "qk_sample_rows_workspace_bytes": (ctypes.c_size_t, [_i, _i]),
    "qk_sample_rows_f32": (_i, [_vp, _i, ctypes.c_int64, _i, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _vp, ctypes.c_size_t,
                                _vp]),
    "qk_llama_create": (_i, [ctypes.POINTER(qk_llama_config), ctypes.POINTER(qk_llama_weights), _vp,
                             ctypes.POINTER(ctypes.c_void_p)]),
    "qk_llama_destroy": (_i, [_vp]),
    "qk_llama_kv_cache": (_i, [_vp, ctypes.POINTER(ctypes.c_void_p), ctypes.POINTER(ctypes.c_void_p)]),
    "qk_llama_logits": (_i, [_vp, ctypes.POINTER(ctypes.c_void_p)]),
    "qk_llama_residual": (_i, [_vp, ctypes.POINTER(ctypes.c_void_p)]),
    "qk_llama_matrix_calls": (_i, [_vp, ctypes.POINTER(ctypes.c_uint64)]),
    "qk_llama_forward": (_i, [_vp, _i, _i, _i, ctypes.POINTER(ctypes.c_int)]),
    "qk_rope_kv_write_batched": (_i, [_vp, _vp, _vp, _vp, _vp, _vp, _vp, _i, ctypes.c_int64, _vp, _i, _i, _i, _i, _i,
                                      _vp]),
    "qk_ffn_batched_workspace_bytes": (ctypes.c_size_t, [_i, _i, _i]),
    "qk_ffn_batched_f32": (_i, [_i, _vp, _i, _vp, _i, _vp, _vp, _i, _vp, _i, _i, _i, _i, _i, _vp, ctypes.c_size_t,
                                _vp]),
    "qk_attention_batched_f32": (_i, [_vp, _vp, _vp, _vp, _i, ctypes.c_int64, _vp, _i, _i, _i, _i, _i, _vp]),
    "qk_attention_split_workspace_bytes": (ctypes.c_size_t, [_i, _i, _i, _i, _i, _i]),
    "qk_attention_split_f32": (_i, [_vp, _vp, _vp, _vp, _i, ctypes.c_int64, _vp, _i, _i, _i, _i, _i, _i, _vp,
                                    ctypes.c_size_t, _vp]),
    "qk_argmax_rows_workspace_bytes": (ctypes.c_size_t, [_i, _i]),
    "qk_argmax_rows_f32": (_i, [_vp, _i, ctypes.c_int64, _i, _vp, _vp, _vp]),
    "qk_llama_batch_create": (_i, [ctypes.POINTER(qk_llama_config), ctypes.POINTER(qk_llama_weights), _i,
                                   ctypes.c_int64, _vp, ctypes.POINTER(ctypes.c_void_p)]),
    "qk_llama_batch_destroy": (_i, [_vp]),
    "qk_llama_memory_bytes": (_i, [_vp, ctypes.POINTER(qk_llama_memory)]),
    "qk_llama_batch_memory_bytes": (_i, [_vp, ctypes.POINTER(qk_llama_memory)]),
    "qk_llama_batch_kv_cache": (_i, [_vp, ctypes.POINTER(ctypes.c_void_p), ctypes.POINTER(ctypes.c_void_p)]),
    "qk_llama_batch_logits": (_i, [_vp, ctypes.POINTER(ctypes.c_void_p)]),
    "qk_llama_batch_residual": (_i, [_vp, ctypes.POINTER(ctypes.c_void_p)]),
    "qk_llama_batch_matrix_calls": (_i, [_vp, ctypes.POINTER(ctypes.c_uint64)]),
    "qk_llama_batch_set_int8": (_i, [_vp, _i, _i]),
    "qk_llama_set_trace": (_i, [_vp, _vp, _vp]),
    "qk_llama_batch_set_trace": (_i, [_vp, _vp, _vp]),
    "qk_llama_batch_forward": (_i, [_vp, ctypes.POINTER(ctypes.c_int32), ctypes.POINTER(qk_batch_token), _i, _i,
                                    ctypes.POINTER(ctypes.c_int32)]),
    "qk_llama_batch_forward_rows": (_i, [_vp, ctypes.POINTER(ctypes.c_int32), ctypes.POINTER(qk_batch_token), _i,
                                         ctypes.POINTER(ctypes.c_int32), _i, ctypes.POINTER(ctypes.c_int32)]),
    "qk_gguf_open": (_i, [ctypes.c_char_p, ctypes.POINTER(ctypes.c_void_p)]),
    "qk_gguf_close": (_i, [_vp]),
    "qk_gguf_param": (_i, [_vp, ctypes.c_char_p, ctypes.POINTER(ctypes.c_double)]),
    "qk_gguf_string": (ctypes.c_char_p, [_vp, ctypes.c_char_p]),
    "qk_gguf_tensor_count": (ctypes.c_int64, [_vp]),
    "qk_gguf_tensor_at": (_i, [_vp, ctypes.c_int64, ctypes.POINTER(qk_gguf_tensor)]),
    "qk_gguf_find_tensor": (_i, [_vp, ctypes.c_char_p, ctypes.POINTER(qk_gguf_tensor)]),
    "qk_gguf_token_count": (ctypes.c_int64, [_vp, _i]),
    "qk_gguf_token": (_vp, [_vp, _i, ctypes.c_int64, ctypes.POINTER(ctypes.c_int64)]),
    "qk_gguf_data": (_i, [_vp, ctypes.POINTER(ctypes.c_void_p), ctypes.POINTER(ctypes.c_uint64),
                          ctypes.POINTER(ctypes.c_uint64)]),
    "qk_gguf_upload": (_i, [_vp, _vp]),
    "qk_gguf_llama": (_i, [_vp, _i, ctypes.POINTER(qk_llama_config), ctypes.POINTER(qk_llama_weights),
                           ctypes.POINTER(qk_llama_layer), _i]),
}

_LIB = None


def lib() -> ctypes.CDLL:
    """The loaded libqk.so with every signature bound (raises if unbuilt)."""
    global _LIB
    if _LIB is None:
        if not LIB_PATH.exists():
            raise ImportError(f"{LIB_PATH} is not built; run __graft_entry__.build()")
        handle = ctypes.CDLL(str(LIB_PATH))
        for name, (res, args) in SIGNATURES.items():
            fn = getattr(handle, name)
            fn.restype = res
            fn.argtypes = args
        _LIB = handle
    return _LIB


def check(status: int, where: str) -> None:
    """Raise QKError for a non-zero status (the cuda_check convention)."""
    if status != QK_OK:
        detail = lib().qk_last_error().decode() or lib().qk_status_string(status).decode()
        raise QKError(where, status, detail)


def ptr(a) -> int | None:
    """Device address of a tensor-like (data_ptr()), an int, or None."""
    if a is None:
        return None
    if isinstance(a, int):
        return a
    return a.data_ptr()


def stream_handle(stream) -> int | None:
    """hipStream_t of a torch stream / raw handle; None = null stream."""
    if stream is None:
        return None
    if isinstance(stream, int):
        return stream
    return stream.cuda_stream


def tensor_bytes(qtype: int, cols: int, rows: int) -> int:
    """Bytes of a quantized tensor: the size rule of inferencer.cu:252-259."""
    if qtype not in BLOCK_BYTES or cols % 256 or cols <= 0 or rows < 0:
        raise QKError("tensor_bytes", QK_ERR_SHAPE, "Invalid quantized tensor shape")
    row = cols // 256 * BLOCK_BYTES[qtype]
    if qtype == Q6_K_SPLIT:
        row = (row + 15) // 16 * 16   # split rows start 16-byte aligned
    return row * rows


@dataclass
class Tensor:
    """A quantized weight view: Tensor{dims, type, gpu} of inferencer.cu:178-186.

    dims[0] = cols (contiguous), dims[1] = rows; data is a device buffer."""
    dims: Sequence[int]
    type: int
    data: object

    def cols(self) -> int:
        return int(self.dims[0])

    def rows(self) -> int:
        return int(self.dims[1])

    @property
    def gpu(self) -> int:
        return ptr(self.data)


def matvec(t: Tensor, inp, out, expected_cols: int, expected_rows: int, stream=None) -> None:
    """FastGPU::matvec (inferencer.cu:1156-1171), FP32 mode: out = W inp."""
    if t.cols() != expected_cols or t.rows() != expected_rows or t.type not in QUANT_TYPES:
        raise QKError("matvec", QK_ERR_SHAPE, "Unexpected quantized matrix shape")
    check(lib().qk_gemv_f32(t.type, t.gpu, ptr(inp), ptr(out), expected_cols, expected_rows,
                            stream_handle(stream)), "quantized matrix launch")


def matvec_argmax(t: Tensor, inp, out, token_out, workspace, stream=None) -> None:
    """The LM head with its greedy pick (inferencer.cu:1414, 1523-1526): out = W inp and token_out[0] = the
    lowest index among the maxima of out; workspace of qk_gemv_argmax_workspace_bytes() bytes."""
    if t.type not in QUANT_TYPES:
        raise QKError("matvec_argmax", QK_ERR_SHAPE, "Unexpected quantized matrix shape")
    check(lib().qk_gemv_argmax_f32(t.type, t.gpu, ptr(inp), ptr(out), t.cols(), t.rows(), ptr(token_out),
                                   ptr(workspace), stream_handle(stream)), "LM head with greedy pick")


def multi_matvec_i8(pairs, xq, xscale, cols: int, stream=None) -> None:
    """qkv_cuda / gate_up_cuda with dp4a (inferencer.cu:753-804): one fused INT8 launch over (Tensor, out) pairs."""
    for t, _ in pairs:
        if t.cols() != cols:
            raise QKError("multi_matvec_i8", QK_ERR_SHAPE, "Unexpected quantized matrix shape")
    arr = _matrices(pairs)
    check(lib().qk_gemv_multi_i8(arr, len(pairs), ptr(xq), ptr(xscale), cols, stream_handle(stream)),
          "fused INT8 matrix launch")


def _matrices(pairs) -> ctypes.Array:
    arr = (qk_matrix * len(pairs))()
    for i, (t, out) in enumerate(pairs):
        arr[i].type, arr[i].rows, arr[i].w, arr[i].y = t.type, t.rows(), t.gpu, ptr(out)
    return arr


def multi_matvec(pairs, inp, cols: int, stream=None) -> None:
    """One fused launch of out_m = W_m inp over (Tensor, out) pairs sharing inp."""
    for t, _ in pairs:
        if t.cols() != cols:
            raise QKError("multi_matvec", QK_ERR_SHAPE, "Unexpected quantized matrix shape")
    arr = _matrices(pairs)
    check(lib().qk_gemv_multi_f32(arr, len(pairs), ptr(inp), cols, stream_handle(stream)),
          "fused quantized matrix launch")


def qkv(wq: Tensor, wk: Tensor, wv: Tensor, x, q, k, v, dim: int, kv_dim: int, stream=None) -> None:
    """qkv_cuda (inferencer.cu:753-784), FP32 mode: Q4_K q/k, Q4_K or Q6_K v."""
    if (wq.rows(), wk.rows(), wv.rows()) != (dim, kv_dim, kv_dim) or wq.type != Q4_K or wk.type != Q4_K \
            or wv.type not in QUANT_TYPES:
        raise QKError("qkv", QK_ERR_SHAPE, "Unexpected QKV quantization")
    multi_matvec([(wq, q), (wk, k), (wv, v)], x, dim, stream)


def gate_up(wgate: Tensor, wup: Tensor, x, gate, up, dim: int, hidden: int, stream=None) -> None:
    """gate_up_cuda (inferencer.cu:786-804), FP32 mode."""
    if wgate.type != Q4_K or wup.type != Q4_K or wgate.rows() != hidden or wup.rows() != hidden:
        raise QKError("gate_up", QK_ERR_SHAPE, "Unexpected feedforward quantization")
    multi_matvec([(wgate, gate), (wup, up)], x, dim, stream)


def batch_workspace_bytes(cols: int, rows: int, count: int) -> int:
    """Workspace bytes of a multi-token call (rows: total output rows)."""
    return int(lib().qk_gemv_batched_workspace_bytes(cols, rows, count))


def batch_matvec(t: Tensor, inp, out, cols: int, rows: int, count: int, workspace=None,
                 workspace_bytes: int = 0, stream=None) -> None:
    """FastRunner::batch_matvec (inferencer.cu:1265-1278) with FP32 semantics:
    out[t*rows + r] = sum_c W[r][c] inp[t*cols + c] for t < count."""
    if t.cols() != cols or t.rows() != rows or t.type not in QUANT_TYPES:
        raise QKError("batch_matvec", QK_ERR_SHAPE, "Unexpected batched matrix shape")
    check(lib().qk_gemv_batched_f32(t.type, t.gpu, ptr(inp), cols, ptr(out), rows, cols, rows, count,
                                    ptr(workspace), workspace_bytes, stream_handle(stream)),
          "batched matrix launch")


def dequant_rows(t: Tensor, out, row0: int, nrows: int, stream=None) -> None:
    """Rows row0 .. row0+nrows-1 of t as fp32 (q4_value / q6_value, inferencer.cu:454-487)."""
    if row0 < 0 or nrows < 0 or row0 + nrows > t.rows():
        raise QKError("dequant_rows", QK_ERR_INVALID_ARG, "row range outside the tensor")
    check(lib().qk_dequant_rows(t.type, t.gpu, ptr(out), t.cols(), row0, nrows, stream_handle(stream)),
          "dequant launch")


def split_q6k(t: Tensor, stream=None) -> Tensor:
    """A copy of a Q6_K tensor in the split layout (qk_q6k_split): same block
    bytes, every field 16-byte aligned."""
    import torch

    if t.type != Q6_K:
        raise QKError("split_q6k", QK_ERR_TYPE, "split_q6k takes a Q6_K tensor")
    dst = torch.empty(tensor_bytes(Q6_K_SPLIT, t.cols(), t.rows()), dtype=torch.uint8, device="cuda")
    check(lib().qk_q6k_split(t.gpu, ptr(dst), t.cols(), t.rows(), stream_handle(stream)), "Q6_K split")
    return Tensor((t.cols(), t.rows()), Q6_K_SPLIT, dst)


def embedding(t: Tensor, tokens, out, n_tokens: int, stream=None) -> None:
    """embedding_cuda / embedding_batch_cuda (inferencer.cu:806-819)."""
    check(lib().qk_embedding(t.type, t.gpu, ptr(tokens), n_tokens, ptr(out), t.cols(), t.rows(),
                             stream_handle(stream)), "embedding launch")


def quantize(x, xq, xscale, cols: int, n_tokens: int = 1, ldx: int | None = None, ldxq: int | None = None,
             ldscale: int | None = None, stream=None) -> None:
    """FastGPU::quantize / quantize_batch_cuda (inferencer.cu:1151-1155, 891-904)."""
    ldx = cols if ldx is None else ldx
    ldxq = cols if ldxq is None else ldxq
    ldscale = (cols + 31) // 32 if ldscale is None else ldscale
    check(lib().qk_quantize_x32(ptr(x), ldx, ptr(xq), ldxq, ptr(xscale), ldscale, cols, n_tokens,
                                stream_handle(stream)), "activation quantization launch")


def rmsnorm_quantize(x, weight, out, xq, xscale, cols: int, n_tokens: int = 1, eps: float = 1e-5,
                     ldx: int | None = None, ldout: int | None = None, ldxq: int | None = None,
                     ldscale: int | None = None, stream=None) -> None:
    """rmsnorm_quantize_cuda / rmsnorm_quantize_batch_cuda (inferencer.cu:839-889): RMSNorm then the
    per-32 quantization in one launch (out may be None)."""
    ldx = cols if ldx is None else ldx
    ldout = cols if ldout is None else ldout
    ldxq = cols if ldxq is None else ldxq
    ldscale = cols // 32 if ldscale is None else ldscale
    check(lib().qk_rmsnorm_quantize_x32(ptr(x), ldx, ptr(weight), ptr(out), ldout, ptr(xq), ldxq, ptr(xscale),
                                        ldscale, cols, n_tokens, eps, stream_handle(stream)),
          "fused RMSNorm quantization launch")


def matvec_i8(t: Tensor, xq, xscale, out, cols: int, rows: int, n_tokens: int = 1, ldxq: int | None = None,
              ldscale: int | None = None, ldy: int | None = None, stream=None) -> None:
    """gemv_q4_dp4a / gemv_q6_dp4a / gemv_batch_dp4a (inferencer.cu:558-569, 663-699)."""
    if t.cols() != cols or t.rows() != rows or t.type not in QUANT_TYPES:
        raise QKError("matvec_i8", QK_ERR_SHAPE, "Unexpected quantized matrix shape")
    ldxq = cols if ldxq is None else ldxq
    ldscale = cols // 32 if ldscale is None else ldscale
    ldy = rows if ldy is None else ldy
    check(lib().qk_gemv_i8(t.type, t.gpu, ptr(xq), ldxq, ptr(xscale), ldscale, ptr(out), ldy, cols, rows,
                           n_tokens, stream_handle(stream)), "INT8 matrix launch")


# ------------------------------------------ paged cache of a serving step --

_KV_DTYPES = {F16: "torch.float16", I8: "torch.int8", F8_E4M3: "torch.float8_e4m3fn", I4: "torch.uint8"}


def _want(where: str, name: str, t, dtypes, shape=None, last_contiguous: bool = False):
    """Check a torch tensor's device, type and shape: dense (QKError otherwise),
    or with last_contiguous of rows that are.  None in shape takes any size."""
    if not getattr(t, "is_cuda", False):
        raise QKError(where, QK_ERR_INVALID_ARG, f"{name} must be a GPU tensor")
    if str(t.dtype) not in dtypes:
        raise QKError(where, QK_ERR_TYPE, f"{name} must be {' or '.join(dtypes)}, got {t.dtype}")
    if shape is not None and (t.dim() != len(shape) or any(w is not None and w != n for w, n in zip(shape, t.shape))):
        raise QKError(where, QK_ERR_SHAPE, f"{name} has shape {tuple(t.shape)}, expected {tuple(shape)}")
    rows = last_contiguous and t.dim() == 2 and (t.shape[1] < 2 or t.stride(1) == 1) and \
        (t.shape[0] < 2 or t.stride(0) >= t.shape[1])
    if not (rows or t.is_contiguous()):
        raise QKError(where, QK_ERR_INVALID_ARG, f"{name} must be contiguous{' in its rows' if last_contiguous else ''}")


_SCALING_FIELDS = {n for n, _ in qk_rope_scaling._fields_} - {"type"}
_TORCH = None


def _torch():
    global _TORCH
    if _TORCH is None:
        import torch
        _TORCH = torch
    return _TORCH


_INT_MAX = 0x7FFFFFFF


def _int(where: str, name: str, n) -> int:
    """n for an int of the C interface, where a larger one would lose its upper bits
    (QKError)."""
    n = int(n)
    if not -_INT_MAX <= n <= _INT_MAX:
        raise QKError(where, QK_ERR_LIMIT, f"{name} of {n} is beyond 2^31 - 1")
    return n


def _gpu(where: str, name: str, t):
    """The GPU a tensor is on (QKError if it is on none)."""
    if not t.is_cuda:
        raise QKError(where, QK_ERR_INVALID_ARG, f"{name} must be a GPU tensor")
    return t.device


def _rows(where: str, name: str, t, n: int, w: int, device, most: int = _INT_MAX) -> int:
    """The leading dimension of a float32 matrix [n][w] of contiguous rows on
    the device (QKError for anything else), `most` at most; of a single row w
    where its own would be refused."""
    if t is not None and t.dtype is _TORCH.float32 and t.device == device and t.shape == (n, w):
        ld, one = t.stride()
        if (one == 1 or w == 1) and (ld >= w or n == 1):
            if n == 1:
                return ld if w <= ld <= most and ld % 4 == 0 else w
            if ld > most:
                raise QKError(where, QK_ERR_LIMIT, f"rows of {name} are {ld} apart, more than 2^31 - 1")
            return ld
    _want(where, name, t, ("torch.float32",), (n, w), last_contiguous=True)
    raise QKError(where, QK_ERR_INVALID_ARG, f"{name} is on {t.device}, the call's other tensors on {device}")


def _dense(where: str, name: str, t, dtype, shape, device) -> int:
    """The address of a contiguous tensor of the type and shape on the device
    (QKError for anything else)."""
    if t is not None and t.dtype is dtype and t.device == device and t.shape == shape and t.is_contiguous():
        return t.data_ptr()
    _want(where, name, t, (str(dtype),), shape)
    raise QKError(where, QK_ERR_INVALID_ARG, f"{name} is on {t.device}, the call's other tensors on {device}")


def _space(where: str, t, device) -> tuple[int | None, int]:
    """Address and bytes of a workspace tensor (None: none) on the device."""
    if t is None:
        return None, 0
    if t.device != device or not t.is_contiguous():
        raise QKError(where, QK_ERR_INVALID_ARG, f"workspace must be a contiguous tensor on {device}")
    return t.data_ptr(), t.numel() * t.element_size()


def _launch(device, stream, fn, *args) -> int:
    """fn(*args, stream) with the tensors' device current: on the given stream,
    or on the device's current torch stream."""
    cuda = _TORCH.cuda
    index = device.index
    if stream is None:
        stream = _TORCH._C._cuda_getCurrentRawStream(index)
    elif not isinstance(stream, int):
        if getattr(stream, "device", device) != device:
            raise QKError(fn.__name__, QK_ERR_INVALID_ARG, f"stream of {stream.device}, tensors on {device}")
        stream = stream.cuda_stream
    if cuda.current_device() == index:
        return fn(*args, stream)
    with cuda.device(index):
        return fn(*args, stream)


class PagedKV:
    """One layer's paged cache (qk_paged_kv): key and value are tensors [pages]
    [kv_heads][page_rows][head_dim] of the type's dtype (F16 float16, I8 int8,
    F8_E4M3 float8_e4m3fn), the scales [pages][kv_heads][page_rows] float32 (I8,
    F8_E4M3).  I4: key and value uint8 [...][head_dim / 2], two codes a byte, the
    scales uint8 [pages][kv_heads][page_rows][8], a row's fp32 scale and its four
    multipliers."""

    def __init__(self, type: int, key, value, key_scale=None, value_scale=None):
        where = "PagedKV"
        _torch()
        if type not in _KV_DTYPES:
            raise QKError(where, QK_ERR_TYPE, f"cache type {type} is not F16, I8, I4 or F8_E4M3")
        _want(where, "key", key, (_KV_DTYPES[type],), (None,) * 4)
        _want(where, "value", value, (_KV_DTYPES[type],), tuple(key.shape))
        if (type == F16) != (key_scale is None) or (type == F16) != (value_scale is None):
            raise QKError(where, QK_ERR_INVALID_ARG, "scales belong to I8, I4 and F8_E4M3 caches, and only to them")
        scales, shape = ("torch.uint8", (8,)) if type == I4 else ("torch.float32", ())
        for name, t in (("key_scale", key_scale), ("value_scale", value_scale)):
            if t is not None:
                _want(where, name, t, (scales,), tuple(key.shape[:3]) + shape)
        for t in (value, key_scale, value_scale):
            if t is not None and t.device != key.device:
                raise QKError(where, QK_ERR_INVALID_ARG, f"tensors on {key.device} and {t.device}")
        self.type, self.key, self.value, self.key_scale, self.value_scale = type, key, value, key_scale, value_scale
        self.pages, self.kv_heads, self.page_rows, self.head_dim = (int(n) for n in key.shape)
        self.head_dim *= 2 if type == I4 else 1
        self.desc = qk_paged_kv(type, self.kv_heads, self.head_dim, self.page_rows, self.pages, ptr(key), ptr(value),
                                ptr(key_scale), ptr(value_scale))
        self.ref, self.device, self.width = ctypes.byref(self.desc), key.device, self.kv_heads * self.head_dim

    @classmethod
    def empty(cls, type: int, pages: int, kv_heads: int, page_rows: int, head_dim: int, device="cuda") -> "PagedKV":
        """A cache whose rows are not written yet."""
        torch = _torch()
        if type not in _KV_DTYPES:
            raise QKError("PagedKV", QK_ERR_TYPE, f"cache type {type} is not F16, I8, I4 or F8_E4M3")
        if type == I4 and head_dim % 2:
            raise QKError("PagedKV", QK_ERR_LIMIT, "head_dim must be 64, 96, 128 or 256")
        dtype = getattr(torch, _KV_DTYPES[type].split(".")[1])
        width = head_dim // 2 if type == I4 else head_dim
        new = lambda: torch.empty(pages, kv_heads, page_rows, width, dtype=dtype, device=device)
        entry = dict(dtype=torch.uint8) if type == I4 else dict(dtype=torch.float32)
        shape = (pages, kv_heads, page_rows) + ((8,) if type == I4 else ())
        scale = lambda: None if type == F16 else torch.empty(*shape, device=device, **entry)
        return cls(type, new(), new(), scale(), scale())


class PagedBatch:
    """The sequences of a call over a paged cache (qk_paged_batch): page_table
    [table_rows][table_stride] int32, seqs [n_seqs][4] int32 of (first, count,
    pos, table), both on the GPU; n_tokens token rows; max_count and max_rows
    bound count and pos + count."""

    def __init__(self, page_table, seqs, n_tokens: int, max_count: int, max_rows: int):
        where = "PagedBatch"
        _want(where, "page_table", page_table, ("torch.int32",), (None, None))
        _want(where, "seqs", seqs, ("torch.int32",), (None, 4))
        if page_table.device != seqs.device:
            raise QKError(where, QK_ERR_INVALID_ARG, f"tensors on {page_table.device} and {seqs.device}")
        self.page_table, self.seqs, self.n_tokens = page_table, seqs, _int(where, "n_tokens", n_tokens)
        self.max_count, self.max_rows = _int(where, "max_count", max_count), _int(where, "max_rows", max_rows)
        rows, stride = (_int(where, "page_table", n) for n in page_table.shape)
        self.desc = qk_paged_batch(ptr(page_table), rows, stride, ptr(seqs), _int(where, "seqs", seqs.shape[0]),
                                   self.n_tokens, self.max_count, self.max_rows)
        self.ref, self.device = ctypes.byref(self.desc), seqs.device


def _one_device(where: str, kv: PagedKV, batch: PagedBatch):
    if kv.device != batch.device:
        raise QKError(where, QK_ERR_INVALID_ARG, f"cache on {kv.device}, batch on {batch.device}")
    return kv.device


def rope_tables(theta: float, rot_dim: int, cosine, sine, first_pos: int = 0, scaling: dict | None = None,
                freq_factors=None, stream=None) -> None:
    """qk_rope_tables_f32: cosine and sine, [positions][rot_dim / 2] float32, of
    positions first_pos, first_pos + 1, ...  scaling: {"type": "none", "linear",
    "llama3" or "yarn", "factor": ..., ...} with the fields of qk_rope_scaling;
    freq_factors: rot_dim / 2 values that divide the frequencies.  Like every
    call of this section it runs on the tensors' device, on the given stream or
    else on that device's current torch stream."""
    where = "rope_tables"
    f32 = _torch().float32
    positions = cosine.shape[0] if cosine.dim() == 2 else -1
    if not 0 <= first_pos <= _INT_MAX - positions:
        raise QKError(where, QK_ERR_LIMIT, f"{positions} positions from {first_pos} on: beyond 0 to 2^31 - 1")
    device = _gpu(where, "cosine", cosine)
    c_ptr = _dense(where, "cosine", cosine, f32, (positions, rot_dim // 2), device)
    s_ptr = _dense(where, "sine", sine, f32, (positions, rot_dim // 2), device)
    f_ptr = None if freq_factors is None else _dense(where, "freq_factors", freq_factors, f32, (rot_dim // 2,), device)
    c = None
    if scaling is not None:
        fields = dict(scaling)
        kind = fields.pop("type", "none")
        if kind not in ROPE_SCALING or not fields.keys() <= _SCALING_FIELDS:
            raise QKError(where, QK_ERR_INVALID_ARG, f"unknown scaling {scaling}")
        c = ctypes.byref(qk_rope_scaling(ROPE_SCALING[kind], **fields))
    check(_launch(device, stream, lib().qk_rope_tables_f32, theta, rot_dim, c, f_ptr, first_pos, positions, c_ptr,
                  s_ptr), "rotary table launch")


def rope_paged_write(kv: PagedKV, batch: PagedBatch, q, q_out, k, v, cosine, sine, heads: int,
                     rot_dim: int | None = None, half: bool = False, stream=None) -> None:
    """qk_rope_paged_write: q [n_tokens][heads * head_dim] rotated into q_out
    (both may be None, or the same), k and v [n_tokens][kv_heads * head_dim]
    into the pages, k rotated.  rot_dim: head_dim when None; 0 needs no tables."""
    where = "rope_paged_write"
    device, n, w, hd = _one_device(where, kv, batch), batch.n_tokens, kv.width, kv.head_dim
    rot_dim = hd if rot_dim is None else rot_dim
    q_ptr = qo_ptr = c_ptr = s_ptr = None
    ldq = ldq_out = positions = 0
    if q is not None or q_out is not None:
        ldq = _rows(where, "q", q, n, heads * hd, device)
        ldq_out = _rows(where, "q_out", q_out, n, heads * hd, device)
        q_ptr, qo_ptr = q.data_ptr(), q_out.data_ptr()
    ldk, ldv = _rows(where, "k", k, n, w, device), _rows(where, "v", v, n, w, device)
    if rot_dim:
        f32 = _TORCH.float32
        positions = _int(where, "positions", cosine.shape[0]) if cosine is not None and cosine.dim() == 2 else -1
        c_ptr = _dense(where, "cosine", cosine, f32, (positions, rot_dim // 2), device)
        s_ptr = _dense(where, "sine", sine, f32, (positions, rot_dim // 2), device)
    check(_launch(device, stream, lib().qk_rope_paged_write, kv.ref, batch.ref, q_ptr, ldq, qo_ptr, ldq_out,
                  k.data_ptr(), ldk, v.data_ptr(), ldv, heads, c_ptr, s_ptr, positions, rot_dim, int(half)),
          "paged cache write launch")


def paged_read(kv: PagedKV, batch: PagedBatch, key_out, value_out, stream=None) -> None:
    """qk_paged_read_f32: the rows of the batch's tokens as fp32, [n_tokens]
    [kv_heads * head_dim] each (either may be None)."""
    where = "paged_read"
    device, n, w = _one_device(where, kv, batch), batch.n_tokens, kv.width
    ldk = ldv = 0
    if key_out is not None:
        ldk = _rows(where, "key_out", key_out, n, w, device)
    if value_out is not None:
        ldv = _rows(where, "value_out", value_out, n, w, device)
    check(_launch(device, stream, lib().qk_paged_read_f32, kv.ref, batch.ref, ptr(key_out), ldk, ptr(value_out), ldv),
          "paged cache read launch")


def paged_attention_workspace_bytes(batch: PagedBatch, heads: int, kv_heads: int, head_dim: int,
                                    window: int = 0) -> int:
    """Workspace bytes of paged_attention."""
    where = "paged_attention_workspace_bytes"
    return int(lib().qk_paged_attention_terms_workspace_bytes(batch.ref, _int(where, "heads", heads),
                                                              _int(where, "kv_heads", kv_heads),
                                                              _int(where, "head_dim", head_dim),
                                                              _int(where, "window", window)))


def paged_attention(kv: PagedKV, batch: PagedBatch, q, out, heads: int, scale: float = 0.0, workspace=None,
                    stream=None, cap: float = 0.0, window: int = 0, slopes=None, prefix=None) -> None:
    """qk_paged_attention_f32: attention of every new token (rows of q, [n_tokens]
    [heads * head_dim], into out) over its sequence's rows up to its own.  With terms
    (qk_attention_terms): scores capped by cap * tanh(score / cap), less slopes[head]
    (float32 [heads]) times the distance; rows of the last `window` positions alone;
    and those below prefix[sequence] (int32 [n_seqs]) seen from before them too."""
    where = "paged_attention"
    device, heads = _one_device(where, kv, batch), _int(where, "heads", heads)
    n, w = batch.n_tokens, heads * kv.head_dim
    ldq, ldout = _rows(where, "q", q, n, w, device), _rows(where, "out", out, n, w, device)
    ws, nbytes = _space(where, workspace, device)
    if not cap and not window and slopes is None and prefix is None:
        check(_launch(device, stream, lib().qk_paged_attention_f32, kv.ref, batch.ref, q.data_ptr(), ldq,
                      out.data_ptr(), ldout, heads, scale, ws, nbytes), "paged attention launch")
        return
    slopes_ptr = None if slopes is None else _dense(where, "slopes", slopes, _TORCH.float32, (heads,), device)
    prefix_ptr = None if prefix is None else _dense(where, "prefix", prefix, _TORCH.int32, (batch.seqs.shape[0],), device)
    terms = qk_attention_terms(cap, _int(where, "window", window), slopes_ptr, prefix_ptr)
    check(_launch(device, stream, lib().qk_paged_attention_terms_f32, kv.ref, batch.ref, q.data_ptr(), ldq,
                  out.data_ptr(), ldout, heads, scale, ctypes.byref(terms), ws, nbytes), "paged attention launch")


class PagePool:
    """A pool of pages (qk_page_pool): page_table int32 [table_rows][table_stride]
    (the one of PagedBatch), refs int32 [pages], of each page the entries that name
    it, and the PagedKV of every layer whose contents follow."""

    def __init__(self, page_table, refs, page_rows: int, layers: Sequence[PagedKV] = ()):
        where = "PagePool"
        _torch()
        _want(where, "page_table", page_table, ("torch.int32",), (None, None))
        _want(where, "refs", refs, ("torch.int32",), (None,))
        for t in (refs, *layers):
            if t.device != page_table.device:
                raise QKError(where, QK_ERR_INVALID_ARG, f"tensors on {page_table.device} and {t.device}")
        self.page_table, self.refs, self.page_rows, self.layers = page_table, refs, _int(where, "page_rows", page_rows), tuple(layers)
        rows, stride = (_int(where, "page_table", n) for n in page_table.shape)
        self._layers = (qk_paged_kv * max(len(self.layers), 1))(*(kv.desc for kv in self.layers))
        self.desc = qk_page_pool(ptr(page_table), rows, stride, ptr(refs), int(refs.shape[0]), self.page_rows,
                                 self._layers, len(self.layers))
        self.ref, self.device, self.rows = ctypes.byref(self.desc), page_table.device, rows

    @classmethod
    def empty(cls, table_rows: int, table_stride: int, pages: int, page_rows: int, layers: Sequence[PagedKV] = (),
              device="cuda") -> "PagePool":
        """A pool of which no page is held."""
        torch = _torch()
        table = torch.full((table_rows, table_stride), -1, dtype=torch.int32, device=device)
        return cls(table, torch.zeros(pages, dtype=torch.int32, device=device), page_rows, layers)


def pages_workspace_bytes(pool: PagePool) -> int:
    """Workspace bytes of pages_resize, pages_fork and pages_compact."""
    n = int(lib().qk_pages_workspace_bytes(pool.ref))
    if n == 0:
        raise QKError("pages_workspace_bytes", QK_ERR_INVALID_ARG, lib().qk_last_error().decode())
    return n


def _row_numbers(where: str, name: str, t, pool: PagePool) -> int:
    return _dense(where, name, t, _TORCH.int32, (pool.rows,), pool.device)


def _one_number(where: str, name: str, t, pool: PagePool):
    return None if t is None else _dense(where, name, t, _TORCH.int32, (1,), pool.device)


def pages_resize(pool: PagePool, lengths, begins=None, missing=None, workspace=None, stream=None) -> None:
    """qk_pages_resize: table row r comes to hold the pages of rows begins[r] ..
    lengths[r] - 1 (int32 [table_rows]; a negative length leaves the row as it is);
    missing (int32 [1]) receives the entries that got none."""
    where = "pages_resize"
    first = None if begins is None else _row_numbers(where, "begins", begins, pool)
    ws, nbytes = _space(where, workspace, pool.device)
    check(_launch(pool.device, stream, lib().qk_pages_resize, pool.ref, first, _row_numbers(where, "lengths", lengths, pool),
                  _one_number(where, "missing", missing, pool), ws, nbytes), "pages resize launch")


def pages_fork(pool: PagePool, parents, lengths, missing=None, workspace=None, stream=None) -> None:
    """qk_pages_fork: table row c becomes a fork of the first lengths[c] rows of table
    row parents[c] (int32 [table_rows]; a negative parent, or c, leaves the row as it
    is): full pages are shared, the last part of one is copied."""
    where = "pages_fork"
    ws, nbytes = _space(where, workspace, pool.device)
    check(_launch(pool.device, stream, lib().qk_pages_fork, pool.ref, _row_numbers(where, "parents", parents, pool),
                  _row_numbers(where, "lengths", lengths, pool), _one_number(where, "missing", missing, pool), ws, nbytes),
          "pages fork launch")


def pages_compact(pool: PagePool, moved=None, workspace=None, stream=None) -> None:
    """qk_pages_compact: the pages that are held move to the pool's front; moved
    (int32 [1]) receives how many did."""
    where = "pages_compact"
    ws, nbytes = _space(where, workspace, pool.device)
    check(_launch(pool.device, stream, lib().qk_pages_compact, pool.ref, _one_number(where, "moved", moved, pool), ws,
                  nbytes), "pages compact launch")


def pages_copy(layers: Sequence[PagedKV], source, target, stream=None) -> None:
    """qk_pages_copy: the contents of pages source into pages target (int32 [n]) in
    every layer."""
    where = "pages_copy"
    _torch()
    if not layers:
        return
    device = layers[0].device
    for kv in layers:
        if kv.device != device:
            raise QKError(where, QK_ERR_INVALID_ARG, f"caches on {device} and {kv.device}")
    _want(where, "source", source, ("torch.int32",), (None,))
    n = _int(where, "source", source.shape[0])
    array = (qk_paged_kv * len(layers))(*(kv.desc for kv in layers))
    check(_launch(device, stream, lib().qk_pages_copy, array, len(layers), _dense(where, "source", source, _TORCH.int32, (n,), device),
                  _dense(where, "target", target, _TORCH.int32, (n,), device), n), "pages copy launch")


def sample_workspace_bytes(n: int, rows: int) -> int:
    """Workspace bytes of sample_rows for rows of n logits."""
    where = "sample_workspace_bytes"
    return int(lib().qk_sample_rows_workspace_bytes(_int(where, "n", n), _int(where, "rows", rows)))


def sample_rows(logits, uniform, out, temperature=None, top_k=None, top_p=None, min_p=None, prob=None, workspace=None,
                stream=None) -> None:
    """qk_sample_rows_f32: the next token of each row of logits [rows][n], out
    int32 [rows], by uniform float32 [rows] in [0, 1).  temperature, top_p, min_p
    (float32) and top_k (int32) hold a value a row, or are None: 1, and no
    filter.  prob (float32 [rows] or None) receives the token's probability."""
    where = "sample_rows"
    torch = _torch()
    if logits.dim() != 2:
        raise QKError(where, QK_ERR_SHAPE, f"logits has shape {tuple(logits.shape)}, expected rows of logits")
    rows, n = logits.shape
    device = _gpu(where, "logits", logits)
    ldv = _rows(where, "logits", logits, _int(where, "rows", rows), _int(where, "logits a row", n), device, most=1 << 62)
    f32, i32, shape = torch.float32, torch.int32, (rows,)
    of = lambda name, t, dt: None if t is None else _dense(where, name, t, dt, shape, device)
    u_ptr, o_ptr = _dense(where, "uniform", uniform, f32, shape, device), _dense(where, "out", out, i32, shape, device)
    ws, nbytes = _space(where, workspace, device)
    check(_launch(device, stream, lib().qk_sample_rows_f32, logits.data_ptr(), n, ldv, rows,
                  of("temperature", temperature, f32), of("top_k", top_k, i32), of("top_p", top_p, f32),
                  of("min_p", min_p, f32), u_ptr, o_ptr, of("prob", prob, f32), ws, nbytes), "sampling launch")


def _upload_weights(owner, cfg: dict, weights: dict):
    """Device copies of workloads.llama_weights-style host arrays, kept alive
    by owner._dev; returns (qk_llama_config, qk_llama_weights)."""
    import numpy as np
    import torch
    owner._dev = []

    def up(a):
        t = torch.from_numpy(np.ascontiguousarray(a)).to("cuda")
        owner._dev.append(t)
        return t.data_ptr()

    layers = (qk_llama_layer * cfg["layers"])()
    for i, L in enumerate(weights["layers"]):
        for name in ("q", "k", "v", "o", "gate", "up", "down"):
            setattr(layers[i], name + "_type", L[name + "_type"])
            setattr(layers[i], name, up(L[name]))
        layers[i].attn_norm = up(L["attn_norm"])
        layers[i].ffn_norm = up(L["ffn_norm"])
    owner._layers = layers
    out = weights.get("output")
    w = qk_llama_weights(embd_type=weights["embd_type"], token_embd=up(weights["token_embd"]),
                         output_type=weights.get("output_type", 0), output=up(out) if out is not None else None,
                         output_norm=up(weights["output_norm"]), layers=layers)
    c = qk_llama_config(**{k: cfg[k] for k in ("dim", "layers", "heads", "kv_heads", "hidden", "vocab",
                                                "context")}, eps=cfg["eps"], rope_theta=cfg["rope_theta"])
    return c, w


class GGUF:
    """A GGUF v3 model file (the reference's GGUF struct, inferencer.cu:204-340)
    through qk_gguf_*: parameters, string values, tokenizer arrays, the
    tensor table, and the device copy made by upload()."""

    def __init__(self, path):
        h = ctypes.c_void_p()
        check(lib().qk_gguf_open(str(path).encode(), ctypes.byref(h)), "GGUF")
        self.handle = h
        self.path = str(path)

    def close(self):
        # At interpreter exit the module's globals may already be gone.
        if getattr(self, "handle", None) and _LIB is not None:
            _LIB.qk_gguf_close(self.handle)
        self.handle = None

    __del__ = close

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.close()

    def param(self, key: str) -> float:
        v = ctypes.c_double()
        check(lib().qk_gguf_param(self.handle, key.encode(), ctypes.byref(v)), "GGUF parameter")
        return v.value

    def string(self, key: str):
        v = lib().qk_gguf_string(self.handle, key.encode())
        return None if v is None else v.decode("utf-8", "surrogateescape")

    def tensors(self) -> list:
        out = []
        for i in range(lib().qk_gguf_tensor_count(self.handle)):
            t = qk_gguf_tensor()
            check(lib().qk_gguf_tensor_at(self.handle, i, ctypes.byref(t)), "GGUF tensor")
            out.append(t)
        return out

    def tensor(self, name: str) -> qk_gguf_tensor:
        t = qk_gguf_tensor()
        check(lib().qk_gguf_find_tensor(self.handle, name.encode(), ctypes.byref(t)), "GGUF tensor")
        return t

    def host_bytes(self, name: str):
        """A copy of a tensor's bytes from the mapping (numpy uint8)."""
        import numpy as np
        t = self.tensor(name)
        return np.frombuffer(ctypes.string_at(t.host, t.bytes), dtype=np.uint8).copy()

    def tokens(self, which: int = 0) -> list:
        """tokenizer.ggml.tokens (0) or tokenizer.ggml.merges (1) as bytes."""
        out = []
        n = ctypes.c_int64()
        for i in range(lib().qk_gguf_token_count(self.handle, which)):
            p = lib().qk_gguf_token(self.handle, which, i, ctypes.byref(n))
            out.append(ctypes.string_at(p, n.value) if n.value else b"")
        return out

    def data(self):
        p, n, a = ctypes.c_void_p(), ctypes.c_uint64(), ctypes.c_uint64()
        check(lib().qk_gguf_data(self.handle, ctypes.byref(p), ctypes.byref(n), ctypes.byref(a)), "GGUF data")
        return p.value, n.value, a.value

    def upload(self, stream=None) -> None:
        check(lib().qk_gguf_upload(self.handle, stream_handle(stream)), "GGUF upload")

    def llama(self, context: int):
        """(qk_llama_config, qk_llama_weights, layer array) of the uploaded model."""
        c, w = qk_llama_config(), qk_llama_weights()
        n = int(self.param("llama.block_count"))
        layers = (qk_llama_layer * max(n, 1))()
        check(lib().qk_gguf_llama(self.handle, context, ctypes.byref(c), ctypes.byref(w), layers, n), "GGUF llama")
        return c, w, layers


def _config_dict(c: qk_llama_config) -> dict:
    return {k: getattr(c, k) for k in ("dim", "layers", "heads", "kv_heads", "hidden", "vocab", "context", "eps",
                                       "rope_theta")}


class Runner:
    """FastRunner (inferencer.cu:1182-1532) over the C ABI's decode driver.

    weights is a dict of host numpy arrays (workloads.llama_weights layout);
    they are copied to device memory owned by this object.  from_gguf builds
    it from an uploaded GGUF file instead."""

    def __init__(self, cfg: dict, weights: dict, stream=None):
        self.cfg = cfg
        c, w = _upload_weights(self, cfg, weights)
        self._create(c, w, stream)

    def _create(self, c, w, stream):
        h = ctypes.c_void_p()
        check(lib().qk_llama_create(ctypes.byref(c), ctypes.byref(w), stream_handle(stream), ctypes.byref(h)),
              "FastRunner")
        self.handle = h

    @classmethod
    def from_gguf(cls, model: GGUF, context: int, stream=None) -> "Runner":
        self = cls.__new__(cls)
        c, w, self._layers = model.llama(context)
        self._model = model
        self.cfg = _config_dict(c)
        self._create(c, w, stream)
        return self

    def close(self):
        # At interpreter exit the module's globals may already be gone.
        if getattr(self, "handle", None) and _LIB is not None:
            _LIB.qk_llama_destroy(self.handle)
        self.handle = None

    __del__ = close

    def memory(self) -> dict:
        """Device bytes the handle holds (qk_llama_memory_bytes)."""
        m = qk_llama_memory()
        check(lib().qk_llama_memory_bytes(self.handle, ctypes.byref(m)), "memory")
        return {k: int(getattr(m, k)) for k, _ in m._fields_}

    def set_int8(self, q4k: bool = True, q6k: bool = True) -> None:
        """The reference's INT8 GEMV modes (use_dp4a, use_q6_dp4a; inferencer.cu:1159-1166)."""
        check(lib().qk_llama_set_int8(self.handle, int(q4k), int(q6k)), "set_int8")

    def kv_cache(self) -> tuple[int, int]:
        k, v = ctypes.c_void_p(), ctypes.c_void_p()
        check(lib().qk_llama_kv_cache(self.handle, ctypes.byref(k), ctypes.byref(v)), "kv_cache")
        return k.value, v.value

    def logits_ptr(self) -> int:
        p = ctypes.c_void_p()
        check(lib().qk_llama_logits(self.handle, ctypes.byref(p)), "logits")
        return p.value

    def residual(self):
        """The residual stream x after the last step (host copy, float32 [dim])."""
        import numpy as np
        p = ctypes.c_void_p()
        check(lib().qk_llama_residual(self.handle, ctypes.byref(p)), "residual")
        return copy_to_host(p.value, self.cfg["dim"], np.float32)

    def set_trace(self, residuals: "DeviceBuffer | None", quantized: "DeviceBuffer | None" = None) -> None:
        """Per-layer residuals [layer][dim] and INT8 inputs [layer][4][max(dim,
        hidden)] of every following step (qk_llama_set_trace); None stops."""
        self._trace = (residuals, quantized)
        check(lib().qk_llama_set_trace(self.handle, residuals.ptr if residuals else None,
                                       quantized.ptr if quantized else None), "set_trace")

    def matrix_calls(self) -> int:
        """Quantized matrix products issued since create (qk_llama_matrix_calls)."""
        n = ctypes.c_uint64()
        check(lib().qk_llama_matrix_calls(self.handle, ctypes.byref(n)), "matrix_calls")
        return n.value

    def forward(self, token: int, pos: int, need_logits: bool = True) -> int:
        nxt = ctypes.c_int(-1)
        check(lib().qk_llama_forward(self.handle, token, pos, int(need_logits), ctypes.byref(nxt)), "forward")
        return nxt.value


class BatchRunner:
    """Ragged decode batches over the C ABI's batched driver
    (qk_llama_batch_*): every token of a step belongs to its own sequence,
    whose KV rows start at desc.kv_row in caches of cache_rows rows per
    layer."""

    def __init__(self, cfg: dict, weights: dict, max_tokens: int, cache_rows: int, stream=None):
        self.cfg = cfg
        self.cache_rows = cache_rows
        c, w = _upload_weights(self, cfg, weights)
        self._create(c, w, max_tokens, cache_rows, stream)

    def _create(self, c, w, max_tokens, cache_rows, stream):
        self.max_tokens = max_tokens
        h = ctypes.c_void_p()
        check(lib().qk_llama_batch_create(ctypes.byref(c), ctypes.byref(w), max_tokens, cache_rows,
                                          stream_handle(stream), ctypes.byref(h)), "batched runner")
        self.handle = h

    @classmethod
    def from_gguf(cls, model: GGUF, context: int, max_tokens: int, cache_rows: int, stream=None) -> "BatchRunner":
        """context bounds every token's position (the RoPE table length)."""
        self = cls.__new__(cls)
        c, w, self._layers = model.llama(context)
        self._model = model
        self.cfg = _config_dict(c)
        self.cache_rows = cache_rows
        self._create(c, w, max_tokens, cache_rows, stream)
        return self

    def close(self):
        # At interpreter exit the module's globals may already be gone.
        if getattr(self, "handle", None) and _LIB is not None:
            _LIB.qk_llama_batch_destroy(self.handle)
        self.handle = None

    __del__ = close

    def kv_cache(self) -> tuple[int, int]:
        k, v = ctypes.c_void_p(), ctypes.c_void_p()
        check(lib().qk_llama_batch_kv_cache(self.handle, ctypes.byref(k), ctypes.byref(v)), "kv_cache")
        return k.value, v.value

    def memory(self) -> dict:
        """Device bytes the handle holds (qk_llama_batch_memory_bytes)."""
        m = qk_llama_memory()
        check(lib().qk_llama_batch_memory_bytes(self.handle, ctypes.byref(m)), "memory")
        return {k: int(getattr(m, k)) for k, _ in m._fields_}

    def forward(self, tokens, pos, kv_row, need_logits: bool = True, seq=None, logit_rows=None):
        """tokens, pos, kv_row: per-token sequences (several tokens of one
        sequence share its kv_row: a prefill chunk).  Returns the greedy next
        tokens (list) or None.  logit_rows: the token indices whose logits
        and successors are computed (qk_llama_batch_forward_rows); by default
        every token when need_logits, none otherwise."""
        n = len(tokens)
        tok = (ctypes.c_int32 * n)(*[int(t) for t in tokens])
        desc = (qk_batch_token * n)()
        for i in range(n):
            desc[i].pos, desc[i].kv_row = int(pos[i]), int(kv_row[i])
            desc[i].seq = int(seq[i]) if seq is not None else i
        if logit_rows is None:
            nxt = (ctypes.c_int32 * n)()
            check(lib().qk_llama_batch_forward(self.handle, tok, desc, n, int(need_logits), nxt), "batched forward")
            return list(nxt) if need_logits else None
        r = len(logit_rows)
        rows = (ctypes.c_int32 * max(r, 1))(*[int(i) for i in logit_rows])
        nxt = (ctypes.c_int32 * max(r, 1))()
        check(lib().qk_llama_batch_forward_rows(self.handle, tok, desc, n, rows, r, nxt), "batched forward")
        return list(nxt)[:r]

    def logits(self, n_tokens: int):
        import numpy as np
        p = ctypes.c_void_p()
        check(lib().qk_llama_batch_logits(self.handle, ctypes.byref(p)), "logits")
        return copy_to_host(p.value, n_tokens * self.cfg["vocab"], np.float32).reshape(n_tokens, self.cfg["vocab"])

    def residual(self, n_tokens: int):
        """The residual streams after the last step (host copy, [n_tokens][dim])."""
        import numpy as np
        p = ctypes.c_void_p()
        check(lib().qk_llama_batch_residual(self.handle, ctypes.byref(p)), "residual")
        return copy_to_host(p.value, n_tokens * self.cfg["dim"], np.float32).reshape(n_tokens, self.cfg["dim"])

    def set_trace(self, residuals: "DeviceBuffer | None", quantized: "DeviceBuffer | None" = None) -> None:
        """Per token of each following step, residuals [token][layer][dim] and
        INT8 inputs [token][layer][4][max(dim, hidden)]
        (qk_llama_batch_set_trace); None stops."""
        self._trace = (residuals, quantized)
        check(lib().qk_llama_batch_set_trace(self.handle, residuals.ptr if residuals else None,
                                             quantized.ptr if quantized else None), "set_trace")

    def set_int8(self, q4k: bool = True, q6k: bool = True) -> None:
        """The reference's INT8 batched arithmetic (both types or neither;
        qk_llama_batch_set_int8)."""
        check(lib().qk_llama_batch_set_int8(self.handle, int(q4k), int(q6k)), "set_int8")

    def matrix_calls(self) -> int:
        """Quantized matrix products issued since create (qk_llama_batch_matrix_calls)."""
        n = ctypes.c_uint64()
        check(lib().qk_llama_batch_matrix_calls(self.handle, ctypes.byref(n)), "matrix_calls")
        return n.value

    def load_kv(self, key_cache, value_cache) -> None:
        """Copy fp32 caches laid out [layer][cache_rows][kv_dim] (the
        reference's layout) into the driver's head-major caches."""
        _load_kv(self.kv_cache(), self.cfg, self.cache_rows, key_cache, value_cache)

    def kv_rows(self, n: int):
        """Rows 0..n-1 of every layer of both caches, as host arrays
        [layer][n][kv_dim] (the reference's layout)."""
        return _kv_rows(self.kv_cache(), self.cfg, self.cache_rows, n)

    def load_kv_rows(self, row0: int, key_rows, value_rows) -> None:
        """Write host rows [layer][n][kv_dim] (one sequence's rows) at cache
        rows row0 .. row0 + n - 1 of every layer."""
        _load_kv_rows(self.kv_cache(), self.cfg, self.cache_rows, row0, key_rows, value_rows)


_HIP = None


def _hip() -> ctypes.CDLL:
    """libamdhip64 for plain device<->host copies of buffers the C ABI owns."""
    global _HIP
    if _HIP is None:
        h = ctypes.CDLL("libamdhip64.so")
        h.hipMemcpy.argtypes = [_vp, _vp, ctypes.c_size_t, _i]
        h.hipMemcpy.restype = _i
        h.hipMemcpy2D.argtypes = [_vp, ctypes.c_size_t, _vp, ctypes.c_size_t, ctypes.c_size_t, ctypes.c_size_t, _i]
        h.hipMemcpy2D.restype = _i
        h.hipDeviceSynchronize.argtypes = []
        h.hipDeviceSynchronize.restype = _i
        h.hipMalloc.argtypes, h.hipMalloc.restype = [ctypes.POINTER(_vp), ctypes.c_size_t], _i
        h.hipFree.argtypes, h.hipFree.restype = [_vp], _i
        h.hipEventCreate.argtypes, h.hipEventCreate.restype = [ctypes.POINTER(_vp)], _i
        h.hipEventDestroy.argtypes, h.hipEventDestroy.restype = [_vp], _i
        h.hipEventRecord.argtypes, h.hipEventRecord.restype = [_vp, _vp], _i
        h.hipEventSynchronize.argtypes, h.hipEventSynchronize.restype = [_vp], _i
        h.hipEventElapsedTime.argtypes = [ctypes.POINTER(ctypes.c_float), _vp, _vp]
        h.hipEventElapsedTime.restype = _i
        _HIP = h
    return _HIP


class DeviceBuffer:
    """nbytes of device memory owned by this object (hipMalloc / hipFree),
    for buffers the C ABI fills, such as the drivers' traces."""

    def __init__(self, nbytes: int):
        self.nbytes = int(nbytes)
        p = _vp()
        if _hip().hipMalloc(ctypes.byref(p), max(self.nbytes, 1)) != 0:
            raise QKError("DeviceBuffer", QK_ERR_DEVICE, f"hipMalloc of {self.nbytes} bytes failed")
        self.ptr = p.value

    def host(self, dtype, count: int | None = None):
        """The first count values (all by default) as a host array."""
        import numpy as np
        size = np.dtype(dtype).itemsize
        return copy_to_host(self.ptr, self.nbytes // size if count is None else count, dtype)

    def close(self) -> None:
        if getattr(self, "ptr", None) and _HIP is not None:
            _HIP.hipDeviceSynchronize()
            _HIP.hipFree(self.ptr)
        self.ptr = None

    __del__ = close


class GpuTimer:
    """Device time from start() to stop() on one stream, summed over every
    interval (FastGPU's start_timer / stop_timer, inferencer.cu:1172-1179):
    two HIP events recorded on the stream; stop() waits for the second."""

    def __init__(self, stream=None):
        h = _hip()
        self._stream = stream_handle(stream)
        self._start, self._end = _vp(), _vp()
        if h.hipEventCreate(ctypes.byref(self._start)) != 0 or h.hipEventCreate(ctypes.byref(self._end)) != 0:
            raise QKError("GpuTimer", QK_ERR_DEVICE, "hipEventCreate failed")
        self.seconds = 0.0

    def start(self) -> None:
        if _hip().hipEventRecord(self._start, self._stream) != 0:
            raise QKError("GpuTimer", QK_ERR_DEVICE, "hipEventRecord failed")

    def stop(self) -> None:
        h = _hip()
        ms = ctypes.c_float()
        if h.hipEventRecord(self._end, self._stream) != 0 or h.hipEventSynchronize(self._end) != 0 or \
                h.hipEventElapsedTime(ctypes.byref(ms), self._start, self._end) != 0:
            raise QKError("GpuTimer", QK_ERR_DEVICE, "GPU timer failed")
        self.seconds += ms.value / 1e3

    def close(self) -> None:
        if getattr(self, "_start", None) and _HIP is not None:
            _HIP.hipEventDestroy(self._start)
            _HIP.hipEventDestroy(self._end)
        self._start = self._end = None

    __del__ = close


def _kv_shape(cfg) -> tuple[int, int, int]:
    """(layers, kv_heads, head_dim) of a model config."""
    return cfg["layers"], cfg["kv_heads"], cfg["dim"] // cfg["heads"]


def _load_kv(ptrs, cfg, rows: int, key_cache, value_cache) -> None:
    """Host caches [layer][rows][kv_heads * head_dim] into a driver's
    [layer][kv_heads][rows][head_dim] device caches."""
    import numpy as np
    layers, kvh, hd = _kv_shape(cfg)
    n = layers * rows * kvh * hd
    for dst, a in zip(ptrs, (key_cache, value_cache)):
        a = _cache_array(a, n).reshape(layers, rows, kvh, hd)
        copy_to_device(dst, np.ascontiguousarray(a.transpose(0, 2, 1, 3)), n * 4)


def _kv_rows(ptrs, cfg, rows: int, n: int):
    """Rows 0..n-1 of a driver's head-major caches as two host arrays
    [layer][n][kv_heads * head_dim] (one strided copy per cache)."""
    import numpy as np
    layers, kvh, hd = _kv_shape(cfg)
    if not 0 <= n <= rows:
        raise QKError("kv_rows", QK_ERR_INVALID_ARG, f"{n} rows of a {rows}-row cache")
    out = []
    for src in ptrs:
        a = np.empty((layers, kvh, n, hd), dtype=np.float32)
        if n:
            _copy_2d(a.ctypes.data, n * hd * 4, src, rows * hd * 4, n * hd * 4, layers * kvh, 2)
        out.append(np.ascontiguousarray(a.transpose(0, 2, 1, 3)).reshape(layers, n, kvh * hd))
    return out[0], out[1]


def _load_kv_rows(ptrs, cfg, rows: int, row0: int, key_rows, value_rows) -> None:
    """Host rows [layer][n][kv_heads * head_dim] into rows row0 .. row0+n-1 of
    a driver's head-major caches (one strided copy per cache)."""
    import numpy as np
    layers, kvh, hd = _kv_shape(cfg)
    k = np.asarray(key_rows)
    n = k.shape[1] if k.ndim == 3 else -1
    if n < 0 or not 0 <= row0 <= rows - n:
        raise QKError("load_kv_rows", QK_ERR_INVALID_ARG, f"rows {row0}..{row0 + n - 1} of a {rows}-row cache")
    for dst, a in zip(ptrs, (key_rows, value_rows)):
        a = _cache_array(a, layers * n * kvh * hd).reshape(layers, n, kvh, hd)
        a = np.ascontiguousarray(a.transpose(0, 2, 1, 3))
        if n:
            _copy_2d(dst + row0 * hd * 4, rows * hd * 4, a.ctypes.data, n * hd * 4, n * hd * 4, layers * kvh, 1)


def copy_kv_rows(dst, src, n: int) -> None:
    """Rows 0..n-1 of every layer and KV head of src's caches into dst's (a
    Runner or BatchRunner each; same model), device to device: one strided
    copy per cache."""
    layers, kvh, hd = _kv_shape(dst.cfg)
    rows_of = lambda r: r.cache_rows if hasattr(r, "cache_rows") else r.cfg["context"]
    dr, sr = rows_of(dst), rows_of(src)
    if not 0 <= n <= min(dr, sr):
        raise QKError("copy_kv_rows", QK_ERR_INVALID_ARG, f"{n} rows between caches of {sr} and {dr} rows")
    if n == 0:
        return
    for d, s_ in zip(dst.kv_cache(), src.kv_cache()):
        _copy_2d(d, dr * hd * 4, s_, sr * hd * 4, n * hd * 4, layers * kvh, 3)


def _copy_2d(dst: int, dpitch: int, src: int, spitch: int, width: int, height: int, kind: int) -> None:
    """height rows of width bytes between pitched buffers (hipMemcpy2D; kind
    1 host->device, 2 device->host, 3 device->device), after a device-wide
    synchronisation so no queued step still uses either buffer."""
    h = _hip()
    if h.hipDeviceSynchronize() != 0 or h.hipMemcpy2D(dst, dpitch, src, spitch, width, height, kind) != 0:
        raise QKError("copy_2d", QK_ERR_DEVICE, "hipMemcpy2D failed")


def _cache_array(a, count: int):
    """a as a contiguous float32 array of exactly count values (QKError
    otherwise): caches are copied whole, never partly or past their end."""
    import numpy as np
    a = np.asarray(a)
    if a.dtype != np.float32 or a.size != count:
        raise QKError("load_kv", QK_ERR_INVALID_ARG,
                      f"cache must be float32 with {count} values, got {a.dtype} with {a.size}")
    return np.ascontiguousarray(a)


def copy_to_device(dst: int, host_array, nbytes: int | None = None) -> None:
    """Copy host_array into device memory at dst.  nbytes, when given, is the
    destination's size and must equal the array's.  The device is
    synchronised first, so no queued step on any stream still uses dst."""
    import numpy as np
    a = np.ascontiguousarray(host_array)
    if nbytes is not None and a.nbytes != nbytes:
        raise QKError("copy_to_device", QK_ERR_INVALID_ARG, f"{a.nbytes} bytes for a {nbytes}-byte buffer")
    h = _hip()
    if h.hipDeviceSynchronize() != 0 or h.hipMemcpy(dst, a.ctypes.data, a.nbytes, 1) != 0:
        raise QKError("copy_to_device", QK_ERR_DEVICE, "hipMemcpy host->device failed")


def copy_to_host(src: int, count: int, dtype) -> "object":
    import numpy as np
    out = np.empty(count, dtype=dtype)
    h = _hip()
    if h.hipDeviceSynchronize() != 0 or h.hipMemcpy(out.ctypes.data, src, out.nbytes, 2) != 0:
        raise QKError("copy_to_host", QK_ERR_DEVICE, "hipMemcpy device->host failed")
    return out


def copy_device(dst: int, src: int, nbytes: int) -> None:
    """Device-to-device copy of nbytes (the device is synchronised first)."""
    h = _hip()
    if h.hipDeviceSynchronize() != 0 or h.hipMemcpy(dst, src, nbytes, 3) != 0:
        raise QKError("copy_device", QK_ERR_DEVICE, "hipMemcpy device->device failed")


def _runner_load_kv(self, key_cache, value_cache) -> None:
    """Copy fp32 caches laid out [layer][context][kv_dim] (the reference's
    layout) into the runner's head-major caches."""
    _load_kv(self.kv_cache(), self.cfg, self.cfg["context"], key_cache, value_cache)


def _runner_kv_rows(self, n: int):
    """Rows 0..n-1 of every layer of both caches, host arrays [layer][n][kv_dim]."""
    return _kv_rows(self.kv_cache(), self.cfg, self.cfg["context"], n)


def _runner_logits(self):
    import numpy as np
    return copy_to_host(self.logits_ptr(), self.cfg["vocab"], np.float32)


Runner.load_kv = _runner_load_kv
Runner.kv_rows = _runner_kv_rows
Runner.logits = _runner_logits
