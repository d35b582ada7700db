"""blog_b200 -- B200-native block-quantized linear path of the local-llm engine.

The product is the native library ``lib/libqlinear_b200.so`` (CUDA, sm_100a)
with the C ABI declared in ``include/qlinear_b200.h``.  This module binds that
ABI through ctypes for Python callers (tests, benchmarks).  It mirrors the
reference's launch layer (AI/codes/local-llm/src/backend/cuda/ops/kernel.cuh):
same function names without the ``launch_`` prefix, same argument order and
meaning, device pointers passed as integers (e.g. ``tensor.data_ptr()``).

There is no CPU fallback: if the library is missing the import of ``lib()``
raises, and every call returns the library's status, raised as ``QLError``.
"""
from __future__ import annotations

import ctypes as C
import os

PKG = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(PKG, "lib", "libqlinear_b200.so")
HEADER = os.path.join(os.path.dirname(PKG), "include", "qlinear_b200.h")

# GGML type codes (reference src/tensor/TensorCommon.h:15-33)
F32, F16, Q4_0, Q5_0, Q8_0, Q4_K, Q6_K = 0, 1, 2, 6, 8, 12, 14
BF16 = 30  # activations of the kv8_* calls
BLOCK = {Q4_0: (32, 18), Q5_0: (32, 22), Q8_0: (32, 34), Q4_K: (256, 144), Q6_K: (256, 210)}
QL_OK, QL_EINVAL, QL_ECUDA, QL_EDEVICE = 0, 1, 2, 3
PATH_AUTO, PATH_GEMV, PATH_TENSOR = 0, 1, 2


class QLError(RuntimeError):
    def __init__(self, status: int, msg: str):
        super().__init__(f"qlinear status {status}: {msg}")
        self.status = status


def row_bytes(t: int, k: int) -> int:
    be, bb = BLOCK[t]
    if k % be:
        raise ValueError(f"in_dim {k} is not a multiple of {be}")
    return k // be * bb


P, I, I32, I64, U64, SZ, F = C.c_void_p, C.c_int, C.c_int32, C.c_int64, C.c_uint64, C.c_size_t, C.c_float
SIGNATURES = {
    "ql_set_stream": (I, [P]),
    "ql_get_stream": (P, []),
    "ql_init": (I, [I]),
    "ql_last_error": (C.c_char_p, []),
    "ql_check_device": (I, []),
    "ql_quant_gemv": (I, [I32, P, SZ, P, P, I, I, I]),
    "ql_quant_gemv_add": (I, [I32, P, SZ, P, P, I, I]),
    "ql_quant_matmul": (I, [I32, P, SZ, P, P, I, I, I]),
    "ql_quant_swiglu": (I, [I32, P, P, SZ, SZ, P, P, I, I]),
    "ql_quant_swiglu_indexed": (I, [I32, P, P, SZ, SZ, SZ, SZ, P, P, P, I, I, I]),
    "ql_quant_down_f32_indexed_accum_ordered": (I, [I32, P, SZ, SZ, P, P, P, P, I, I, I]),
    "ql_moe_router_topk": (I, [P, P, P, I, I, I, F]),
    "ql_full_attention_attend": (I, [P, P, P, P, I, P, I, I, I, I, P]),
    "ql_q8_1_row_bytes": (SZ, [I]),
    "ql_quantize_q8_1": (I, [P, P, I, I, I]),
    "ql_quant_gemv_q8_1": (I, [I32, P, SZ, P, P, I, I]),
    "ql_quant_matmul_q8_1": (I, [I32, P, SZ, P, P, I, I, I]),
    "ql_q8_1_mmq_row_bytes": (SZ, [I]),
    "ql_quantize_q8_1_mmq": (I, [P, P, I, I, I]),
    "ql_quant_matmul_q8_1_mmq": (I, [I32, P, SZ, P, P, I, I, I]),
    "ql_full_attention_attend_batch": (I, [P, P, P, P, I, P, I, I, I, I, I, I]),
    "ql_kv8_append": (I, [P, I32, P, I64, P, I64, P, I64, P, I64, I, P, P, F, P, I, I, P, P, I, I]),
    "ql_kv8_attend_workspace": (SZ, [I, I, I, I, I, I, I]),
    "ql_kv8_attend": (I, [P, I32, P, I64, P, I64, P, I64, I, F, P, P, I, I, I, P, SZ]),
    "ql_kv8_attend_form": (I, [P]),
    "ql_kv8_gather": (I, [P, I32, P, P, P, I, P]),
    "ql_logits_apply": (I, [P, I64, P, I64, I, I, P, P, P, SZ]),
    "ql_add_rms_norm": (I, [I32, P, I64, P, I64, P, I64, P, F, P, I64, P, I, I, I, I]),
    "ql_moe_route": (I, [P, I64, P, P, I, I, I, P]),
    "ql_lora_add": (I, [P, P, I64, P, I64, P, I64, P, I, P, I]),
    "ql_lora_add_form": (I, [P]),
    "ql_moe_swiglu_grouped": (I, [I32, P, P, SZ, SZ, SZ, SZ, P, I64, P, I, I, P, I, I, I, I]),
    "ql_moe_down_grouped_accum_ordered": (I, [I32, P, SZ, SZ, P, P, I, I, P, P, I64, I, I, I, I]),
    "ql_quant_embedding": (I, [I32, P, P, P, SZ, I, I]),
    "ql_dequantize_to_f16": (I, [I32, P, P, I64]),
    "ql_dequantize_q4k_to_f16": (I, [P, P, I64]),
    "ql_dequantize_q80_to_f16": (I, [P, P, I64]),
    "ql_dequantize_q50_to_f16": (I, [P, P, I64]),
    "ql_dequantize_q6k_to_f16": (I, [P, P, I64]),
    "ql_dequantize_q40_to_f16": (I, [P, P, I64]),
    "ql_argmax": (I, [P, I, P]),
    "ql_argmax_noalloc": (I, [P, I, P]),
    "ql_quant_gemv_ex": (I, [I32, P, SZ, P, I64, P, I64, I, I, I, P, F, P, I]),
    "ql_quant_swiglu_ex": (I, [I32, P, P, SZ, SZ, P, I64, P, I64, I, I, I, P, F]),
    "ql_quant_gemv_stacked_ex": (I, [I32, I, P, P, P, P, I64, P, I64, I, I, P, F, P]),
    "ql_quant_matmul_ex": (I, [I32, P, SZ, P, I64, P, I64, I, I, I, P, F, P, I, I]),
    "ql_reserve_prefill": (I, [I, I]),
    "ql_quant_gemv_argmax_ex": (I, [I32, P, SZ, P, I64, P, I64, I, I, I, P, F, I, P, P]),
    "ql_gemv_chain_create": (I, [P, I, C.POINTER(C.c_void_p)]),
    "ql_gemv_chain_exchange_bytes": (SZ, [P, I, I]),
    "ql_gemv_chain_create_tp": (I, [P, I, I, I, P, C.POINTER(C.c_void_p)]),
    "ql_gemv_chain_create_batch": (I, [P, I, I, C.POINTER(C.c_void_p)]),
    "ql_ipc_alloc": (I, [SZ, C.POINTER(C.c_void_p), C.c_char_p]),
    "ql_ipc_free": (I, [P]),
    "ql_ipc_open": (I, [C.c_char_p, C.POINTER(C.c_void_p)]),
    "ql_ipc_close": (I, [P]),
    "ql_gemv_chain_run": (I, [P]),
    "ql_gemv_chain_destroy": (I, [P]),
    "ql_comm_bytes": (SZ, [I, I, I]),
    "ql_comm_alloc": (I, [I, I, I, C.POINTER(C.c_void_p), C.c_char_p]),
    "ql_comm_create": (I, [I, I, I, I, P, C.c_char_p, C.POINTER(C.c_void_p)]),
    "ql_comm_destroy": (I, [P]),
    "ql_allreduce_f32": (I, [P, P, I, I]),
    "ql_comm_step": (I, [P]),
    "ql_rms_norm_f32": (I, [P, P, P, I, I, F]),
    "ql_synth_quantized": (I, [I32, U64, I64, I, F, P]),
    "ql_gguf_open": (I, [C.c_char_p, C.POINTER(C.c_void_p)]),
    "ql_gguf_close": (I, [P]),
    "ql_gguf_version": (I, [P]),
    "ql_gguf_tensor_count": (I64, [P]),
    "ql_gguf_find_tensor": (I64, [P, C.c_char_p]),
    "ql_gguf_tensor_info": (I, [P, I64, C.POINTER(C.c_char_p), C.POINTER(C.c_int32), C.POINTER(C.c_int32), P,
                                C.POINTER(C.c_void_p), C.POINTER(C.c_size_t)]),
    "ql_gguf_metadata_type": (I, [P, C.c_char_p]),
    "ql_gguf_metadata_int": (I, [P, C.c_char_p, C.POINTER(C.c_int64)]),
    "ql_gguf_metadata_float": (I, [P, C.c_char_p, C.POINTER(C.c_double)]),
    "ql_gguf_metadata_string": (I, [P, C.c_char_p, C.POINTER(C.c_char_p)]),
    "ql_gguf_metadata_array_len": (I64, [P, C.c_char_p]),
    "ql_gguf_metadata_array_int": (I, [P, C.c_char_p, I64, C.POINTER(C.c_int64)]),
    "ql_gguf_metadata_array_float": (I, [P, C.c_char_p, I64, C.POINTER(C.c_double)]),
    "ql_gguf_metadata_array_string": (I, [P, C.c_char_p, I64, C.POINTER(C.c_char_p)]),
    "ql_gguf_validate": (I, [P]),
    "ql_weight_upload": (I, [P, SZ, I64, I64, SZ, SZ, P]),
    "ql_row_bytes": (SZ, [I32, I]),
    "ql_last_launch_count": (I, []),
}

_lib = None


def lib() -> C.CDLL:
    """The loaded native library (raises if it has not been built)."""
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise ImportError(f"{LIB_PATH} is missing: run `python -m blog_b200.build` (there is no CPU fallback)")
        L = C.CDLL(LIB_PATH)
        for name, (res, args) in SIGNATURES.items():
            fn = getattr(L, name)
            fn.restype = res
            fn.argtypes = args
        _lib = L
    return _lib


def _check(status: int) -> None:
    if status != QL_OK:
        raise QLError(status, lib().ql_last_error().decode(errors="replace"))


def _call(name: str, *args) -> None:
    _check(getattr(lib(), name)(*args))


# ---- thin wrappers, names follow the reference's launch_* functions ----------
def set_stream(stream_handle: int | None) -> None:
    _call("ql_set_stream", stream_handle or None)


def init(device: int = 0) -> None:
    _call("ql_init", device)


def check_device() -> None:
    _call("ql_check_device")


def quant_gemv(t, weight, rb, x, y, out_dim, in_dim, m):
    _call("ql_quant_gemv", t, weight, rb, x, y, out_dim, in_dim, m)


def quant_gemv_add(t, weight, rb, x, y, out_dim, in_dim):
    _call("ql_quant_gemv_add", t, weight, rb, x, y, out_dim, in_dim)


def quant_matmul(t, weight, rb, x, y, out_dim, in_dim, m):
    _call("ql_quant_matmul", t, weight, rb, x, y, out_dim, in_dim, m)


def quant_matmul_ex(t, w, rb, x, x_stride, y, y_stride, out_dim, in_dim, m, gamma=None, eps=0.0, bias=None,
                    accumulate=False, path=PATH_AUTO):
    """Prefill GEMM; path PATH_TENSOR forces the tcgen05 kernel, PATH_GEMV the streaming engine."""
    _call("ql_quant_matmul_ex", t, w, rb, x, x_stride, y, y_stride, out_dim, in_dim, m, gamma, eps, bias,
          1 if accumulate else 0, path)


IPC_HANDLE_BYTES = 64


class Comm:
    """Peer-memory all-reduce communicator of one rank (see include/qlinear_b200.h).

    `exchange_handles(own_handle) -> list of handles in rank order` is supplied by the
    caller (e.g. torch.distributed.all_gather_object); the library stays host-agnostic."""

    def __init__(self, rank, world, max_floats, slots, exchange_handles):
        ptr = C.c_void_p()
        hbuf = C.create_string_buffer(IPC_HANDLE_BYTES)
        _call("ql_comm_alloc", world, max_floats, slots, C.byref(ptr), hbuf)
        handles = exchange_handles(bytes(hbuf.raw))
        if len(handles) != world or any(len(h) != IPC_HANDLE_BYTES for h in handles):
            raise ValueError("exchange_handles must return one 64-byte handle per rank")
        comm = C.c_void_p()
        _call("ql_comm_create", rank, world, max_floats, slots, ptr, b"".join(handles), C.byref(comm))
        self.handle, self.max_floats, self.slots = comm, max_floats, slots

    def allreduce(self, buf_ptr, n, slot):
        _call("ql_allreduce_f32", self.handle, buf_ptr, n, slot)

    def step(self):
        _call("ql_comm_step", self.handle)

    def close(self):
        if self.handle:
            _call("ql_comm_destroy", self.handle)
            self.handle = None


def quant_gemv_argmax_ex(t, w, rb, x, x_stride, logits, logits_stride, out_dim, in_dim, m, gamma=None, eps=0.0,
                         index_offset=0, out_idx=None, out_key=None):
    """Fused LM head + greedy argmax (see include/qlinear_b200.h)."""
    _call("ql_quant_gemv_argmax_ex", t, w, rb, x, x_stride, logits, logits_stride, out_dim, in_dim, m, gamma, eps,
          index_offset, out_idx, out_key)


OP_STORE, OP_ADD, OP_SWIGLU, OP_MLP = 0, 1, 2, 3


class ChainOp(C.Structure):
    """ql_chain_op (include/qlinear_b200.h)."""
    _fields_ = [("kind", C.c_int32), ("quant_type", C.c_int32), ("nsrc", C.c_int32),
                ("w", C.c_void_p * 3), ("row_bytes", C.c_size_t * 3), ("rows", C.c_int32 * 3),
                ("in_dim", C.c_int32), ("x", C.c_void_p), ("gamma", C.c_void_p), ("eps", C.c_float),
                ("bias", C.c_void_p), ("y", C.c_void_p), ("argmax_idx", C.c_void_p), ("argmax_offset", C.c_int32),
                ("reduce", C.c_int32), ("x_stride", C.c_int64), ("y_stride", C.c_int64),
                ("rope_pos", C.c_void_p), ("rope_theta", C.c_float), ("rope_rows", C.c_int32),
                ("head_dim", C.c_int32)]


def chain_op(kind, weights, row_bytes, rows, in_dim, x, y, gamma=None, eps=0.0, bias=None, argmax_idx=None,
             argmax_offset=0, quant_type=Q4_K, reduce=False, x_stride=0, y_stride=0, rope_pos=None, rope_theta=0.0,
             rope_rows=0, head_dim=0):
    op = ChainOp()
    op.kind, op.quant_type, op.nsrc, op.in_dim = kind, quant_type, len(weights), in_dim
    for i, (w, rb, r) in enumerate(zip(weights, row_bytes, rows)):
        op.w[i], op.row_bytes[i], op.rows[i] = w, rb, r
    op.x, op.y, op.gamma, op.eps, op.bias = x, y, gamma, eps, bias
    op.argmax_idx, op.argmax_offset, op.reduce = argmax_idx, argmax_offset, 1 if reduce else 0
    op.x_stride, op.y_stride = x_stride, y_stride
    op.rope_pos, op.rope_theta, op.rope_rows, op.head_dim = rope_pos, rope_theta, rope_rows, head_dim
    return op


class GemvChain:
    """A list of single-token GEMV ops run as one persistent launch (ql_gemv_chain_*).

    Tensor parallel: pass rank, world and `exchange_handles(own_handle) -> handles in rank
    order` (any host channel, e.g. torch.distributed.all_gather_object); ops with reduce=True
    then sum their partials over ranks inside the kernel through peer memory."""

    def __init__(self, ops, rank=0, world=1, exchange_handles=None, tokens=None):
        """tokens=None: the one-token chain; tokens=M (1..32): the batched chain over M tokens."""
        arr = (ChainOp * len(ops))(*ops)
        h = C.c_void_p()
        self.own, self.mapped = None, []
        if tokens is not None:
            _call("ql_gemv_chain_create_batch", C.cast(arr, C.c_void_p), len(ops), tokens, C.byref(h))
        elif world == 1:
            _call("ql_gemv_chain_create", C.cast(arr, C.c_void_p), len(ops), C.byref(h))
        else:
            nbytes = lib().ql_gemv_chain_exchange_bytes(C.cast(arr, C.c_void_p), len(ops), world)
            own = C.c_void_p()
            hb = C.create_string_buffer(IPC_HANDLE_BYTES)
            _call("ql_ipc_alloc", max(nbytes, 256), C.byref(own), hb)
            self.own = own
            handles = exchange_handles(bytes(hb.raw))
            ptrs = (C.c_void_p * world)()
            for r, hr in enumerate(handles):
                if r == rank:
                    ptrs[r] = own.value
                else:
                    m = C.c_void_p()
                    _call("ql_ipc_open", hr, C.byref(m))
                    self.mapped.append(m)
                    ptrs[r] = m.value
            _call("ql_gemv_chain_create_tp", C.cast(arr, C.c_void_p), len(ops), rank, world, C.cast(ptrs, C.c_void_p),
                  C.byref(h))
        self.handle = h

    def run(self):
        _call("ql_gemv_chain_run", self.handle)

    def close(self):
        """Release the chain; with world > 1 call it on every rank after a host barrier."""
        if self.handle:
            _call("ql_gemv_chain_destroy", self.handle)
            self.handle = None
        for m in self.mapped:
            _call("ql_ipc_close", m)
        self.mapped = []
        if self.own is not None:
            _call("ql_ipc_free", self.own)
            self.own = None


def reserve_prefill(max_tokens, max_in_dim):
    _call("ql_reserve_prefill", max_tokens, max_in_dim)


def quant_swiglu(t, gw, uw, grb, urb, x, act, ffn_dim, in_dim):
    _call("ql_quant_swiglu", t, gw, uw, grb, urb, x, act, ffn_dim, in_dim)


def quant_swiglu_indexed(t, gw, uw, geb, ueb, grb, urb, x, ids, act, k, ffn_dim, in_dim):
    _call("ql_quant_swiglu_indexed", t, gw, uw, geb, ueb, grb, urb, x, ids, act, k, ffn_dim, in_dim)


def quant_down_f32_indexed_accum_ordered(t, dw, deb, drb, act, ids, rw, out, k, hidden, ffn_dim):
    _call("ql_quant_down_f32_indexed_accum_ordered", t, dw, deb, drb, act, ids, rw, out, k, hidden, ffn_dim)


def moe_router_topk(logits, idx, w, tokens, n_experts, k, scale):
    _call("ql_moe_router_topk", logits, idx, w, tokens, n_experts, k, scale)


def q8_1_row_bytes(in_dim):
    return lib().ql_q8_1_row_bytes(in_dim)


def quantize_q8_1(x, xq, in_dim, m, store_raw_sum=False):
    _call("ql_quantize_q8_1", x, xq, in_dim, m, int(store_raw_sum))


def quant_gemv_q8_1(t, w, rb, xq, y, out_dim, in_dim):
    _call("ql_quant_gemv_q8_1", t, w, rb, xq, y, out_dim, in_dim)


def quant_matmul_q8_1(t, w, rb, xq, y, out_dim, in_dim, m):
    _call("ql_quant_matmul_q8_1", t, w, rb, xq, y, out_dim, in_dim, m)


def q8_1_mmq_row_bytes(in_dim):
    return lib().ql_q8_1_mmq_row_bytes(in_dim)


def quantize_q8_1_mmq(x, xq, in_dim, m, store_raw_sum=False):
    _call("ql_quantize_q8_1_mmq", x, xq, in_dim, m, int(store_raw_sum))


def quant_matmul_q8_1_mmq(t, w, rb, xq, y, out_dim, in_dim, m):
    _call("ql_quant_matmul_q8_1_mmq", t, w, rb, xq, y, out_dim, in_dim, m)


def full_attention_attend(q, gate, kc, vc, kv_bf16, attn, n_heads, kv_heads, head_dim, max_seq_len, pos_dev):
    _call("ql_full_attention_attend", q, gate, kc, vc, int(kv_bf16), attn, n_heads, kv_heads, head_dim, max_seq_len,
          pos_dev)


def full_attention_attend_batch(q, gate, kc, vc, kv_bf16, attn, tokens, n_heads, kv_heads, head_dim, max_seq_len,
                                start_pos):
    _call("ql_full_attention_attend_batch", q, gate, kc, vc, int(kv_bf16), attn, tokens, n_heads, kv_heads, head_dim,
          max_seq_len, start_pos)


KV8_BLOCK = 32


class KV8Cache(C.Structure):
    """ql_kv8_cache (include/qlinear_b200.h): the caller's buffers of a paged 8-bit KV cache."""
    _fields_ = [("k_codes", C.c_void_p), ("v_codes", C.c_void_p), ("k_scale", C.c_void_p), ("v_scale", C.c_void_p),
                ("k_open", C.c_void_p), ("v_open", C.c_void_p), ("page_table", C.c_void_p), ("slots", C.c_void_p),
                ("n_pages", C.c_int32), ("n_slots", C.c_int32), ("n_seqs", C.c_int32), ("max_pages", C.c_int32),
                ("kv_heads", C.c_int32), ("head_dim", C.c_int32)]


def kv8_cache(k_codes, v_codes, k_scale, v_scale, k_open, v_open, page_table, slots, n_pages, n_slots, n_seqs,
              max_pages, kv_heads, head_dim):
    return KV8Cache(k_codes, v_codes, k_scale, v_scale, k_open, v_open, page_table, slots, n_pages, n_slots, n_seqs,
                    max_pages, kv_heads, head_dim)


def kv8_append(cache, t, q, q_stride, k, k_stride, v, v_stride, q_out, q_out_stride, n_heads, q_gamma, k_gamma, eps,
               rope, rotary_dim, max_positions, kv_len, q_start, rows, max_q_len):
    """Norm and rotation of q and k per head, k and v stored into the cache (see include/qlinear_b200.h)."""
    _call("ql_kv8_append", C.byref(cache), t, q, q_stride, k, k_stride, v, v_stride, q_out, q_out_stride, n_heads,
          q_gamma, k_gamma, eps, rope, rotary_dim, max_positions, kv_len, q_start, rows, max_q_len)


def kv8_attend_workspace(n_heads, kv_heads, head_dim, n_seqs, rows, max_q_len, max_kv_len) -> int:
    return int(lib().ql_kv8_attend_workspace(n_heads, kv_heads, head_dim, n_seqs, rows, max_q_len, max_kv_len))


def kv8_attend(cache, t, q, q_stride, gate, gate_stride, out, out_stride, n_heads, scale, kv_len, q_start, rows,
               max_q_len, max_kv_len, workspace, workspace_bytes):
    _call("ql_kv8_attend", C.byref(cache), t, q, q_stride, gate, gate_stride, out, out_stride, n_heads, scale, kv_len,
          q_start, rows, max_q_len, max_kv_len, workspace, workspace_bytes)


KV8_FORM_SPLIT, KV8_FORM_TILES = 1, 2


def kv8_attend_form():
    """(form, CTAs that shared a row's keys) of this thread's last kv8_attend (see include/qlinear_b200.h)."""
    ctas = C.c_int(0)
    return int(lib().ql_kv8_attend_form(C.byref(ctas))), ctas.value


def kv8_gather(cache, t, k_out, v_out, start, count, kv_len):
    _call("ql_kv8_gather", C.byref(cache), t, k_out, v_out, start, count, kv_len)


class LogitsRules(C.Structure):
    """ql_logits_rules (include/qlinear_b200.h)."""
    _fields_ = [("history", C.c_void_p), ("history_stride", C.c_int64), ("history_len", C.c_void_p),
                ("prompt_len", C.c_void_p), ("repetition", C.c_void_p), ("frequency", C.c_void_p),
                ("presence", C.c_void_p), ("bias_ids", C.c_void_p), ("bias_values", C.c_void_p),
                ("bias_start", C.c_void_p), ("mask", C.c_void_p), ("mask_stride", C.c_int64),
                ("mask_rows", C.c_int32), ("mask_row", C.c_void_p)]


def logits_rules(history=None, history_stride=0, history_len=None, prompt_len=None, repetition=None, frequency=None,
                 presence=None, bias_ids=None, bias_values=None, bias_start=None, mask=None, mask_stride=0, mask_rows=0,
                 mask_row=None):
    return LogitsRules(history, history_stride, history_len, prompt_len, repetition, frequency, presence, bias_ids,
                       bias_values, bias_start, mask, mask_stride, mask_rows, mask_row)


def logits_apply(logits, logits_stride, out, out_stride, rows, vocab, rules, token, workspace, workspace_bytes):
    _call("ql_logits_apply", logits, logits_stride, out, out_stride, rows, vocab, C.byref(rules), token, workspace,
          workspace_bytes)


Q8_NONE, Q8_ROWS, Q8_MMQ = 0, 1, 2


def add_rms_norm(t, x, x_stride, residual, residual_stride, sum_, sum_stride, gamma, eps, y, y_stride, xq, layout,
                 store_raw_sum, rows, hidden):
    """Residual addition, RMS norm and its Q8_1 rows in one launch (see include/qlinear_b200.h)."""
    _call("ql_add_rms_norm", t, x, x_stride, residual, residual_stride, sum_, sum_stride, gamma, eps, y, y_stride, xq,
          layout, int(store_raw_sum), rows, hidden)


ROUTE_SOFTMAX, ROUTE_SIGMOID = 0, 1


class MoeRouteRule(C.Structure):
    """ql_moe_route_rule (include/qlinear_b200.h)."""
    _fields_ = [("score", C.c_int32), ("bias", C.c_void_p), ("n_groups", C.c_int32), ("top_groups", C.c_int32),
                ("group_best", C.c_int32), ("renormalise", C.c_int32), ("scale", C.c_float)]


def moe_route_rule(score, bias=None, n_groups=1, top_groups=1, group_best=1, renormalise=False, scale=1.0):
    return MoeRouteRule(score, bias, n_groups, top_groups, group_best, int(renormalise), scale)


def moe_route(logits, logits_stride, idx, w, tokens, n_experts, k, rule):
    """The k experts of each token and their weights (see include/qlinear_b200.h)."""
    _call("ql_moe_route", logits, logits_stride, idx, w, tokens, n_experts, k, C.byref(rule))


class LoraPool(C.Structure):
    """ql_lora_pool (include/qlinear_b200.h): slots of low-rank adapters for one to three projections of one input."""
    _fields_ = [("type", C.c_int32), ("n_proj", C.c_int32), ("a", C.c_void_p * 3), ("b", C.c_void_p * 3),
                ("out_dim", C.c_int32 * 3), ("in_dim", C.c_int32), ("n_adapters", C.c_int32), ("max_rank", C.c_int32),
                ("rank", C.c_void_p), ("scale", C.c_void_p)]


def lora_pool(t, a, b, out_dims, in_dim, n_adapters, max_rank, rank=None, scale=None):
    """a, b and out_dims are Python sequences, one entry per projection (<= 3)."""
    if not len(a) == len(b) == len(out_dims) or len(a) > 3:
        raise ValueError("a, b and out_dims have one entry per projection, at most 3")
    pool = LoraPool(type=t, n_proj=len(a), in_dim=in_dim, n_adapters=n_adapters, max_rank=max_rank, rank=rank, scale=scale)
    for i in range(len(a)):
        pool.a[i], pool.b[i], pool.out_dim[i] = a[i], b[i], out_dims[i]
    return pool


def lora_add(pool, x, x_stride, base, base_stride, y, y_stride, adapter, n_seqs, q_start, rows):
    """y = base + the rows' adapters applied to x (see include/qlinear_b200.h)."""
    _call("ql_lora_add", C.byref(pool), x, x_stride, base, base_stride, y, y_stride, adapter, n_seqs, q_start, rows)


LORA_FORM_ROWS, LORA_FORM_TILES = 1, 2


def lora_add_form():
    """(form, CTAs that shared a tile of rows) of this thread's last lora_add (see include/qlinear_b200.h)."""
    ctas = C.c_int(0)
    return int(lib().ql_lora_add_form(C.byref(ctas))), ctas.value


def moe_swiglu_grouped(t, gw, uw, geb, ueb, grb, urb, x, x_stride, ids, expert_begin, n_experts, act, tokens, k,
                       ffn_dim, in_dim):
    _call("ql_moe_swiglu_grouped", t, gw, uw, geb, ueb, grb, urb, x, x_stride, ids, expert_begin, n_experts, act,
          tokens, k, ffn_dim, in_dim)


def moe_down_grouped_accum_ordered(t, dw, deb, drb, act, ids, expert_begin, n_experts, rw, out, out_stride, tokens,
                                   k, hidden, ffn_dim):
    _call("ql_moe_down_grouped_accum_ordered", t, dw, deb, drb, act, ids, expert_begin, n_experts, rw, out,
          out_stride, tokens, k, hidden, ffn_dim)


def quant_embedding(t, ids, out, table, rb, hidden, n):
    _call("ql_quant_embedding", t, ids, out, table, rb, hidden, n)


def dequantize_to_f16(t, src, out, n):
    _call("ql_dequantize_to_f16", t, src, out, n)


def argmax(logits, n, out_idx):
    _call("ql_argmax", logits, n, out_idx)


def argmax_noalloc(logits, n, out_idx):
    """ql_argmax without device allocation (fixed in-library scratch; see the header)."""
    _call("ql_argmax_noalloc", logits, n, out_idx)


def quant_gemv_ex(t, w, rb, x, x_stride, y, y_stride, out_dim, in_dim, m, gamma=None, eps=0.0, bias=None,
                  accumulate=False):
    _call("ql_quant_gemv_ex", t, w, rb, x, x_stride, y, y_stride, out_dim, in_dim, m, gamma, eps, bias,
          1 if accumulate else 0)


def quant_gemv_stacked_ex(t, weights, row_bytes_list, rows, x, x_stride, y, y_stride, in_dim, m, gamma=None,
                          eps=0.0, bias=None):
    """Stacked projections (e.g. fused q/k/v): weights, row_bytes_list, rows are Python sequences (<= 3)."""
    n = len(weights)
    W = (C.c_void_p * n)(*weights)
    RB = (C.c_size_t * n)(*row_bytes_list)
    R = (C.c_int * n)(*rows)
    _call("ql_quant_gemv_stacked_ex", t, n, C.cast(W, C.c_void_p), C.cast(RB, C.c_void_p), C.cast(R, C.c_void_p), x,
          x_stride, y, y_stride, in_dim, m, gamma, eps, bias)


def quant_swiglu_ex(t, gw, uw, grb, urb, x, x_stride, act, act_stride, ffn_dim, in_dim, m, gamma=None, eps=0.0):
    _call("ql_quant_swiglu_ex", t, gw, uw, grb, urb, x, x_stride, act, act_stride, ffn_dim, in_dim, m, gamma, eps)


def rms_norm_f32(x, y, gamma, rows, hidden, eps):
    _call("ql_rms_norm_f32", x, y, gamma, rows, hidden, eps)


def synth_quantized(t, seed, rows, in_dim, std, dst):
    _call("ql_synth_quantized", t, seed, rows, in_dim, std, dst)


def weight_upload(host_ptr, row_bytes, row0, nrows, byte0, nbytes_per_row, dst):
    """Host GGUF rows (a matrix or a tensor-parallel shard of it) to device memory (ql_weight_upload)."""
    _call("ql_weight_upload", host_ptr, row_bytes, row0, nrows, byte0, nbytes_per_row, dst)


def last_launch_count() -> int:
    return int(lib().ql_last_launch_count())
