"""Python binding of the hesa-b200 C ABI (include/hesa_cuda.h) over ctypes.

This is the host-side mirror of the reference's operator interface for the
hot path: ``qmatvec`` is ``hesa::Backend::matmul`` (include/hesa/backend.hpp:
43-44) for a quantized weight, with the same argument meaning (W [n_out, k],
activations [batch, k], out = scale * W @ x) and the same error codes
(``hesa::Error``, include/hesa/result.hpp:14-30), raised as ``HesaError``.

PyTorch is only plumbing here: it owns device memory and streams. Every
computation runs in ``libhesa_cuda.so``; if that library cannot be built or
loaded, every call raises -- there is no fallback path.
"""
from __future__ import annotations

import ctypes
import os

import hesa_build as _build

Q4_0, Q8_0, Q4_K, Q5_K, Q6_K = 2, 8, 12, 13, 14
QTYPES = {"Q4_0": Q4_0, "Q8_0": Q8_0, "Q4_K": Q4_K, "Q5_K": Q5_K, "Q6_K": Q6_K}
BLOCK_ELEMS = {Q4_0: 32, Q8_0: 32, Q4_K: 256, Q5_K: 256, Q6_K: 256}
BLOCK_BYTES = {Q4_0: 18, Q8_0: 34, Q4_K: 144, Q5_K: 176, Q6_K: 210}

ERRORS = {0: "SUCCESS", 1: "OUT_OF_MEMORY", 2: "INVALID_ARGUMENT", 3: "BACKEND_NOT_AVAILABLE",
          6: "SHAPE_MISMATCH", 8: "INVALID_FORMAT", 9: "CUDA_ERROR", 14: "INTERNAL_ERROR"}

# (name, restype, argtypes) of every function include/hesa_cuda.h declares
_vp, _i64, _sz, _int, _f = ctypes.c_void_p, ctypes.c_int64, ctypes.c_size_t, ctypes.c_int, ctypes.c_float


class Model(ctypes.Structure):
    """hesa_cuda_model (include/hesa_cuda.h)."""
    _fields_ = [("n_layer", ctypes.c_int32), ("d_model", ctypes.c_int32), ("n_head", ctypes.c_int32),
                ("n_kv_head", ctypes.c_int32), ("head_dim", ctypes.c_int32), ("d_ff", ctypes.c_int32),
                ("vocab", ctypes.c_int32), ("ctx", ctypes.c_int32), ("rms_eps", ctypes.c_float),
                ("rope_base", ctypes.c_float), ("qtype", ctypes.c_int32)]


class Layer(ctypes.Structure):
    """hesa_cuda_layer (include/hesa_cuda.h): device pointers of one layer."""
    _fields_ = [(n, ctypes.c_void_p) for n in ("wq", "wk", "wv", "wo", "w_gate", "w_up", "w_down", "attn_norm",
                                              "ffn_norm", "k_cache", "v_cache")]



class PagedKVStruct(ctypes.Structure):
    """hesa_cuda_paged_kv (include/hesa_cuda.h)."""
    _fields_ = [("k", ctypes.c_void_p), ("v", ctypes.c_void_p), ("page_stride", ctypes.c_int64),
                ("layer_stride", ctypes.c_int64), ("n_layer", ctypes.c_int32), ("n_pages", ctypes.c_int32),
                ("page_size", ctypes.c_int32), ("n_kv_head", ctypes.c_int32), ("head_dim", ctypes.c_int32),
                ("table", ctypes.c_void_p), ("seq_len", ctypes.c_void_p), ("page_refs", ctypes.c_void_p),
                ("n_slots", ctypes.c_int32), ("max_pages", ctypes.c_int32)]


class TokenBatchStruct(ctypes.Structure):
    """hesa_cuda_token_batch (include/hesa_cuda.h)."""
    _fields_ = [("slots", ctypes.c_void_p), ("q_start", ctypes.c_void_p), ("n_seq", ctypes.c_int32),
                ("n_tokens", ctypes.c_int32), ("max_new", ctypes.c_int32), ("max_len", ctypes.c_int32)]


class AttnOptionsStruct(ctypes.Structure):
    """hesa_cuda_attn_options (include/hesa_cuda.h)."""
    _fields_ = [("scale", ctypes.c_float), ("softcap", ctypes.c_float), ("window", ctypes.c_int32),
                ("slopes", ctypes.c_void_p), ("prefix", ctypes.c_void_p)]


_kvp, _batchp, _optp = ctypes.POINTER(PagedKVStruct), ctypes.POINTER(TokenBatchStruct), ctypes.POINTER(AttnOptionsStruct)
_i32 = ctypes.c_int32

SIGNATURES = [
    ("hesa_cuda_paged_attention_workspace_size", _sz, [_kvp, _batchp, _i64]),
    ("hesa_cuda_paged_attention", _int, [_kvp, _i32, _batchp, _vp, _i64, _vp, _i64, _i64, _optp, _vp, _sz, _vp]),
    ("hesa_cuda_rope_kv_paged", _int, [_kvp, _i32, _batchp, _vp, _i64, _vp, _i64, _vp, _i64, _i64, _vp, _i32, _vp]),
    ("hesa_cuda_kv_pages_workspace_size", _sz, [_kvp]),
    ("hesa_cuda_kv_reserve", _int, [_kvp, _vp, _vp, _i32, _vp, _sz, _vp]),
    ("hesa_cuda_kv_free", _int, [_kvp, _vp, _i32, _vp, _sz, _vp]),
    ("hesa_cuda_kv_fork", _int, [_kvp, _vp, _vp, _i32, _vp, _sz, _vp]),
    ("hesa_cuda_kv_compact", _int, [_kvp, _vp, _vp, _sz, _vp]),
    ("hesa_cuda_kv_copy_pages", _int, [_kvp, _vp, _vp, _i32, _vp, _sz, _vp]),
    ("hesa_cuda_token_logprobs_workspace_size", _sz, [_i64, _i64, _i32]),
    ("hesa_cuda_token_logprobs", _int, [_vp, _i64, _i64, _i64, _vp, _i32, _vp, _vp, _vp, _vp, _vp, _sz, _vp]),
    ("hesa_cuda_version", ctypes.c_char_p, []),
    ("hesa_cuda_row_bytes", _sz, [_int, _i64]),
    ("hesa_cuda_qmatvec_workspace_size", _sz, [_int, _i64, _i64, _i64]),
    ("hesa_cuda_qmatvec", _int, [_int, _vp, _i64, _i64, _vp, _i64, _i64, _vp, _i64, _f, _vp, _sz, _vp]),
    ("hesa_cuda_qmatvec_noalloc", _int, [_int, _vp, _i64, _i64, _vp, _i64, _i64, _vp, _i64, _f, _vp]),
    ("hesa_cuda_dequantize", _int, [_int, _vp, _i64, _i64, _vp, _i64, _vp]),
    ("hesa_cuda_quantize", _int, [_int, _vp, _i64, _i64, _i64, _vp, _vp]),
    ("hesa_cuda_device_status", _int, [_vp, ctypes.POINTER(_int)]),
    ("hesa_cuda_clear_device_status", _int, [_vp]),
    ("hesa_cuda_last_error", ctypes.c_char_p, []),
    ("hesa_cuda_matmul_f32", _int, [_vp, _i64, _i64, _vp, _i64, _i64, _vp, _i64, _f, _vp]),
    ("hesa_cuda_rms_norm", _int, [_vp, _vp, _vp, _i64, _i64, _f, _vp]),
    ("hesa_cuda_silu_mul", _int, [_vp, _vp, _vp, _i64, _vp]),
    ("hesa_cuda_add", _int, [_vp, _vp, _vp, _i64, _vp]),
    ("hesa_cuda_mul", _int, [_vp, _vp, _vp, _i64, _vp]),
    ("hesa_cuda_softmax", _int, [_vp, _vp, _i64, _i64, _vp]),
    ("hesa_cuda_rope_table", _int, [_vp, ctypes.c_int32, _i64, _f]),
    ("hesa_cuda_rope", _int, [_vp, _i64, _i64, _vp, ctypes.c_int32, _vp, ctypes.c_int32, _vp]),
    ("hesa_cuda_kv_store", _int, [_vp, _vp, _vp, _vp, _i64, _i64, _vp, ctypes.c_int32, _vp]),
    ("hesa_cuda_attention_workspace_size", _sz, [_i64, _i64, _i64]),
    ("hesa_cuda_attention", _int, [_vp, _vp, _vp, _vp, _i64, _i64, _i64, _i64, _vp, ctypes.c_int32, _vp, _sz,
                                   _vp]),
    ("hesa_cuda_decode_workspace_size", _sz, [ctypes.POINTER(Model)]),
    ("hesa_cuda_embed", _int, [_int, _vp, _i64, _i64, _vp, _vp, _vp]),
    ("hesa_cuda_decode_step", _int, [ctypes.POINTER(Model), ctypes.POINTER(Layer), _vp, _vp, _vp, ctypes.c_int32,
                                     _vp, _vp, _vp, _vp, _sz, _vp]),
    ("hesa_cuda_peer_alloc", _int, [_sz, ctypes.POINTER(_vp), _vp]),
    ("hesa_cuda_peer_free", _int, [_vp]),
    ("hesa_cuda_peer_open", _int, [_vp, ctypes.POINTER(_vp)]),
    ("hesa_cuda_peer_close", _int, [_vp]),
    ("hesa_cuda_qmatvec_gather", _int, [_int, _vp, _i64, _i64, _vp, _f, ctypes.POINTER(_vp), _int, _vp, _vp]),
    ("hesa_cuda_peer_barrier", _int, [ctypes.POINTER(_vp), _int, _int, _vp, _vp]),
    ("hesa_cuda_gather_tagged_workspace_size", _sz, [_int, _i64, _i64]),
    ("hesa_cuda_qmatvec_gather_tagged", _int, [_int, _vp, _i64, _i64, _vp, _f, ctypes.POINTER(_vp), _i64, _int,
                                               _vp, _vp, _sz, _vp]),
    ("hesa_cuda_peer_collect", _int, [_vp, _i64, _i64, _vp, _vp, _vp]),
    ("hesa_cuda_set_peer_wait_limit_us", _int, [ctypes.c_uint32]),
    ("hesa_cuda_decode_step_sharded", _int, [ctypes.POINTER(Model), _vp, ctypes.POINTER(Layer), _vp, _vp, _vp,
                                             ctypes.c_int32, _vp, _vp, _vp, _vp, _sz, _vp]),
]


class Shard(ctypes.Structure):
    """hesa_cuda_shard (include/hesa_cuda.h): one rank of a head-sharded decode."""
    _fields_ = [("rank", ctypes.c_int32), ("world", ctypes.c_int32), ("a_peers", ctypes.c_void_p),
                ("gu_peers", ctypes.c_void_p), ("logits_peers", ctypes.c_void_p), ("token_count", ctypes.c_void_p)]

    def __init__(self, rank, world, a, gu, logits, token_count):
        super().__init__(rank, world, ctypes.cast(a, ctypes.c_void_p), ctypes.cast(gu, ctypes.c_void_p),
                         ctypes.cast(logits, ctypes.c_void_p), token_count)


class HesaError(RuntimeError):
    def __init__(self, code: int, msg: str):
        super().__init__(f"{ERRORS.get(code, code)} ({code}): {msg}")
        self.code = code


_lib = None


def library_path() -> str:
    return _build.CUDA_SO


def lib() -> ctypes.CDLL:
    """Load libhesa_cuda.so, building it first if it is missing or stale."""
    global _lib
    if _lib is None:
        path = _build.build_cuda()
        L = ctypes.CDLL(path)
        for name, res, args in SIGNATURES:
            fn = getattr(L, name)
            fn.restype = res
            fn.argtypes = args
        _lib = L
    return _lib


def _check(rc: int) -> None:
    if rc != 0:
        raise HesaError(rc, lib().hesa_cuda_last_error().decode())


def _stream_handle(stream) -> int | None:
    if stream is None:
        import torch
        return torch.cuda.current_stream().cuda_stream or None
    if isinstance(stream, int):
        return stream or None
    return stream.cuda_stream or None


def row_bytes(qtype: int, k: int) -> int:
    return int(lib().hesa_cuda_row_bytes(qtype, k))


def workspace_bytes(qtype: int, n_out: int, k: int, batch: int = 1) -> int:
    return int(lib().hesa_cuda_qmatvec_workspace_size(qtype, n_out, k, batch))


def make_workspace(qtype: int, n_out: int, k: int, batch: int = 1, device=None):
    """A zero-filled device workspace of the size the matvec asks for."""
    import torch
    nbytes = max(16, workspace_bytes(qtype, n_out, k, batch))
    return torch.zeros(nbytes, dtype=torch.uint8, device=device or "cuda")


def qmatvec(qtype: int, w, x, y=None, scale: float = 1.0, workspace=None, stream=None, k: int | None = None):
    """y = scale * W @ x for packed W [n_out, row_bytes] (uint8, CUDA) and fp32
    x [k] or [batch, k]; returns y [n_out] or [batch, n_out]."""
    import torch
    squeeze = x.dim() == 1
    x2 = x.unsqueeze(0) if squeeze else x
    batch, kk = x2.shape
    k = k or kk
    n_out = w.shape[0]
    if y is None:
        y = torch.empty((batch, n_out), dtype=torch.float32, device=x.device)
    y2 = y.unsqueeze(0) if y.dim() == 1 else y
    if workspace is None:
        workspace = make_workspace(qtype, n_out, k, batch, device=x.device)
    rc = lib().hesa_cuda_qmatvec(qtype, w.data_ptr(), n_out, k, x2.data_ptr(), x2.stride(0), batch,
                                 y2.data_ptr(), y2.stride(0), float(scale), workspace.data_ptr(),
                                 workspace.numel(), _stream_handle(stream))
    _check(rc)
    return y2[0] if squeeze else y2


def dequantize(qtype: int, w, k: int, out=None, stream=None):
    import torch
    n_rows = w.shape[0]
    if out is None:
        out = torch.empty((n_rows, k), dtype=torch.float32, device=w.device)
    _check(lib().hesa_cuda_dequantize(qtype, w.data_ptr(), n_rows, k, out.data_ptr(), out.stride(0),
                                      _stream_handle(stream)))
    return out


def quantize(qtype: int, x, out=None, stream=None):
    """Packed GGUF rows [n_rows, row_bytes] (uint8, CUDA) of fp32 x [n_rows, k]
    (CUDA), deterministic round-to-nearest (hesa_cuda_quantize)."""
    import torch
    x2 = x.unsqueeze(0) if x.dim() == 1 else x
    n_rows, k = x2.shape
    if x2.stride(1) != 1:
        raise ValueError("rows of x must be contiguous")
    rb = row_bytes(qtype, k)
    if rb == 0:
        raise HesaError(6, f"k={k} is not a multiple of the block size of qtype {qtype}")
    if out is None:
        out = torch.empty((n_rows, rb), dtype=torch.uint8, device=x.device)
    _check(lib().hesa_cuda_quantize(qtype, x2.data_ptr(), n_rows, k, x2.stride(0), out.data_ptr(),
                                    _stream_handle(stream)))
    return out


# ---- row-sharded matvec with the all-gather fused in (hesa_cuda_qmatvec_gather) ----

def peer_alloc(nbytes: int) -> tuple[int, bytes]:
    """A zero-filled device allocation shared with the other ranks of the node:
    (device pointer, 64-byte CUDA IPC handle)."""
    ptr = ctypes.c_void_p()
    handle = ctypes.create_string_buffer(64)
    _check(lib().hesa_cuda_peer_alloc(nbytes, ctypes.byref(ptr), handle))
    return ptr.value, handle.raw


def peer_free(ptr: int) -> None:
    _check(lib().hesa_cuda_peer_free(ptr))


def peer_open(handle: bytes) -> int:
    """Map another rank's peer_alloc allocation into this process."""
    ptr = ctypes.c_void_p()
    buf = ctypes.create_string_buffer(bytes(handle), 64)
    _check(lib().hesa_cuda_peer_open(buf, ctypes.byref(ptr)))
    return ptr.value


def peer_close(ptr: int) -> None:
    _check(lib().hesa_cuda_peer_close(ptr))


def qmatvec_gather(qtype: int, w, x, y_peers, world: int, epoch: int, scale: float = 1.0, stream=None):
    """This rank's rows of y = scale * W x (w: its packed rows [n_rows, row_bytes],
    x [k]) stored into every rank's gathered buffer: y_peers lists 2 * world
    device addresses (parity-major) of this shard's first row in each rank's
    buffer; epoch is the device address of this rank's barrier count."""
    n_rows, k = w.shape[0], x.shape[-1]
    arr = (ctypes.c_void_p * (2 * world))(*y_peers)
    _check(lib().hesa_cuda_qmatvec_gather(qtype, w.data_ptr(), n_rows, k, x.data_ptr(), float(scale), arr, world,
                                          epoch, _stream_handle(stream)))


def gather_tagged_workspace(qtype: int, n_rows: int, k: int, device=None):
    """The workspace qmatvec_gather_tagged needs for this shape (None when the
    row-strip kernel takes it and none is needed)."""
    import torch
    nbytes = lib().hesa_cuda_gather_tagged_workspace_size(qtype, n_rows, k)
    return torch.zeros(nbytes, dtype=torch.uint8, device=device or "cuda") if nbytes else None


def qmatvec_gather_tagged(qtype: int, w, x, y_peers, row0: int, world: int, sync: int, scale: float = 1.0,
                          workspace=None, stream=None):
    """As qmatvec_gather, every row stored as a tagged 64-bit word: row i is
    element row0 + i of the gathered vector; y_peers lists 2 * world device
    addresses (parity-major) of word 0 of each rank's gathered buffers; sync
    is the device address of this rank's [step count, ticket] pair. The step
    ends with peer_collect. Rows longer than the strip kernel takes need
    `workspace` (gather_tagged_workspace)."""
    n_rows, k = w.shape[0], x.shape[-1]
    if workspace is None and lib().hesa_cuda_gather_tagged_workspace_size(qtype, n_rows, k):
        workspace = gather_tagged_workspace(qtype, n_rows, k, device=x.device)
    arr = (ctypes.c_void_p * (2 * world))(*y_peers)
    _check(lib().hesa_cuda_qmatvec_gather_tagged(qtype, w.data_ptr(), n_rows, k, x.data_ptr(), float(scale), arr,
                                                 row0, world, sync,
                                                 workspace.data_ptr() if workspace is not None else None,
                                                 workspace.numel() if workspace is not None else 0,
                                                 _stream_handle(stream)))


def peer_collect(words: int, n: int, parity_stride: int, out, sync: int, stream=None) -> None:
    """Wait for this step's n tagged elements in this rank's buffer (device
    address of word 0 `words`, parity 1 `parity_stride` words further, a
    multiple of 256), unpack them into out (fp32 device tensor of n values)
    and advance the step count."""
    import torch
    if out.numel() < n or out.dtype != torch.float32:
        raise ValueError("out must hold n fp32 values")
    _check(lib().hesa_cuda_peer_collect(words, n, parity_stride, out.data_ptr(), sync, _stream_handle(stream)))


def peer_barrier(flags, rank: int, world: int, epoch: int, stream=None) -> None:
    arr = (ctypes.c_void_p * world)(*flags)
    _check(lib().hesa_cuda_peer_barrier(arr, rank, world, epoch, _stream_handle(stream)))


def set_peer_wait_limit(seconds: float) -> None:
    """How long each peer barrier waits for the other ranks before it gives up
    and records device status 4 (0 restores the default, 2 s)."""
    _check(lib().hesa_cuda_set_peer_wait_limit_us(int(round(seconds * 1e6))))


def device_view(ptr: int, numel: int, device=None, dtype: str = "<f4"):
    """A torch tensor over raw device memory (no copy), through the CUDA array
    interface."""
    import torch

    class _View:
        __cuda_array_interface__ = {"shape": (numel,), "typestr": dtype, "data": (ptr, False), "version": 3,
                                    "strides": None}
    return torch.as_tensor(_View(), device=device or "cuda")


def device_status(stream=None) -> int:
    v = ctypes.c_int(0)
    _check(lib().hesa_cuda_device_status(_stream_handle(stream), ctypes.byref(v)))
    return v.value


def clear_device_status(stream=None) -> None:
    _check(lib().hesa_cuda_clear_device_status(_stream_handle(stream)))


def loaded_library_files() -> list[str]:
    """Shared objects of this package mapped into the current process."""
    out = []
    try:
        with open("/proc/self/maps") as f:
            for line in f:
                p = line.split()[-1]
                if p.endswith(".so") and os.path.dirname(p) == os.path.dirname(library_path()):
                    out.append(p)
    except OSError:
        pass
    return sorted(set(out))


# --------------------------------------------------------------------------
# decode-step helpers (device tensors in, device tensors out)
# --------------------------------------------------------------------------

def _ptr(t):
    return None if t is None else t.data_ptr()


def matmul_f32(a, x, y=None, scale: float = 1.0, stream=None):
    import torch
    x2 = x.unsqueeze(0) if x.dim() == 1 else x
    batch, k = x2.shape
    n_out = a.shape[0]
    if y is None:
        y = torch.empty((batch, n_out), dtype=torch.float32, device=x.device)
    y2 = y.unsqueeze(0) if y.dim() == 1 else y
    _check(lib().hesa_cuda_matmul_f32(a.data_ptr(), n_out, k, x2.data_ptr(), x2.stride(0), batch, y2.data_ptr(),
                                      y2.stride(0), float(scale), _stream_handle(stream)))
    return y2[0] if x.dim() == 1 else y2


def rms_norm(x, w, eps: float = 1e-6, out=None, stream=None):
    import torch
    out = torch.empty_like(x) if out is None else out
    n = x.shape[-1]
    _check(lib().hesa_cuda_rms_norm(x.data_ptr(), w.data_ptr(), out.data_ptr(), x.numel() // n, n, float(eps),
                                    _stream_handle(stream)))
    return out


def silu_mul(g, u=None, out=None, stream=None):
    import torch
    out = torch.empty_like(g) if out is None else out
    _check(lib().hesa_cuda_silu_mul(g.data_ptr(), _ptr(u), out.data_ptr(), g.numel(), _stream_handle(stream)))
    return out


def add(a, b, out=None, stream=None):
    import torch
    out = torch.empty_like(a) if out is None else out
    _check(lib().hesa_cuda_add(a.data_ptr(), b.data_ptr(), out.data_ptr(), a.numel(), _stream_handle(stream)))
    return out


def mul(a, b, out=None, stream=None):
    import torch
    out = torch.empty_like(a) if out is None else out
    _check(lib().hesa_cuda_mul(a.data_ptr(), b.data_ptr(), out.data_ptr(), a.numel(), _stream_handle(stream)))
    return out


def softmax(x, out=None, stream=None):
    import torch
    out = torch.empty_like(x) if out is None else out
    n = x.shape[-1]
    _check(lib().hesa_cuda_softmax(x.data_ptr(), out.data_ptr(), x.numel() // n, n, _stream_handle(stream)))
    return out


def rope_table(n_pos: int, head_dim: int, base: float = 10000.0):
    """Host-computed rotate-half angle table [n_pos, head_dim] (numpy)."""
    import numpy as np
    t = np.empty((n_pos, head_dim), dtype=np.float32)
    _check(lib().hesa_cuda_rope_table(t.ctypes.data, n_pos, head_dim, float(base)))
    return t


def rope(x, n_heads: int, head_dim: int, table, pos=None, pos_dev=None, stream=None):
    _check(lib().hesa_cuda_rope(x.data_ptr(), n_heads, head_dim, table.data_ptr(), table.shape[0],
                                _ptr(pos_dev), int(pos or 0), _stream_handle(stream)))
    return x


def kv_store(k, v, k_cache, v_cache, ctx: int, pos=None, pos_dev=None, stream=None):
    _check(lib().hesa_cuda_kv_store(k.data_ptr(), v.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), k.numel(),
                                    ctx, _ptr(pos_dev), int(pos or 0), _stream_handle(stream)))


def attention_workspace(n_head: int, head_dim: int, ctx: int, device=None):
    import torch
    nb = int(lib().hesa_cuda_attention_workspace_size(n_head, head_dim, ctx))
    return torch.zeros(max(nb, 16), dtype=torch.uint8, device=device or "cuda")


def attention(q, k_cache, v_cache, n_head: int, n_kv_head: int, head_dim: int, ctx: int, pos=None, pos_dev=None,
              workspace=None, out=None, stream=None):
    import torch
    out = torch.empty_like(q) if out is None else out
    if workspace is None:
        workspace = attention_workspace(n_head, head_dim, ctx, device=q.device)
    _check(lib().hesa_cuda_attention(q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), out.data_ptr(), n_head,
                                     n_kv_head, head_dim, ctx, _ptr(pos_dev), int(pos or 0), workspace.data_ptr(),
                                     workspace.numel(), _stream_handle(stream)))
    return out


# ---------------------------------------------------------------------------
# decode step
# ---------------------------------------------------------------------------

def decode_workspace(model: Model, device=None):
    """Zero-filled workspace of hesa_cuda_decode_step (uint8, 256-byte aligned)."""
    import torch
    nb = int(lib().hesa_cuda_decode_workspace_size(ctypes.byref(model)))
    if nb == 0:
        raise HesaError(6, "bad model shape")
    return torch.zeros(nb, dtype=torch.uint8, device=device or "cuda")


def embed(qtype: int, w_emb, d_model: int, token_dev, out=None, stream=None):
    import torch
    out = torch.empty(d_model, dtype=torch.float32, device=w_emb.device) if out is None else out
    _check(lib().hesa_cuda_embed(qtype, w_emb.data_ptr(), w_emb.shape[0], d_model, token_dev.data_ptr(),
                                 out.data_ptr(), _stream_handle(stream)))
    return out


def decode_step(model: Model, layers, out_norm, w_out, rope_table, x_embed, pos_dev, logits, workspace,
                stream=None):
    """One token through the decoder (hesa_cuda_decode_step). `layers` is a
    ctypes array of Layer (see make_layers)."""
    _check(lib().hesa_cuda_decode_step(ctypes.byref(model), layers, out_norm.data_ptr(), w_out.data_ptr(),
                                       rope_table.data_ptr(), rope_table.shape[0], x_embed.data_ptr(),
                                       pos_dev.data_ptr(), logits.data_ptr(), workspace.data_ptr(),
                                       workspace.numel(), _stream_handle(stream)))
    return logits


def decode_step_sharded(model: Model, shard, layers, out_norm, w_out, rope_table, x_embed, pos_dev, logits,
                        workspace, stream=None):
    """This rank's part of one token of a head-sharded decode
    (hesa_cuda_decode_step_sharded); every rank gets all the logits."""
    _check(lib().hesa_cuda_decode_step_sharded(ctypes.byref(model), ctypes.byref(shard), layers, out_norm.data_ptr(),
                                               w_out.data_ptr(), rope_table.data_ptr(), rope_table.shape[0],
                                               x_embed.data_ptr(), pos_dev.data_ptr(), logits.data_ptr(),
                                               workspace.data_ptr(), workspace.numel(), _stream_handle(stream)))


def make_layers(per_layer):
    """ctypes array of Layer from a list of dicts of CUDA tensors with the
    keys of Layer's fields."""
    arr = (Layer * len(per_layer))()
    for i, d in enumerate(per_layer):
        for name, _ in Layer._fields_:
            setattr(arr[i], name, d[name].data_ptr())
    return arr


# --------------------------------------------------------------------------
# paged KV cache and token log probabilities
# --------------------------------------------------------------------------

def _want(t, dtype, what: str, device=None, dims: int | None = None):
    """A CUDA tensor of this type on `device` (None: the current one); ValueError else."""
    import torch
    if device is None:
        device = torch.cuda.current_device()
    if isinstance(t, torch.Tensor) and t.dtype is dtype and t.get_device() == device and (dims is None or t.dim() == dims):
        return
    if not isinstance(t, torch.Tensor) or t.dtype != dtype or not t.is_cuda:
        raise ValueError(f"{what} must be a CUDA tensor of {dtype}")
    if t.get_device() != device:
        raise ValueError(f"{what} is on {t.device}: every tensor must be on the current CUDA device, the cache's")
    if dims is not None and t.dim() != dims:
        raise ValueError(f"{what} must have {dims} dimensions")


def _ints(t, what: str, n: int | None = None, device=None):
    import torch
    _want(t, torch.int32, what, device, 1)
    if t.numel() > 1 and t.stride(0) != 1:
        raise ValueError(f"{what} must be contiguous")
    if n is not None and t.numel() != n:
        raise ValueError(f"{what} must hold {n} values")
    return t.data_ptr()


def _stream_on(device: int, stream):
    """The stream's handle for a call on `device`, which is the current one."""
    if stream is None:
        import torch
        return torch._C._cuda_getCurrentRawStream(device) or None
    return _stream_handle(stream)


def _stream_object(stream):
    """torch's object for a stream that is given as one or as a handle."""
    import torch
    if not isinstance(stream, int):
        return stream
    return torch.cuda.ExternalStream(stream) if stream else torch.cuda.default_stream()


def _new(make, stream):
    """A tensor made for a call on `stream`: allocated and filled there, so that it may be freed in that stream's order."""
    import torch
    if stream is None:
        return make()
    with torch.cuda.stream(_stream_object(stream)):
        return make()


def _page_strides(t) -> tuple:
    """The strides of a pool; of a dimension of one entry, which may have any in torch, what a contiguous one would have."""
    out = []
    for size, stride in zip(reversed(t.shape), reversed(t.stride())):
        out.append(stride if size != 1 else 1 if not out else out[-1] * below)
        below = size
    return tuple(reversed(out))


class PagedKV:
    """A paged fp16 KV cache (hesa_cuda_paged_kv): the page pools k, v
    [n_layer, n_pages, page_size, n_kv_head, head_dim] (any layer and page
    strides, the rest contiguous), the tables table [n_slots, max_pages],
    seq_len [n_slots] and page_refs [n_pages] (int32; page_refs may be None
    without page operations). Keeps the tensors, and scratch of the page
    operations for each stream that they ran on; everything lies on one CUDA
    device."""

    def __init__(self, k, v, table, seq_len, page_refs=None):
        import torch
        _want(k, torch.float16, "k", dims=5)
        dev = k.device.index
        _want(v, torch.float16, "v", dev, 5)
        _want(table, torch.int32, "table", dev, 2)
        n_layer, n_pages, page, n_kv, hd = k.shape
        strides = _page_strides(k)
        if v.shape != k.shape or _page_strides(v) != strides:
            raise ValueError("k and v must have the same shape and strides")
        if strides[2:] != (n_kv * hd, hd, 1):
            raise ValueError("places, heads and dims of a page must be contiguous")
        if not table.is_contiguous():
            raise ValueError("table must be contiguous")
        _ints(seq_len, "seq_len", table.shape[0], dev)
        if page_refs is not None:
            _ints(page_refs, "page_refs", n_pages, dev)
        self.device, self.n_slots, self.n_pages, self.n_kv_head, self.head_dim = dev, table.shape[0], n_pages, n_kv, hd
        self.k, self.v, self.table, self.seq_len, self.page_refs = k, v, table, seq_len, page_refs
        self.struct = PagedKVStruct(k.data_ptr(), v.data_ptr(), strides[1], strides[0], n_layer, n_pages, page, n_kv, hd,
                                    table.data_ptr(), seq_len.data_ptr(), _ptr(page_refs), table.shape[0], table.shape[1])
        self.ref = ctypes.byref(self.struct)
        self.scratch = {}   # of the page operations, by stream handle

    @classmethod
    def empty(cls, n_layer: int, n_pages: int, page_size: int, n_kv_head: int, head_dim: int, n_slots: int, max_pages: int):
        """A new cache on the current device with every page free and every slot empty."""
        import torch
        shape = (n_layer, n_pages, page_size, n_kv_head, head_dim)
        return cls(torch.zeros(shape, dtype=torch.float16, device="cuda"), torch.zeros(shape, dtype=torch.float16, device="cuda"),
                   torch.full((n_slots, max_pages), -1, dtype=torch.int32, device="cuda"),
                   torch.zeros(n_slots, dtype=torch.int32, device="cuda"), torch.zeros(n_pages, dtype=torch.int32, device="cuda"))


class TokenBatch:
    """New tokens of several sequences (hesa_cuda_token_batch): q_start
    [n_seq + 1] and slots [n_seq] (None: sequence i is in slot i), int32 on the
    device; n_tokens rows in all, at most max_new new tokens and max_len tokens
    for any sequence. The tensors may be refilled for every step within these
    bounds."""

    def __init__(self, q_start, n_tokens: int, max_new: int, max_len: int, slots=None):
        _ints(q_start, "q_start")
        n_seq = q_start.numel() - 1
        if slots is not None:
            _ints(slots, "slots", n_seq, q_start.device.index)
        self.device, self.n_tokens, self.n_seq = q_start.device.index, n_tokens, n_seq
        self.q_start, self.slots = q_start, slots
        self.struct = TokenBatchStruct(_ptr(slots), q_start.data_ptr(), n_seq, n_tokens, max_new, max_len)
        self.ref = ctypes.byref(self.struct)


def _rows(t, n: int, width: int, what: str, device):
    """Pointer and row stride of fp32 rows [n, width] (a column slice of a wider matrix is one)."""
    import torch
    _want(t, torch.float32, what, device, 2)
    if t.shape[0] != n or t.shape[1] != width or (t.stride(1) != 1 and width > 1):
        raise ValueError(f"{what} must be [{n}, {width}] with contiguous rows")
    return t.data_ptr(), (t.stride(0) if n > 1 else width + (-width) % 4)


def _same_device(cache, batch=None):
    import torch
    if torch.cuda.current_device() != cache.device or (batch is not None and batch.device != cache.device):
        raise ValueError("the cache and the batch must be on the current CUDA device")


def paged_attention_workspace(cache, batch, n_head: int):
    """A workspace for paged_attention of batches of these bounds."""
    import torch
    _same_device(cache, batch)
    nb = int(lib().hesa_cuda_paged_attention_workspace_size(cache.ref, batch.ref, n_head))
    if nb == 0:
        raise HesaError(6, lib().hesa_cuda_last_error().decode())
    return torch.empty(nb, dtype=torch.uint8, device="cuda")


def paged_attention(cache, layer: int, batch, q, n_head: int, out=None, scale: float | None = None, softcap: float = 0.0,
                    window: int = 0, slopes=None, prefix=None, workspace=None, stream=None):
    """Attention of the batch's new tokens, q [n_tokens, n_head * head_dim] fp32,
    over layer `layer` of the cache (hesa_cuda_paged_attention); returns out."""
    import torch
    _same_device(cache, batch)
    dev, n, width = cache.device, batch.n_tokens, n_head * cache.head_dim
    qp, ldq = _rows(q, n, width, "q", dev)
    if scale is not None and not scale > 0:
        raise ValueError("scale must be positive")
    opts = None
    if scale is not None or softcap or window or slopes is not None or prefix is not None:
        if slopes is not None:
            _want(slopes, torch.float32, "slopes", dev, 1)
            if slopes.numel() != n_head or not slopes.is_contiguous():
                raise ValueError("slopes must hold n_head contiguous values")
        if prefix is not None:
            _ints(prefix, "prefix", batch.n_seq, dev)
        opts = AttnOptionsStruct(scale or 0.0, softcap, window, _ptr(slopes), _ptr(prefix))
    if out is None:
        out = _new(lambda: torch.zeros((n, width), dtype=torch.float32, device="cuda"), stream)
    op, ldo = _rows(out, n, width, "out", dev)
    if workspace is None:
        workspace = _new(lambda: paged_attention_workspace(cache, batch, n_head), stream)
    else:
        _want(workspace, torch.uint8, "workspace", dev)
    _check(lib().hesa_cuda_paged_attention(cache.ref, layer, batch.ref, qp, ldq, op, ldo, n_head,
                                           None if opts is None else ctypes.byref(opts), workspace.data_ptr(),
                                           workspace.numel(), _stream_on(cache.device, stream)))
    return out


def rope_kv_paged(cache, layer: int, batch, q, k, v, n_head: int, rope_table=None, stream=None) -> None:
    """The batch's new k, v [n_tokens, n_kv_head * head_dim] into layer `layer` of
    the cache; with rope_table (a device copy of rope_table()) q is rotated in
    place and k before it is stored (hesa_cuda_rope_kv_paged). q may be None
    without a table."""
    import torch
    _same_device(cache, batch)
    dev, n, width = cache.device, batch.n_tokens, cache.n_kv_head * cache.head_dim
    qp, ldq = (None, 0) if q is None else _rows(q, n, n_head * cache.head_dim, "q", dev)
    kp, ldk = _rows(k, n, width, "k", dev)
    vp, ldv = _rows(v, n, width, "v", dev)
    if rope_table is not None:
        _want(rope_table, torch.float32, "rope_table", dev, 2)
        if rope_table.shape[1] != cache.head_dim or not rope_table.is_contiguous():
            raise ValueError("rope_table must be [rows, head_dim] and contiguous")
    _check(lib().hesa_cuda_rope_kv_paged(cache.ref, layer, batch.ref, qp, ldq, kp, ldk, vp, ldv, n_head, _ptr(rope_table),
                                         0 if rope_table is None else rope_table.shape[0], _stream_on(cache.device, stream)))


def kv_pages_workspace(cache):
    """Scratch for the page operations on this cache."""
    import torch
    _same_device(cache)
    nb = int(lib().hesa_cuda_kv_pages_workspace_size(cache.ref))
    if nb == 0:
        raise HesaError(6, lib().hesa_cuda_last_error().decode() or "page operations take at most 2^20 pages")
    return torch.empty(nb, dtype=torch.uint8, device="cuda")


def _page_workspace(cache, workspace, stream):
    """The workspace of a page operation: the caller's, or scratch that was allocated on the very stream that the call
    runs on (nothing else orders its kernels behind the memory's earlier use there). The cache keeps one for each stream
    that was current at such a call; a given stream's, and a captured call's, lasts for the call alone (in a graph: is
    the graph's own)."""
    import torch
    _same_device(cache)
    if workspace is not None:
        _want(workspace, torch.uint8, "workspace", cache.device)
        return workspace
    if stream is not None or torch.cuda.is_current_stream_capturing():
        return _new(lambda: kv_pages_workspace(cache), stream)
    handle = torch._C._cuda_getCurrentRawStream(cache.device)
    workspace = cache.scratch.get(handle)
    if workspace is None:
        workspace = cache.scratch[handle] = kv_pages_workspace(cache)
    return workspace


def kv_reserve(cache, slots, n_new, workspace=None, stream=None) -> None:
    """n_new[i] more tokens, and the pages for them, for slot slots[i] (hesa_cuda_kv_reserve)."""
    ws = _page_workspace(cache, workspace, stream)
    n = slots.numel()
    _check(lib().hesa_cuda_kv_reserve(cache.ref, _ints(slots, "slots", n, cache.device), _ints(n_new, "n_new", n, cache.device), n,
                                      ws.data_ptr(), ws.numel(), _stream_on(cache.device, stream)))


def kv_free(cache, slots, workspace=None, stream=None) -> None:
    """Give back the pages of these slots and empty them (hesa_cuda_kv_free)."""
    ws = _page_workspace(cache, workspace, stream)
    n = slots.numel()
    _check(lib().hesa_cuda_kv_free(cache.ref, _ints(slots, "slots", n, cache.device), n, ws.data_ptr(), ws.numel(),
                                   _stream_on(cache.device, stream)))


def kv_fork(cache, src, dst, workspace=None, stream=None) -> None:
    """The empty slots dst become copies of the slots src, sharing full pages (hesa_cuda_kv_fork)."""
    ws = _page_workspace(cache, workspace, stream)
    n = src.numel()
    _check(lib().hesa_cuda_kv_fork(cache.ref, _ints(src, "src", n, cache.device), _ints(dst, "dst", n, cache.device), n,
                                   ws.data_ptr(), ws.numel(), _stream_on(cache.device, stream)))


def kv_compact(cache, n_live=None, workspace=None, stream=None) -> None:
    """Move the pages in use to the front of the pool (hesa_cuda_kv_compact); n_live: int32 [1] for their count."""
    ws = _page_workspace(cache, workspace, stream)
    p = None if n_live is None else _ints(n_live, "n_live", 1, cache.device)
    _check(lib().hesa_cuda_kv_compact(cache.ref, p, ws.data_ptr(), ws.numel(), _stream_on(cache.device, stream)))


def kv_copy_pages(cache, src_pages, dst_pages, workspace=None, stream=None) -> None:
    """Page dst_pages[i] becomes a copy of page src_pages[i] in every layer (hesa_cuda_kv_copy_pages)."""
    ws = _page_workspace(cache, workspace, stream)
    n = src_pages.numel()
    _check(lib().hesa_cuda_kv_copy_pages(cache.ref, _ints(src_pages, "src_pages", n, cache.device),
                                         _ints(dst_pages, "dst_pages", n, cache.device), n, ws.data_ptr(), ws.numel(),
                                         _stream_on(cache.device, stream)))


def token_logprobs_workspace(n_rows: int, vocab: int, top_k: int = 0):
    """A zero-filled workspace for token_logprobs."""
    import torch
    nb = int(lib().hesa_cuda_token_logprobs_workspace_size(n_rows, vocab, top_k))
    return torch.zeros(max(nb, 16), dtype=torch.uint8, device="cuda")


def token_logprobs(logits, tokens=None, top_k: int = 0, workspace=None, stream=None):
    """From logits [n_rows, vocab] fp32 (any row stride): the log probability of
    each row's token (tokens [n_rows] int32; None: none), the row's entropy, and
    the top_k most probable ids with their log probabilities
    (hesa_cuda_token_logprobs). Returns (logprob or None, entropy, top_ids,
    top_logprobs), the last two [n_rows, top_k]."""
    import torch
    _want(logits, torch.float32, "logits", dims=2)
    n, vocab = logits.shape
    if vocab > 1 and logits.stride(1) != 1:
        raise ValueError("rows of logits must be contiguous")
    dev = logits.device.index
    tp = None if tokens is None else _ints(tokens, "tokens", n, dev)

    where = logits.device

    def outputs():
        return (None if tokens is None else torch.empty(n, dtype=torch.float32, device=where), torch.empty(n, dtype=torch.float32, device=where),
                torch.empty((n, top_k), dtype=torch.int32, device=where), torch.empty((n, top_k), dtype=torch.float32, device=where))
    logprob, entropy, ids, top = outputs() if stream is None else _new(outputs, stream)
    if workspace is None:
        workspace = _new(lambda: token_logprobs_workspace(n, vocab, top_k), stream)
    else:
        _want(workspace, torch.uint8, "workspace", dev)
    _check(lib().hesa_cuda_token_logprobs(logits.data_ptr(), logits.stride(0) if n > 1 else vocab, n, vocab, tp, top_k,
                                          None if tokens is None else logprob.data_ptr(), entropy.data_ptr(),
                                          ids.data_ptr() if top_k else None, top.data_ptr() if top_k else None,
                                          workspace.data_ptr(), workspace.numel(), _stream_on(dev, stream)))
    return logprob, entropy, ids, top
