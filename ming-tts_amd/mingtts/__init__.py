"""Python binding of libmingtts_hip.so (the gfx950 linear hot path of MingTTS).

The library is the product; this module only loads it with ctypes and forwards
device pointers.  It raises if the library is missing: there is no CPU fallback.

The classes ``Linear``, ``ActView``, ``GemvFlags`` and ``Encoder`` mirror the
reference's operator layer (Sources/MingTTS/Engine/Kernels.swift:7-44, 128-206) so
callers and tests read like the reference's own: ``Encoder.linear(x, rows, linear, y,
flags, gate)`` forwards to ``mt_linear`` with the same argument meaning.  Tensors are
torch device tensors (plumbing for memory and streams only).
"""
from __future__ import annotations

import ctypes
import functools
import os
from dataclasses import dataclass
from typing import Optional, Sequence

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.normpath(os.path.join(_HERE, "..", "csrc", "libmingtts_hip.so"))

F32, F16, BF16, F8 = 0, 1, 2, 3
OK, EHIP, ENOMEM, EINVAL, ERANGE, ENOTSUP = 0, -5, -12, -22, -34, -95
KERNEL_GEMV, KERNEL_GEMM, KERNEL_GEMV_MFMA = 1, 2, 3
(TUNE_GEMV_ROWS_MAX, TUNE_GEMV_LANES, TUNE_GEMM_SPLITK, TUNE_SEQ_GROUPS, TUNE_SEQ_LAUNCH, TUNE_GEMM_TILE,
 TUNE_GEMM_STAGES, TUNE_GEMV_MFMA, TUNE_SEQ_LAYER, TUNE_F8_TILE) = 1, 2, 3, 4, 5, 6, 7, 8, 9, 10
SEQ_GENERAL, SEQ_DECODE_LAYER, SEQ_DIT_BLOCK = 0, 1, 2

# Every symbol include/mingtts_hip.h declares.
EXPORTS = (
    "mt_linear", "mt_linear_static", "mt_linear_rmsnorm", "mt_rmsnorm", "mt_linear_kernel", "mt_set_tuning", "mt_seq_create",
    "mt_seq_create_items", "mt_seq_run",
    "mt_seq_destroy", "mt_seq_groups", "mt_seq_kernel", "mt_seq_check", "mt_rope_cache", "mt_rope_cache_decode",
    "mt_attention", "mt_attention_decode", "mt_rope_attention", "mt_dit_attention", "mt_dit_attention_linear", "mt_flow_assemble",
    "mt_flow_euler", "mt_flow_euler_assemble", "mt_rope_append", "mt_kv_copy", "mt_attention_shared",
    "mt_attention_shared_workspace", "mt_quantize_f8", "mt_linear_f8",
    "mt_upsample4", "mt_istft_frames", "mt_istft_emit", "mt_st_open", "mt_st_close", "mt_st_count", "mt_st_name", "mt_st_find", "mt_arena_create", "mt_arena_tensor",
    "mt_arena_padded", "mt_arena_bytes", "mt_arena_upload", "mt_arena_audit", "mt_arena_destroy",
    "mt_last_error", "mt_version",
)


class GemvFlags:
    """GemvFlags, Kernels.swift:21-28."""
    bias = 1
    accumulate = 2
    gelu = 4
    siluGate = 8
    silu = 16


class MingTTSError(RuntimeError):
    """An error code returned by the library, with mt_last_error()'s text."""

    def __init__(self, code: int, msg: str):
        super().__init__(f"[{code}] {msg}")
        self.code = code


class GemvParams(ctypes.Structure):
    """mt_gemv_params == GemvParams (Shaders.swift:39)."""
    _fields_ = [("M", ctypes.c_uint32), ("N", ctypes.c_uint32), ("K", ctypes.c_uint32),
                ("ldx", ctypes.c_uint32), ("ldy", ctypes.c_uint32), ("flags", ctypes.c_uint32),
                ("eps", ctypes.c_float)]


class LinearOp(ctypes.Structure):
    """mt_linear_op: one op of a persistent sequence."""
    _fields_ = [("x", ctypes.c_void_p), ("w", ctypes.c_void_p), ("w2", ctypes.c_void_p),
                ("bias", ctypes.c_void_p), ("norm", ctypes.c_void_p), ("y", ctypes.c_void_p),
                ("p", GemvParams), ("xt", ctypes.c_int32), ("wt", ctypes.c_int32)]


class AttnOp(ctypes.Structure):
    """mt_attn_op: the decode attention of one layer as an item of a sequence."""
    _fields_ = [("qkv", ctypes.c_void_p), ("ldq", ctypes.c_uint32), ("B", ctypes.c_uint32),
                ("hq", ctypes.c_uint32), ("hkv", ctypes.c_uint32), ("pos", ctypes.c_void_p),
                ("k_cache", ctypes.c_void_p), ("v_cache", ctypes.c_void_p), ("cache_t", ctypes.c_int32),
                ("cache_len", ctypes.c_uint32), ("cache_stride", ctypes.c_uint64), ("inv_freq", ctypes.c_void_p),
                ("out", ctypes.c_void_p), ("ldo", ctypes.c_uint32), ("window", ctypes.c_uint32),
                ("scale", ctypes.c_float)]


class DitAttnOp(ctypes.Structure):
    """mt_dit_attn_op: the DiT's full attention (mt_dit_attention) as an item of a sequence."""
    _fields_ = [("qkv", ctypes.c_void_p), ("ldq", ctypes.c_uint32), ("B", ctypes.c_uint32), ("S", ctypes.c_uint32),
                ("H", ctypes.c_uint32), ("inv_freq", ctypes.c_void_p), ("out", ctypes.c_void_p),
                ("ldo", ctypes.c_uint32), ("scale", ctypes.c_float)]


SEQ_LINEAR, SEQ_ATTENTION, SEQ_DIT_ATTENTION = 0, 1, 2


class SeqItem(ctypes.Structure):
    """mt_seq_item: a linear, a decode attention or a DiT attention item of a sequence."""
    _fields_ = [("kind", ctypes.c_int32), ("linear", LinearOp), ("attn", AttnOp), ("dit", DitAttnOp)]


class KvStruct(ctypes.Structure):
    """mt_kv: the caches of one layer for a batch of sequences."""
    _fields_ = [("k", ctypes.c_void_p), ("v", ctypes.c_void_p), ("k_scale", ctypes.c_void_p),
                ("v_scale", ctypes.c_void_p), ("stride", ctypes.c_uint64), ("scale_stride", ctypes.c_uint64),
                ("cache_len", ctypes.c_uint32), ("cache_t", ctypes.c_int32)]


class StEntry(ctypes.Structure):
    """mt_st_entry: one tensor of a .safetensors file."""
    _fields_ = [("dtype", ctypes.c_int32), ("ndim", ctypes.c_uint32), ("shape", ctypes.c_uint64 * 8),
                ("bytes", ctypes.c_uint64), ("host", ctypes.c_void_p)]


_lib: Optional[ctypes.CDLL] = None


def load(path: str = LIB_PATH) -> ctypes.CDLL:
    """Loads libmingtts_hip.so (raises if it is not built)."""
    global _lib
    if _lib is not None:
        return _lib
    if not os.path.exists(path):
        raise RuntimeError(f"libmingtts_hip.so is not built at {path}; run __graft_entry__.build()")
    L = ctypes.CDLL(path)
    vp, u32, u64, i32, f32 = ctypes.c_void_p, ctypes.c_uint32, ctypes.c_uint64, ctypes.c_int, ctypes.c_float
    L.mt_linear.argtypes = [vp, i32, vp, vp, i32, vp, vp, GemvParams, vp]
    L.mt_linear.restype = i32
    L.mt_linear_static.argtypes = [vp, i32, vp, vp, i32, vp, vp, GemvParams, vp]
    L.mt_linear_static.restype = i32
    L.mt_linear_rmsnorm.argtypes = [vp, i32, vp, vp, vp, i32, vp, vp, GemvParams, vp]
    L.mt_linear_rmsnorm.restype = i32
    L.mt_rmsnorm.argtypes = [vp, u32, u32, u32, vp, i32, vp, u32, f32, vp]
    L.mt_rmsnorm.restype = i32
    L.mt_linear_kernel.argtypes = [u32, u32, u32, i32, i32]
    L.mt_linear_kernel.restype = i32
    L.mt_set_tuning.argtypes = [i32, i32]
    L.mt_set_tuning.restype = i32
    L.mt_seq_create.argtypes = [ctypes.POINTER(LinearOp), u32, ctypes.POINTER(vp)]
    L.mt_seq_create.restype = i32
    L.mt_seq_create_items.argtypes = [ctypes.POINTER(SeqItem), u32, ctypes.POINTER(vp)]
    L.mt_seq_create_items.restype = i32
    L.mt_seq_run.argtypes = [vp, vp]
    L.mt_seq_run.restype = i32
    L.mt_seq_destroy.argtypes = [vp]
    L.mt_seq_destroy.restype = i32
    L.mt_seq_groups.argtypes = [vp]
    L.mt_seq_groups.restype = i32
    L.mt_seq_kernel.argtypes = [vp]
    L.mt_seq_kernel.restype = i32
    L.mt_seq_check.argtypes = [vp]
    L.mt_seq_check.restype = i32
    L.mt_rope_cache.argtypes = [vp, u32, u32, u32, u32, u32, vp, vp, i32, u32, vp, vp]
    L.mt_rope_cache.restype = i32
    L.mt_rope_cache_decode.argtypes = [vp, u32, u32, u32, u32, vp, vp, vp, i32, u32, u64, vp, vp]
    L.mt_rope_cache_decode.restype = i32
    L.mt_attention.argtypes = [vp, u32, u32, u32, u32, u32, u32, vp, vp, i32, u32, vp, u32, f32, vp]
    L.mt_rope_attention.argtypes = [vp, u32, u32, u32, u32, u32, u32, vp, vp, i32, u32, vp, vp, u32, f32, vp]
    L.mt_rope_attention.restype = i32
    L.mt_attention.restype = i32
    L.mt_attention_decode.argtypes = [vp, u32, u32, u32, u32, vp, u32, vp, vp, i32, u32, u64, vp, u32, f32, vp]
    L.mt_attention_decode.restype = i32
    L.mt_dit_attention.argtypes = [vp, u32, u32, u32, u32, vp, vp, u32, f32, vp]
    L.mt_dit_attention.restype = i32
    L.mt_dit_attention_linear.argtypes = [vp, u32, u32, u32, vp, f32, vp, i32, vp, vp, GemvParams, vp]
    L.mt_dit_attention_linear.restype = i32
    L.mt_flow_assemble.argtypes = [vp, vp, vp, vp, vp, vp, vp, i32, vp, u32, u32, u32, vp]
    L.mt_flow_assemble.restype = i32
    L.mt_flow_euler.argtypes = [vp, vp, u32, u32, u32, vp, u32, f32, f32, vp]
    L.mt_flow_euler.restype = i32
    L.mt_flow_euler_assemble.argtypes = [vp, vp, u32, u32, u32, vp, f32, f32, vp, vp, vp, vp, vp, vp, i32, vp, u32, u32,
                                         u32, vp]
    L.mt_flow_euler_assemble.restype = i32
    L.mt_upsample4.argtypes = [vp, vp, vp, vp, u32, u32, vp]
    L.mt_upsample4.restype = i32
    L.mt_istft_frames.argtypes = [vp, u32, u32, u32, vp, vp, vp, u32, u32, vp]
    L.mt_istft_frames.restype = i32
    L.mt_istft_emit.argtypes = [vp, vp, u32, u32, u32, u32, u32, u32, vp, vp]
    L.mt_istft_emit.restype = i32
    kv = ctypes.POINTER(KvStruct)
    L.mt_rope_append.argtypes = [vp, u32, u32, u32, u32, u32, vp, vp, u32, kv, vp, vp, u32, vp]
    L.mt_rope_append.restype = i32
    L.mt_kv_copy.argtypes = [kv, kv, u32, u32, u32, vp, vp, vp]
    L.mt_kv_copy.restype = i32
    L.mt_attention_shared_workspace.argtypes = [u32, u32, u32, u32, u32, u32, u32, i32]
    L.mt_attention_shared_workspace.restype = u64
    L.mt_attention_shared.argtypes = [vp, u32, u32, u32, u32, u32, vp, vp, kv, kv, u32, u32, u32, vp, u32, f32, vp, u64, vp]
    L.mt_attention_shared.restype = i32
    L.mt_quantize_f8.argtypes = [vp, i32, u32, u32, u32, vp, i32, f32, vp, u32, vp, u32, vp]
    L.mt_quantize_f8.restype = i32
    L.mt_linear_f8.argtypes = [vp, i32, vp, u32, vp, vp, vp, vp, vp, vp, i32, vp, GemvParams, vp]
    L.mt_linear_f8.restype = i32
    cp = ctypes.c_char_p
    L.mt_st_open.argtypes = [cp, ctypes.POINTER(vp)]
    L.mt_st_open.restype = i32
    L.mt_st_close.argtypes = [vp]
    L.mt_st_close.restype = i32
    L.mt_st_count.argtypes = [vp]
    L.mt_st_count.restype = i32
    L.mt_st_name.argtypes = [vp, u32, ctypes.POINTER(cp)]
    L.mt_st_name.restype = i32
    L.mt_st_find.argtypes = [vp, cp, ctypes.POINTER(StEntry)]
    L.mt_st_find.restype = i32
    L.mt_arena_create.argtypes = [vp, i32, ctypes.POINTER(vp)]
    L.mt_arena_create.restype = i32
    L.mt_arena_tensor.argtypes = [vp, ctypes.POINTER(cp), u32, ctypes.POINTER(u64), ctypes.POINTER(u64)]
    L.mt_arena_tensor.restype = i32
    L.mt_arena_padded.argtypes = [vp, cp, u32, u32, u32, ctypes.POINTER(u64)]
    L.mt_arena_padded.restype = i32
    L.mt_arena_bytes.argtypes = [vp]
    L.mt_arena_bytes.restype = u64
    L.mt_arena_upload.argtypes = [vp, vp, vp]
    L.mt_arena_upload.restype = i32
    L.mt_arena_audit.argtypes = [vp, ctypes.POINTER(u64), ctypes.POINTER(u64)]
    L.mt_arena_audit.restype = i32
    L.mt_arena_destroy.argtypes = [vp]
    L.mt_arena_destroy.restype = i32
    L.mt_last_error.argtypes = []
    L.mt_last_error.restype = ctypes.c_char_p
    L.mt_version.argtypes = []
    L.mt_version.restype = ctypes.c_char_p
    _lib = L
    return L


def last_error() -> str:
    return load().mt_last_error().decode()


def check(rc: int) -> int:
    if rc < 0:
        raise MingTTSError(rc, last_error())
    return rc


def _ptr(t) -> Optional[int]:
    if t is None or t.__class__ is int:
        return t
    if isinstance(t, int):
        return t
    return t.data_ptr()


# A call's own Python is what bounds the smallest calls (one decode linear: 8.9 us of host work
# against 3.6 us on the GPU), so the helpers below keep the torch names they need instead of
# importing them in each call, and take the current stream's handle without a Stream object.
_dtypes: dict = {}
_current_device = None  # torch's current-device and raw-stream functions, once torch has initialised the GPU
_raw_stream = None


def _stream(stream) -> Optional[int]:
    if stream is None:
        if _raw_stream is not None:
            return _raw_stream(_current_device())
        return _first_stream()
    if isinstance(stream, int):
        return stream
    return stream.cuda_stream


def _first_stream() -> int:
    """torch.cuda.current_stream() initialises the GPU where nothing has; later calls ask torch for the
    handle directly where this torch has the functions."""
    global _current_device, _raw_stream
    import torch
    handle = torch.cuda.current_stream().cuda_stream
    device, raw = getattr(torch._C, "_cuda_getDevice", None), getattr(torch._C, "_cuda_getCurrentRawStream", None)
    if device is not None and raw is not None and raw(device()) == handle:
        _current_device, _raw_stream = device, raw
    return handle


def dtype_code(t) -> int:
    if not _dtypes:
        import torch
        _dtypes.update({torch.float32: F32, torch.float16: F16, torch.bfloat16: BF16})
    return _dtypes[t.dtype]


# ------------------------------------------------------------ raw calls --

def linear_raw(x, xt, w, w2, wt, bias, y, M, N, K, ldx, ldy, flags, stream=None) -> int:
    """mt_linear on raw pointers / tensors; returns the raw return code."""
    p = GemvParams(M, N, K, ldx, ldy, flags, 0.0)
    return load().mt_linear(_ptr(x), xt, _ptr(w), _ptr(w2), wt, _ptr(bias), _ptr(y), p, _stream(stream))


def linear_static_raw(x, xt, w, w2, wt, bias, y, M, N, K, ldx, ldy, flags, stream=None) -> int:
    """mt_linear_static on raw pointers / tensors; returns the raw return code."""
    p = GemvParams(M, N, K, ldx, ldy, flags, 0.0)
    return load().mt_linear_static(_ptr(x), xt, _ptr(w), _ptr(w2), wt, _ptr(bias), _ptr(y), p, _stream(stream))


def linear_rmsnorm_raw(x, xt, norm, w, w2, wt, bias, y, M, N, K, ldx, ldy, flags, eps=1e-6, stream=None) -> int:
    """mt_linear_rmsnorm on raw pointers / tensors; returns the raw return code."""
    p = GemvParams(M, N, K, ldx, ldy, flags, eps)
    return load().mt_linear_rmsnorm(_ptr(x), xt, _ptr(norm), _ptr(w), _ptr(w2), wt, _ptr(bias), _ptr(y), p,
                                    _stream(stream))


def linear(x, w, y, M=None, flags=0, w2=None, bias=None, ldx=None, ldy=None, norm=None, eps=1e-6,
           stream=None) -> None:
    """y[:M] (op)= x[:M] @ w.T with the epilogue in ``flags``; torch tensors, w: [N, K].
    With ``norm`` (gain [K]) x is RMS-normalised first (mt_linear_rmsnorm)."""
    N, K = w.shape
    if M is None:
        M = x.shape[0]
    if ldx is None:
        ldx = x.stride(0)
    if ldy is None:
        ldy = y.stride(0)
    if norm is not None:
        check(linear_rmsnorm_raw(x, dtype_code(x), norm, w, w2, dtype_code(w), bias, y, M, N, K, ldx, ldy, flags,
                                 eps, stream))
    else:
        check(linear_raw(x, dtype_code(x), w, w2, dtype_code(w), bias, y, M, N, K, ldx, ldy, flags, stream))


def rmsnorm_raw(x, ldx, rows, width, g, wt, y, ldy, eps=1e-6, stream=None) -> int:
    """mt_rmsnorm on raw pointers / tensors; returns the raw return code."""
    return load().mt_rmsnorm(_ptr(x), ldx, rows, width, _ptr(g), wt, _ptr(y), ldy, eps, _stream(stream))


def rmsnorm(x, g, y, rows=None, eps=1e-6, stream=None) -> None:
    """y[:rows] = x[:rows] * rsqrt(mean(x^2) + eps) * g (mt_rmsnorm); torch tensors, g [width]."""
    rows = x.shape[0] if rows is None else rows
    check(rmsnorm_raw(x, x.stride(0), rows, g.shape[0], g, dtype_code(g), y, y.stride(0), eps, stream))


def linear_kernel(M, N, K, xt=F32, wt=BF16) -> int:
    return load().mt_linear_kernel(M, N, K, xt, wt)


def set_tuning(key: int, value: int) -> int:
    return check(load().mt_set_tuning(key, value))


class Seq:
    """A persistent sequence plan (mt_seq_*) of linears (``LinearOp``) and, optionally,
    decode attention items (``AttnOp``) or DiT attention items (``DitAttnOp``)."""

    def __init__(self, ops: Sequence):
        h = ctypes.c_void_p()
        if all(isinstance(o, LinearOp) for o in ops):
            arr = (LinearOp * len(ops))(*ops)
            check(load().mt_seq_create(arr, len(ops), ctypes.byref(h)))
        else:
            items = (SeqItem * len(ops))()
            for i, o in enumerate(ops):
                if isinstance(o, AttnOp):
                    items[i].kind = SEQ_ATTENTION
                    items[i].attn = o
                elif isinstance(o, DitAttnOp):
                    items[i].kind = SEQ_DIT_ATTENTION
                    items[i].dit = o
                else:
                    items[i].kind = SEQ_LINEAR
                    items[i].linear = o
            check(load().mt_seq_create_items(items, len(ops), ctypes.byref(h)))
        self.handle = h
        self.n_ops = len(ops)

    def run(self, stream=None) -> None:
        check(load().mt_seq_run(self.handle, _stream(stream)))

    def check(self) -> None:
        check(load().mt_seq_check(self.handle))

    @property
    def groups(self) -> int:
        return check(load().mt_seq_groups(self.handle))

    @property
    def kernel(self) -> int:
        """SEQ_DECODE_LAYER when the plan runs the kernel specialised for Qwen2-0.5B decode
        layers, SEQ_DIT_BLOCK for the flow head's DiT blocks, else SEQ_GENERAL."""
        return check(load().mt_seq_kernel(self.handle))

    def close(self) -> None:
        if self.handle:
            load().mt_seq_destroy(self.handle)
            self.handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


def op(x, w, y, M, flags=0, w2=None, bias=None, ldx=None, ldy=None, xt=None, wt=None, norm=None,
       eps=1e-6) -> LinearOp:
    """An mt_linear_op over torch tensors (w: [N, K]); ``norm`` fuses an RMSNorm prologue."""
    N, K = w.shape
    if bias is not None:
        flags |= GemvFlags.bias
    return LinearOp(_ptr(x), _ptr(w), _ptr(w2), _ptr(bias), _ptr(norm), _ptr(y),
                    GemvParams(M, N, K, x.stride(0) if ldx is None else ldx, y.stride(0) if ldy is None else ldy,
                               flags, eps if norm is not None else 0.0),
                    dtype_code(x) if xt is None else xt, dtype_code(w) if wt is None else wt)


def dit_attn_op(qkv, B, S, H, inv_freq, out, ldq=None, ldo=None, scale=0.125) -> DitAttnOp:
    """An mt_dit_attn_op over torch tensors: B sequences of S rows of qkv ([B S, 3 H 64] at
    stride ldq), out [B S, H 64]."""
    return DitAttnOp(_ptr(qkv), qkv.stride(0) if ldq is None else ldq, B, S, H, _ptr(inv_freq), _ptr(out),
                     out.stride(0) if ldo is None else ldo, scale)


def attn_op(qkv, B, hq, hkv, pos, kc, vc, cache_len, cache_stride, inv_freq, out, ldq=None, ldo=None,
            window=0, scale=0.125) -> AttnOp:
    """An mt_attn_op over torch tensors: rows b < B of qkv ([B, (hq + 2 hkv) 64] at stride
    ldq), positions pos (device uint32/int32 [B]), caches kc / vc ([B, hkv, cache_len, 64]
    at cache_stride elements per row), out [B, hq 64]."""
    return AttnOp(_ptr(qkv), qkv.stride(0) if ldq is None else ldq, B, hq, hkv, _ptr(pos), _ptr(kc), _ptr(vc),
                  dtype_code(kc), cache_len, cache_stride, _ptr(inv_freq), _ptr(out),
                  out.stride(0) if ldo is None else ldo, window, scale)


def rope_cache(qkv, ldq, M, hq, hkv, pos0, kc, vc, cache_len, inv_freq, stream=None) -> None:
    check(load().mt_rope_cache(_ptr(qkv), ldq, M, hq, hkv, pos0, _ptr(kc), _ptr(vc), dtype_code(kc), cache_len,
                               _ptr(inv_freq), _stream(stream)))


def rope_cache_decode(qkv, ldq, B, hq, hkv, pos, kc, vc, cache_len, cache_stride, inv_freq, stream=None) -> None:
    check(load().mt_rope_cache_decode(_ptr(qkv), ldq, B, hq, hkv, _ptr(pos), _ptr(kc), _ptr(vc), dtype_code(kc),
                                      cache_len, cache_stride, _ptr(inv_freq), _stream(stream)))


def attention(q, ldq, M, hq, hkv, pos0, window, kc, vc, cache_len, out, ldo, scale=0.125, stream=None) -> None:
    check(load().mt_attention(_ptr(q), ldq, M, hq, hkv, pos0, window, _ptr(kc), _ptr(vc), dtype_code(kc),
                              cache_len, _ptr(out), ldo, scale, _stream(stream)))


def rope_attention(qkv, ldq, M, hq, hkv, pos0, window, kc, vc, cache_len, inv_freq, out, ldo, scale=0.125,
                   stream=None) -> None:
    """rope_cache then attention over the same M rows in one launch (mt_rope_attention)."""
    check(load().mt_rope_attention(_ptr(qkv), ldq, M, hq, hkv, pos0, window, _ptr(kc), _ptr(vc), dtype_code(kc),
                                   cache_len, _ptr(inv_freq), _ptr(out), ldo, scale, _stream(stream)))


def attention_decode(q, ldq, B, hq, hkv, lens, window, kc, vc, cache_len, cache_stride, out, ldo, scale=0.125,
                     stream=None) -> None:
    check(load().mt_attention_decode(_ptr(q), ldq, B, hq, hkv, _ptr(lens), window, _ptr(kc), _ptr(vc),
                                     dtype_code(kc), cache_len, cache_stride, _ptr(out), ldo, scale,
                                     _stream(stream)))


# ----------------------------------- 8-bit storage and shared prefixes --

_slot_types: tuple = ()  # torch types of pos and counts
_row_type = None         # and of activations


def _storage_code(t) -> int:
    """dtype_code, and F8 for codes (uint8 or float8_e4m3fn).  Every cache and matrix passes here, so the types that
    the calls check are known behind it."""
    global _slot_types, _row_type
    import torch
    _slot_types, _row_type = (torch.int32, torch.uint32), torch.float32
    if t.dtype in (torch.uint8, torch.float8_e4m3fn):
        return F8
    return dtype_code(t)


class KV:
    """The caches of one layer (mt_kv): k and v torch tensors [B, hkv, cache_len, 64], or [hkv, cache_len, 64]
    for one sequence (a shared prefix), fp32, fp16 or 8-bit codes (uint8 or float8_e4m3fn); 8-bit caches have
    scale bytes k_scale and v_scale [B, hkv, cache_len].  A sequence's caches are contiguous; the batch may be strided,
    the same way for k and v (and for both scales)."""

    def __init__(self, k, v, k_scale=None, v_scale=None):
        t = _storage_code(k)
        for name, x, y, inner in (("k and v", k, v, 3), ("k_scale and v_scale", k_scale, v_scale, 2)):
            if inner == 2 and t != F8:
                continue
            if x is None or y is None or x.shape != y.shape or x.dtype != y.dtype or x.stride() != y.stride():
                raise ValueError(f"{name} must be two tensors of one shape, type and layout")
            if x.dim() not in (inner, inner + 1) or not x[(0,) * (x.dim() - inner)].is_contiguous():
                raise ValueError(f"{name}: [B, hkv, cache_len{', 64' if inner == 3 else ''}], contiguous but for B")
        if k.shape[-1] != 64 or t == BF16:
            raise ValueError("caches hold heads of 64 fp32, fp16 or 8-bit values")
        if t == F8 and (k_scale.shape != k.shape[:-1] or k_scale.element_size() != 1):
            raise ValueError("one scale byte a head and position")
        if any(x is not None and x.device != k.device for x in (v, k_scale, v_scale)):
            raise ValueError("caches and scales must be on one device")
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.hkv, self.cache_len, self.type = k.shape[-3], k.shape[-2], t
        self.batch = k.shape[0] if k.dim() == 4 else 1
        batched = k.dim() == 4
        self.device = k.get_device()
        self.struct = KvStruct(_ptr(k), _ptr(v), _ptr(k_scale), _ptr(v_scale), k.stride(0) if batched else 0,
                               k_scale.stride(0) if batched and t == F8 else 0, self.cache_len, t)
        self.ref = ctypes.byref(self.struct)

    @staticmethod
    def empty(batch, hkv, cache_len, dtype, device):
        """Zeroed caches of torch type ``dtype`` (uint8: 8 bits) for ``batch`` sequences."""
        import torch
        k = torch.zeros(batch, hkv, cache_len, 64, dtype=dtype, device=device)
        if _storage_code(k) != F8:
            return KV(k, torch.zeros_like(k))
        s = torch.ones(batch, hkv, cache_len, dtype=torch.uint8, device=device)
        return KV(k, torch.zeros_like(k), s, torch.ones_like(s))


def _refuse_kv(kv, B, hkv):
    raise ValueError(f"caches of {kv.batch} sequences and {kv.hkv} heads for {B} and {hkv}")


def _rows(device, t, rows, width, ld=None):
    """The address and row stride of `rows` fp32 rows of `width` values: a tensor [rows, width] or larger (several
    dimensions count as one where they can, before the rows' values and in them), or any tensor that holds them at a
    stride `ld` from its first element on."""
    if t.dtype is not _row_type or t.get_device() != device:
        raise ValueError("activations are fp32, on the caches' or weights' device")
    if ld is None:
        shape = t.shape
        if len(shape) == 2 and shape[0] >= rows and shape[1] >= width:
            ld, unit = t.stride()
            if unit == 1 or width == 1:
                return t.data_ptr(), ld
        return _folded_rows(device, t, rows, width)
    if rows and (rows - 1) * ld + width > t.untyped_storage().nbytes() // 4 - t.storage_offset():
        raise ValueError(f"no {rows} rows of {width} values at a stride of {ld} in {tuple(t.shape)}")
    return t.data_ptr(), ld


def _folded_rows(device, t, rows, width):
    if rows == 0:
        return t.data_ptr(), width
    if t.dim() > 2 and t.numel():
        w = 1  # the last dimensions that hold a row
        for n in reversed(t.shape):
            w *= n
            if w >= width:
                break
        try:
            return _rows(device, t.view(-1, w), rows, width)
        except RuntimeError:  # dimensions that are not one
            pass
    raise ValueError(f"not {rows} rows of {width} values side by side: {tuple(t.shape)} at strides {t.stride()}")


def _frequencies(device, t):
    if t.dtype is not _row_type or t.get_device() != device or t.numel() < 32 or not t.is_contiguous():
        raise ValueError("inv_freq holds 32 fp32 values side by side, on the caches' device")
    return t.data_ptr()


def _slots(device, t, B):
    """The address of pos or counts (None: none), a number a sequence."""
    if t is None:
        return None
    if t.dtype not in _slot_types or t.get_device() != device or t.numel() < B or not t.is_contiguous():
        raise ValueError("pos and counts are int32, one a sequence side by side, on the caches' device")
    return t.data_ptr()


def _on(device, stream):
    """The stream's handle; the kernels run on the current device, so it has to be the tensors'."""
    if stream is None and _raw_stream is not None:
        current = _current_device()
        s = _raw_stream(current)
    else:
        s = _stream(stream)
        current = device if _current_device is None else _current_device()
    if current != device:
        raise ValueError("the tensors are not on the current device")
    return s


def rope_append(qkv, B, T, hq, hkv, pos, kv, inv_freq, q=None, counts=None, offset=0, ldq=None, ldo=None, stream=None) -> None:
    """mt_rope_append: B x T rows of qkv rotated at offset + pos[b] + t, their keys and values appended to ``kv`` at
    slot pos[b] + t (pos None: 0), the rotated queries written to q.  counts (int32 [B]): a sequence's rows of T."""
    if kv.hkv != hkv or kv.batch < B:
        _refuse_kv(kv, B, hkv)
    d = kv.device
    src, ldq = _rows(d, qkv, B * T, (hq + 2 * hkv) * 64, ldq)
    dst, ldo = (None, 0) if q is None else _rows(d, q, B * T, hq * 64, ldo)
    rc = (_lib or load()).mt_rope_append(src, ldq, B, T, hq, hkv, _slots(d, pos, B), _slots(d, counts, B), offset, kv.ref,
                                         _frequencies(d, inv_freq), dst, ldo, _on(d, stream))
    if rc < 0:
        check(rc)


def kv_copy(src, dst, B, T, pos=None, counts=None, stream=None) -> None:
    """mt_kv_copy: slots pos[b] .. pos[b] + counts[b] - 1 of ``src`` to the same slots of ``dst``, converted."""
    if src.hkv != dst.hkv or src.batch < B or dst.batch < B:
        _refuse_kv(src if src.batch < B else dst, B, src.hkv)
    d = src.device
    if dst.device != d:
        raise ValueError("src and dst are on different devices")
    rc = (_lib or load()).mt_kv_copy(src.ref, dst.ref, B, T, src.hkv, _slots(d, pos, B),
                                     _slots(d, counts, B), _on(d, stream))
    if rc < 0:
        check(rc)


@functools.lru_cache(maxsize=4096)
def _shared_need(*sizes) -> int:
    """mt_attention_shared_workspace: the sizes alone decide."""
    return load().mt_attention_shared_workspace(*sizes)


def attention_shared(q, B, T, hq, hkv, pos, kv, out, prefix=None, prefix_len=None, len_max=0, window=0, counts=None,
                     scale=0.125, ldq=None, ldo=None, workspace=None, stream=None) -> None:
    """mt_attention_shared: the rows' attention over ``prefix`` (one sequence's KV, its first prefix_len slots; all
    by default) and then their own keys in ``kv`` up to their slot.  The workspace, where the split of the keys
    needs one, comes from torch's allocator (so a captured graph keeps its own) unless given as a uint8 tensor."""
    if kv.hkv != hkv or kv.batch < B:
        _refuse_kv(kv, B, hkv)
    d = kv.device
    if prefix is None:
        if prefix_len:
            raise ValueError(f"prefix_len {prefix_len} without a prefix")
        prefix_len, pre = 0, None
    else:
        if prefix.hkv != hkv:
            _refuse_kv(prefix, 1, hkv)
        if prefix.device != d:
            raise ValueError("prefix and kv are on different devices")
        if prefix_len is None:
            prefix_len = prefix.cache_len
        pre = prefix.ref
    src, ldq = _rows(d, q, B * T, hq * 64, ldq)
    dst, ldo = _rows(d, out, B * T, hq * 64, ldo)
    need = _shared_need(B, T, hq, hkv, prefix_len, len_max or kv.cache_len, window, kv.type)
    if workspace is not None:
        if workspace.get_device() != d or not workspace.is_contiguous():
            raise ValueError("the workspace is contiguous and on the caches' device")
    elif need:
        workspace = _scratch(need, q, stream)
    rc = (_lib or load()).mt_attention_shared(
        src, ldq, B, T, hq, hkv, _slots(d, pos, B), _slots(d, counts, B), kv.ref, pre, prefix_len, len_max, window, dst, ldo,
        scale, None if workspace is None else workspace.data_ptr(),
        0 if workspace is None else workspace.numel() * workspace.element_size(), _on(d, stream))
    if rc < 0:
        check(rc)


def _scratch(nbytes, like, stream):
    """Device memory for one call on ``stream``, from that stream's pool of torch's allocator: what is freed there is
    used again in the stream's order only."""
    import torch
    if stream is None:
        return torch.empty(nbytes, dtype=torch.uint8, device=like.device)
    if isinstance(stream, int):  # (torch takes a zero handle for a stream of its own pool)
        stream = torch.cuda.ExternalStream(stream, device=like.device) if stream else torch.cuda.default_stream(like.device)
    with torch.cuda.stream(stream):
        return torch.empty(nbytes, dtype=torch.uint8, device=like.device)


class F8Matrix:
    """A matrix in 8 bits: codes [rows, K] (uint8 or float8_e4m3fn, rows contiguous) and scale bytes
    [rows, 4 ceil(K / 512)], one a block of 128 values."""

    def __init__(self, codes, scales):
        if codes.dim() != 2 or _storage_code(codes) != F8 or codes.stride(1) != 1 or codes.shape[1] % 16:
            raise ValueError("codes: [rows, K] of 8 bits, K a multiple of 16")
        n, k = codes.shape
        if tuple(scales.shape) != (n, 4 * ((k + 511) // 512)) or scales.element_size() != 1 or scales.stride(1) != 1:
            raise ValueError("scales: [rows, 4 ceil(K / 512)] bytes")
        if scales.device != codes.device:
            raise ValueError("codes and scales must be on one device")
        self.codes, self.scales, self.shape = codes, scales, (n, k)
        self.whole = codes.is_contiguous() and scales.is_contiguous()  # as weights have to be
        self.device = codes.get_device()
        self.args = (_ptr(codes), codes.stride(0), _ptr(scales), scales.stride(0))

    @staticmethod
    def quantize(x, norm=None, eps=1e-6, stream=None):
        """mt_quantize_f8 of x [rows, K] into new tensors."""
        import torch
        n, k = x.shape
        lds = 4 * ((k + 511) // 512)
        m = F8Matrix(_scratch(n * k, x, stream).view(n, k), _scratch(n * lds, x, stream).view(n, lds))
        quantize_f8(x, m, norm=norm, eps=eps, stream=stream)
        return m


def quantize_f8(x, out, norm=None, eps=1e-6, stream=None) -> None:
    """mt_quantize_f8: the rows of x [rows, K], RMS-normalised with gain ``norm`` if given, into an F8Matrix.  The bytes
    between the rows of strided scales are set to 0, up to the last row's whole stride."""
    if tuple(x.shape) != tuple(out.shape) or x.stride(1) != 1:
        raise ValueError("x and the matrix must be of one shape, x's rows contiguous")
    s = out.scales
    if s.storage_offset() + s.shape[0] * s.stride(0) > s.untyped_storage().nbytes():
        raise ValueError("the scales end before their last row's stride")
    if x.get_device() != out.device or (norm is not None and norm.get_device() != out.device):
        raise ValueError("x, norm and the matrix must be on one device")
    if norm is not None and (norm.numel() < x.shape[1] or not norm.is_contiguous()):
        raise ValueError("norm holds K values side by side")
    check(load().mt_quantize_f8(_ptr(x), dtype_code(x), x.shape[0], x.shape[1], x.stride(0), _ptr(norm),
                                dtype_code(norm) if norm is not None else F16, eps, _ptr(out.codes), out.codes.stride(0),
                                _ptr(out.scales), out.scales.stride(0), _on(out.device, stream)))


LINEAR_F8_ROWS, LINEAR_F8_NORM_K = 16, 32768  # most rows mt_linear_f8 quantises itself, most values a row it normalises


def linear_f8(x, w, y, M=None, flags=0, w2=None, bias=None, norm=None, eps=1e-6, ldy=None, stream=None) -> None:
    """mt_linear_f8: y[:M] (op)= x[:M] @ w.T, w (and w2) F8Matrix [N, K]; x an F8Matrix or a float tensor, which is
    quantised in blocks of 128 on the way (after the RMSNorm with gain ``norm``), more than 16 rows by a call of
    mt_quantize_f8 first."""
    N, K = w.shape
    M = x.shape[0] if M is None else M
    rows, k = x.shape
    if k != K or rows < M or (w2 is not None and w2.shape != w.shape):
        raise ValueError("x, w and w2 must agree in K, w and w2 in shape")
    if (bias is not None and (bias.numel() < N or not bias.is_contiguous())) \
            or (norm is not None and (norm.numel() < K or not norm.is_contiguous())):
        raise ValueError("bias holds N values, norm K, side by side")
    if not w.whole or (w2 is not None and not w2.whole):
        raise ValueError("weights must be contiguous")
    if not isinstance(x, F8Matrix) and (M > LINEAR_F8_ROWS or (norm is not None and K > LINEAR_F8_NORM_K)):
        x, norm = F8Matrix.quantize(x[:M], norm=norm, eps=eps, stream=stream), None
    b = bias if bias is not None else norm
    bt = dtype_code(b) if b is not None else F16
    if bias is not None and norm is not None and dtype_code(norm) != bt:
        raise ValueError("bias and norm must be of one type")
    d = w.device
    if isinstance(x, F8Matrix):
        xp, ldx, xs, ldxs = x.args
        xt, on = F8, x.device
    else:
        ldx, unit = x.stride()
        if unit != 1:
            raise ValueError("x's rows must be contiguous")
        xp, xt, xs, ldxs, on = x.data_ptr(), dtype_code(x), None, 0, x.get_device()
    if on != d or (w2 is not None and w2.device != d) \
            or (bias is not None and bias.get_device() != d) or (norm is not None and norm.get_device() != d):
        raise ValueError("x, w, w2, bias and norm must be on one device")
    yp, ldy = _rows(d, y, M, N, ldy)
    wp, _, ws, _ = w.args
    up, _, us, _ = w2.args if w2 is not None else (None, 0, None, 0)
    rc = (_lib or load()).mt_linear_f8(xp, xt, xs, ldxs, _ptr(norm), wp, ws, up, us, _ptr(bias), bt, yp,
                                       GemvParams(M, N, K, ldx, ldy, flags, eps), _on(d, stream))
    if rc < 0:
        check(rc)


def dit_attention(qkv, B, S, H, inv_freq, out, ld=None, ldo=None, scale=0.125, stream=None) -> None:
    """Encoder.ditAttention: full attention with interleaved RoPE inside each of B sequences
    of S rows (Kernels.swift:208-220)."""
    check(load().mt_dit_attention(_ptr(qkv), qkv.stride(0) if ld is None else ld, B, S, H, _ptr(inv_freq), _ptr(out),
                                  out.stride(0) if ldo is None else ldo, scale, _stream(stream)))


def dit_attention_linear(qkv, B, S, H, inv_freq, w, y, flags=0, bias=None, scale=0.125, ldq=None, ldy=None,
                         stream=None) -> None:
    """Encoder.ditAttention then Encoder.linear of its output (DiT.swift:44-45) in one launch:
    y[:B S] (op)= dit_attention(qkv) @ w.T with the epilogue in ``flags``; w: [N, 64 H]."""
    N, K = w.shape
    p = GemvParams(B * S, N, K, qkv.stride(0) if ldq is None else ldq, y.stride(0) if ldy is None else ldy, flags, 0.0)
    check(load().mt_dit_attention_linear(_ptr(qkv), B, S, H, _ptr(inv_freq), scale, _ptr(w), dtype_code(w), _ptr(bias),
                                         _ptr(y), p, _stream(stream)))


def flow_assemble(y, history, cemb, cond_bias, temb, x_w, x_b, x, ldx=None, stream=None) -> None:
    """Encoder.flowAssemble: the six flow-input rows (Kernels.swift:222-235); x_w [hidden,
    latent_dim] of the weights' 16-bit type."""
    hidden, latent = x_w.shape
    check(load().mt_flow_assemble(_ptr(y), _ptr(history), _ptr(cemb), _ptr(cond_bias), _ptr(temb), _ptr(x_w),
                                  _ptr(x_b), dtype_code(x_w), _ptr(x), x.stride(0) if ldx is None else ldx, hidden,
                                  latent, _stream(stream)))


def flow_euler(y, pred, pred_row, null_row, cfg, dt, capture=None, ldp=None, stream=None) -> None:
    """Encoder.flowEuler: y += (c + (c - u) cfg) dt with c, u rows of pred (Kernels.swift:237-246)."""
    latent = y.numel()
    check(load().mt_flow_euler(_ptr(y), _ptr(pred), pred.stride(0) if ldp is None else ldp, pred_row, null_row,
                               _ptr(capture), latent, cfg, dt, _stream(stream)))


def flow_euler_assemble(y, pred, pred_row, null_row, cfg, dt, history, cemb, cond_bias, temb, x_w, x_b, x,
                        capture=None, ldp=None, ldx=None, stream=None) -> None:
    """flow_euler of one ODE step then flow_assemble of the next, in one launch."""
    hidden, latent = x_w.shape
    check(load().mt_flow_euler_assemble(_ptr(y), _ptr(pred), pred.stride(0) if ldp is None else ldp, pred_row, null_row,
                                        _ptr(capture), cfg, dt, _ptr(history), _ptr(cemb), _ptr(cond_bias), _ptr(temb),
                                        _ptr(x_w), _ptr(x_b), dtype_code(x_w), _ptr(x),
                                        x.stride(0) if ldx is None else ldx, hidden, latent, _stream(stream)))


def upsample4(prev, cur, nxt, frames, ldf=None, stream=None) -> None:
    """Encoder.upsample4 (Kernels.swift:247-257): prev / nxt None when absent."""
    check(load().mt_upsample4(_ptr(prev), _ptr(cur), _ptr(nxt), _ptr(frames), frames.stride(0) if ldf is None else ldf,
                              cur.numel(), _stream(stream)))


def istft_frames(spec, count, nfft, cos_table, window, ring_frames, frame0, ring, ld_spec=None, stream=None) -> None:
    """Encoder.istftFrames (Kernels.swift:259-270)."""
    check(load().mt_istft_frames(_ptr(spec), spec.stride(0) if ld_spec is None else ld_spec, count, nfft, _ptr(cos_table),
                                 _ptr(window), _ptr(ring_frames), frame0, ring, _stream(stream)))


def istft_emit(ring_frames, window, nfft, hop, s0, count, last_frame, ring, out, stream=None) -> None:
    """Encoder.istftEmit (Kernels.swift:272-283)."""
    check(load().mt_istft_emit(_ptr(ring_frames), _ptr(window), nfft, hop, s0, count, last_frame, ring, _ptr(out),
                               _stream(stream)))


# ------------------------------------------- mirror of the reference types --

@dataclass
class GPUTensor:
    """GPUTensor (Kernels.swift:7-11): a tensor at an element offset of a buffer, ``count``
    elements long; ``dtype`` names the element type when the buffer is a byte arena (a
    WeightArena's tensors sit at byte offsets of one uint8 buffer)."""
    buffer: object
    offset: int = 0
    count: int = 0
    dtype: Optional[int] = None

    def ptr(self) -> int:
        return self.buffer.data_ptr() + self.offset * self.buffer.element_size()

    def elem_type(self) -> int:
        return self.dtype if self.dtype is not None else dtype_code(self.buffer)


@dataclass
class Linear:
    """Linear (Kernels.swift:13-19): y = x W^T (+ bias), w [n, k] row-major."""
    w: GPUTensor
    bias: Optional[GPUTensor]
    n: int
    k: int


@dataclass
class ActView:
    """ActView (Kernels.swift:30-44): a view of rows at an element offset, stride ``ld``."""
    buffer: object
    offset: int = 0
    ld: int = 0

    def row(self, r: int) -> "ActView":
        return ActView(self.buffer, self.offset + r * self.ld, self.ld)

    def column(self, c: int) -> "ActView":
        return ActView(self.buffer, self.offset + c, self.ld)

    def ptr(self) -> int:
        return self.buffer.data_ptr() + self.offset * self.buffer.element_size()


class Encoder:
    """The reference's Encoder (Kernels.swift:89-206) over the C ABI, on one stream."""

    def __init__(self, stream=None):
        self.stream = stream

    def linear(self, x: ActView, rows: int, linear: Linear, y: ActView, flags: int = 0,
               gate: Optional[GPUTensor] = None) -> None:
        """Encoder.linear (Kernels.swift:132-161)."""
        wt = linear.w.elem_type()
        check(linear_raw(x.ptr(), dtype_code(x.buffer), linear.w.ptr(), gate.ptr() if gate else None, wt,
                         linear.bias.ptr() if linear.bias else None, y.ptr(), rows, linear.n, linear.k, x.ld, y.ld,
                         flags, self.stream))

    def rmsnorm(self, x: ActView, rows: int, width: int, weight: GPUTensor, y: ActView, eps: float = 1e-6) -> None:
        """Encoder.rmsnorm (Kernels.swift:163-171)."""
        check(rmsnorm_raw(x.ptr(), x.ld, rows, width, weight.ptr(), weight.elem_type(), y.ptr(), y.ld, eps,
                          self.stream))


# ----------------------------------------------------------- weight path --

class SafeTensors:
    """SafeTensors (SafeTensors.swift:7-87): a memory-mapped .safetensors file (mt_st_*).
    ``entries`` maps names (header order) to (dtype code or -1, shape, byte count)."""

    def __init__(self, path: str):
        h = ctypes.c_void_p()
        check(load().mt_st_open(os.fsencode(path), ctypes.byref(h)))
        self.handle = h
        L = load()
        self.entries = {}
        for i in range(check(L.mt_st_count(h))):
            name = ctypes.c_char_p()
            check(L.mt_st_name(h, i, ctypes.byref(name)))
            e = self.entry(name.value.decode())
            self.entries[name.value.decode()] = (e.dtype, tuple(e.shape[:e.ndim]), e.bytes)

    def entry(self, name: str) -> StEntry:
        e = StEntry()
        check(load().mt_st_find(self.handle, name.encode(), ctypes.byref(e)))
        return e

    def raw(self, name: str) -> bytes:
        """The tensor's bytes as stored."""
        e = self.entry(name)
        return ctypes.string_at(e.host, e.bytes)

    def close(self) -> None:
        if self.handle:
            load().mt_st_close(self.handle)
            self.handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class WeightArena:
    """WeightArena (Weights.swift:8-79) over mt_arena_*: plan tensors (``tensor``, ``linear``,
    ``padded_linear``), then ``upload`` into one 256-byte-aligned device buffer (a torch uint8
    tensor this object owns); the planned GPUTensor / Linear objects are bound to it then.
    ``convert_to`` F16 converts the bf16 weights to fp16 at upload (``audit`` gives the
    overflow and flush-to-zero counts)."""

    def __init__(self, st: SafeTensors, convert_to: int = BF16):
        h = ctypes.c_void_p()
        check(load().mt_arena_create(st.handle, convert_to, ctypes.byref(h)))
        self.handle, self.st, self.dtype = h, st, convert_to
        self.buffer = None
        self._planned = []

    def tensor(self, *names: str) -> "GPUTensor":
        arr = (ctypes.c_char_p * len(names))(*[n.encode() for n in names])
        off, cnt = ctypes.c_uint64(), ctypes.c_uint64()
        check(load().mt_arena_tensor(self.handle, arr, len(names), ctypes.byref(off), ctypes.byref(cnt)))
        t = GPUTensor(None, off.value, cnt.value)
        self._planned.append(t)
        return t

    def linear(self, prefix: str, n: int, k: int, bias: bool) -> "Linear":
        w = self.tensor(prefix + ".weight")
        if w.count != n * k:
            raise MingTTSError(EINVAL, f"bad checkpoint: {prefix}.weight has {w.count} elements, expected {n}x{k}")
        return Linear(w, self.tensor(prefix + ".bias") if bias else None, n, k)

    def padded_linear(self, prefix: str, n: int, k: int, stored_k: int) -> "Linear":
        off = ctypes.c_uint64()
        check(load().mt_arena_padded(self.handle, (prefix + ".weight").encode(), n, k, stored_k, ctypes.byref(off)))
        t = GPUTensor(None, off.value, n * k)
        self._planned.append(t)
        return Linear(t, None, n, k)

    @property
    def nbytes(self) -> int:
        return load().mt_arena_bytes(self.handle)

    def upload(self, device=None, stream=None) -> None:
        import torch
        dev = torch.device("cuda", 0) if device is None else device
        self.buffer = torch.empty(max(self.nbytes, 256), dtype=torch.uint8, device=dev)
        check(load().mt_arena_upload(self.handle, self.buffer.data_ptr(), _stream(stream)))
        for t in self._planned:
            t.buffer, t.dtype = self.buffer, self.dtype

    def audit(self) -> tuple:
        ov, un = ctypes.c_uint64(), ctypes.c_uint64()
        check(load().mt_arena_audit(self.handle, ctypes.byref(ov), ctypes.byref(un)))
        return ov.value, un.value

    def close(self) -> None:
        if self.handle:
            load().mt_arena_destroy(self.handle)
            self.handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    @staticmethod
    def load(st: SafeTensors, build, convert_to: int = BF16, device=None):
        """WeightArena.load (Weights.swift:15-22): plans with ``build(arena)``, allocates and
        uploads, and returns the build's result bound to the arena (kept on ``result``'s
        arena attribute by the caller as needed)."""
        arena = WeightArena(st, convert_to)
        result = build(arena)
        arena.upload(device)
        return result, arena


from .flow import FlowSchedule, time_embeddings  # noqa: E402  (host side of the flow sampler)
