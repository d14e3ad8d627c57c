"""Python binding of the ema_attn C ABI (include/ema_attn.h).

Thin ctypes layer used by the tests and the benchmark: tensors are torch
device tensors (bf16 / int32), every call goes through ``libema_attn.so`` and
fails loudly when the library is missing or a call returns an error. There is
no fallback path.

The names mirror the reference's API for this path:
``KvCache``/``StaticCache`` (crates/kvcache/src/lib.rs:52-76) and
``gqa_attention`` (crates/attention/src/gqa.rs:62-107) minus the projections.
"""
from __future__ import annotations

import ctypes
import math
import os

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_HERE, "libema_attn.so")

EMA_OK = 0
EMA_ERR_INVALID_ARG = -1
EMA_ERR_SHAPE = -2
EMA_ERR_CAPACITY = -3
EMA_ERR_WORKSPACE = -4
EMA_ERR_UNSUPPORTED = -5
EMA_ERR_HIP = -6

EMA_DTYPE_BF16 = 1
EMA_DTYPE_FP8_E4M3 = 2
EMA_DTYPE_F16 = 3
EMA_DTYPE_F32 = 4
EMA_DTYPE_INT4_AFFINE = 5
EMA_PRE_NO_NORM = 1
EMA_PRE_NO_ROPE = 2
EMA_PRE_NO_Q_NORM = 8
EMA_PRE_NO_K_NORM = 16
EMA_STEP_ADVANCE = 4
EMA_DECODE_COUNTER_BYTES = 131072
EMA_KV_ROTATING = 1
EMA_PREFILL_CAUSAL = 1
EMA_PREFILL_CHUNK_ONLY = 2
EMA_PREFILL_ROWS_DECODED = 4
EMA_CONV_SILU = 1
EMA_SSM_SOFTPLUS = 1
EMA_NORM_GATE_FIRST = 1
EMA_NORM_GATE_SIGMOID = 2
EMA_NORM_SHARED_WEIGHT = 4
EMA_NORM_UNIT_OFFSET = 8

EXPORTED = (
    "ema_last_error", "ema_version", "ema_kvcache_init", "ema_kvcache_alloc", "ema_kvcache_free",
    "ema_kvcache_init_fp8", "ema_kvcache_alloc_fp8", "ema_kvcache_init_int4", "ema_kvcache_alloc_int4",
    "ema_kvcache_quantize_int4", "ema_kvcache_convert", "ema_position_write",
    "ema_kvcache_memory_bytes", "ema_pre_attention", "ema_pre_attention_ws", "ema_decode_workspace_size",
    "ema_decode_attention", "ema_decode_step", "ema_decode_step_noalloc", "ema_prefill_attention", "ema_prefill_workspace_size",
    "ema_prefill_attention_ws", "ema_gdn_scan", "ema_gdn_scan_workspace_size", "ema_gdn_scan_ws",
    "ema_quantized_matmul", "ema_paged_append", "ema_paged_workspace_size", "ema_paged_attention",
    "ema_prefix_attention", "ema_causal_conv", "ema_ssm_workspace_size", "ema_ssm_scan", "ema_gated_norm",
    "ema_residual_norm",
)


class EmaError(RuntimeError):
    def __init__(self, code: int, op: str, msg: str):
        super().__init__(f"{op} failed with code {code}: {msg}")
        self.code = code
        self.op = op
        self.msg = msg


class KvCacheDesc(ctypes.Structure):
    _fields_ = [
        ("k", ctypes.c_void_p), ("v", ctypes.c_void_p),
        ("batch", ctypes.c_int32), ("n_kv_heads", ctypes.c_int32),
        ("capacity", ctypes.c_int32), ("head_dim", ctypes.c_int32),
        ("stride_batch", ctypes.c_int64), ("stride_head", ctypes.c_int64),
        ("stride_pos", ctypes.c_int64), ("dtype", ctypes.c_int32), ("flags", ctypes.c_int32),
        ("k_exp", ctypes.c_void_p), ("v_exp", ctypes.c_void_p),
        ("k_scales", ctypes.c_void_p), ("k_biases", ctypes.c_void_p),
        ("v_scales", ctypes.c_void_p), ("v_biases", ctypes.c_void_p),
        ("n_rot", ctypes.c_int32),
    ]


_lib = None


def lib() -> ctypes.CDLL:
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise RuntimeError(f"ema_attn HIP library not built: {LIB_PATH} (run __graft_entry__.build())")
        L = ctypes.CDLL(LIB_PATH)
        vp, i32, u32, f32, u64 = ctypes.c_void_p, ctypes.c_int32, ctypes.c_uint32, ctypes.c_float, ctypes.c_uint64
        i64 = ctypes.c_int64
        D = ctypes.POINTER(KvCacheDesc)
        sig = {
            "ema_last_error": (ctypes.c_char_p, []),
            "ema_version": (ctypes.c_char_p, []),
            "ema_kvcache_init": (i32, [D, vp, vp, i32, i32, i32, i32]),
            "ema_kvcache_alloc": (i32, [D, i32, i32, i32, i32]),
            "ema_kvcache_init_fp8": (i32, [D, vp, vp, vp, vp, i32, i32, i32, i32, i32]),
            "ema_kvcache_alloc_fp8": (i32, [D, i32, i32, i32, i32, i32]),
            "ema_kvcache_init_int4": (i32, [D, vp, vp, vp, vp, vp, vp, i32, i32, i32, i32]),
            "ema_kvcache_alloc_int4": (i32, [D, i32, i32, i32, i32]),
            "ema_kvcache_quantize_int4": (i32, [vp, D, i32, D, i32, i32]),
            "ema_kvcache_convert": (i32, [vp, D, i32, D, i32, i32]),
            "ema_position_write": (i32, [vp, vp, i32]),
            "ema_kvcache_free": (i32, [D]),
            "ema_kvcache_memory_bytes": (i32, [D, ctypes.POINTER(u64)]),
            "ema_pre_attention": (i32, [vp, vp, vp, vp, f32, f32, vp, i32, i32, i32, i32, i32, u32, vp, D]),
            "ema_pre_attention_ws": (i32, [vp, vp, vp, vp, f32, f32, vp, i32, i32, i32, i32, i32, u32, vp, D, i32, vp,
                                           u64]),
            "ema_decode_workspace_size": (i32, [i32, i32, i32, i32, i32, ctypes.POINTER(u64)]),
            "ema_decode_attention": (i32, [vp, vp, D, vp, i32, i32, f32, vp, vp, u64]),
            "ema_decode_step": (i32, [vp, vp, vp, vp, f32, f32, vp, i32, i32, u32, f32, D, vp, vp, u64]),
            "ema_decode_step_noalloc": (i32, [vp, vp, vp, vp, f32, f32, vp, i32, i32, u32, f32, D, vp]),
            "ema_prefill_attention": (i32, [vp, vp, D, vp, i32, i32, f32, u32, vp]),
            "ema_prefill_workspace_size": (i32, [D, i32, ctypes.POINTER(u64)]),
            "ema_prefill_attention_ws": (i32, [vp, vp, D, vp, i32, i32, f32, u32, vp, i32, vp, u64]),
            "ema_gdn_scan": (i32, [vp, vp, vp, vp, vp, vp, vp, vp, i32, i32, i32, i32, i32, i32, i32]),
            "ema_gdn_scan_workspace_size": (i32, [i32, i32, i32, i32, i32, i32, ctypes.POINTER(u64)]),
            "ema_gdn_scan_ws": (i32, [vp, vp, vp, vp, vp, vp, vp, vp, i32, i32, i32, i32, i32, i32, i32, vp, u64]),
            "ema_paged_append": (i32, [vp, vp, vp, vp, f32, f32, vp, vp, vp, i32, i32, i32, u32, vp, D, vp, i32]),
            "ema_paged_workspace_size": (i32, [i32] * 8 + [ctypes.POINTER(u64)]),
            "ema_paged_attention": (i32, [vp, vp, D, vp, i32, vp, vp, i32, i32, i32, i32, i32, f32, u32, vp, vp, u64]),
            "ema_prefix_attention": (i32, [vp, vp, D, vp, i32, vp, i32, vp, i32, vp, vp, i32, i32, i32, i32, i32, f32,
                                           vp, vp, u64]),
            "ema_causal_conv": (i32, [vp, vp, i64, vp, vp, vp, vp, vp, i32, i32, i32, i32, i32, u32, vp, i32, vp, i64, i32]),
            "ema_ssm_workspace_size": (i32, [i32] * 8 + [ctypes.POINTER(u64)]),
            "ema_ssm_scan": (i32, [vp, vp, i64, vp, i64, vp, i64, vp, i64, vp, vp, vp, f32, f32, vp, vp, vp, i32, i32, i32,
                                   i32, i32, i32, i32, u32, vp, i32, vp, i64, i32, vp, u64]),
            "ema_gated_norm": (i32, [vp, vp, i64, vp, i64, vp, f32, i32, i32, i32, u32, vp, i64, i32]),
            "ema_residual_norm": (i32, [vp, vp, i64, vp, vp, i64, f32, vp, i64, i32, vp, f32, i32, i32, u32, vp, i64, i32]),
            "ema_quantized_matmul": (i32, [vp, vp, i64, vp, vp, vp, vp, i64, i32, i32, i32, i32, i32, i32]),
        }
        for name, (res, args) in sig.items():
            fn = getattr(L, name)
            fn.restype = res
            fn.argtypes = args
        _lib = L
    return _lib


def last_error() -> str:
    return lib().ema_last_error().decode()


def version() -> str:
    return lib().ema_version().decode()


def _check(rc: int, op: str) -> None:
    if rc != EMA_OK:
        raise EmaError(rc, op, last_error())


def _ptr(t) -> int | None:
    return None if t is None else t.data_ptr()


def _stream(stream) -> int | None:
    import torch

    if stream is None:
        stream = torch.cuda.current_stream()
    return stream.cuda_stream


class StaticCache:
    """Static pre-allocated KV cache of one layer, [B, Hkv, cap, D], bf16 or FP8.

    Mirrors the reference's static KV state (crates/serve/src/engine.rs:31-42,
    alloc_kv_static at crates/serve/src/engine_ext.rs:266-306) behind the
    KvCache trait surface (crates/kvcache/src/lib.rs:52-76): ``len`` is the
    number of valid positions per sequence, ``reset`` only rewinds the offsets
    (stale rows stay and are excluded by length, engine_ext.rs:218-228).

    ``dtype="fp8"``: the stored form of the reference's Fp8Cache
    (crates/kvcache/src/fp8.rs): ``k``/``v`` are uint8 E4M3FN codes and
    ``k_exp``/``v_exp`` int8 [B, Hkv, cap, D/64] block exponents
    (value = code * 2^exp); head_dim 128. ``n_rot=64`` (Fp8Cache::new(128, 64)): the last
    64 dims of each row are kept as bf16, so a row of ``k``/``v`` is [B, Hkv, cap, 192]
    bytes, 64 codes then the 64 bf16 values (block 1's exponent is 0).

    ``dtype="int4"``: the reference's int4 KV buffers (alloc_kv_int4,
    crates/serve/src/engine_ext.rs:92-129): ``k``/``v`` are int32 words [B, Hkv, cap, D/8]
    (8 four-bit codes each, lowest bits first) and ``k_scales``/``k_biases``/``v_scales``/
    ``v_biases`` bf16 [B, Hkv, cap, D/64] (value = scale * code + bias); head_dim 128,
    capacity a multiple of 32, decode only (static or rotating).

    ``rotating=True``: the reference's RotatingCache (crates/kvcache/src/rotating.rs) as a
    ring of ``capacity`` rows (EMA_KV_ROTATING): position p lives in row p % capacity and
    attention covers the last ``capacity`` tokens; ``len`` is then min(tokens, capacity).
    """

    def __init__(self, batch: int, n_kv_heads: int, capacity: int, head_dim: int, device="cuda",
                 k=None, v=None, dtype="bf16", k_exp=None, v_exp=None, rotating=False, k_scales=None,
                 k_biases=None, v_scales=None, v_biases=None, n_rot=0):
        import torch

        shape = (batch, n_kv_heads, capacity, head_dim)
        self.desc = KvCacheDesc()
        self.dtype = dtype
        if dtype == "bf16":
            self.k = k if k is not None else torch.zeros(shape, dtype=torch.bfloat16, device=device)
            self.v = v if v is not None else torch.zeros(shape, dtype=torch.bfloat16, device=device)
            self.k_exp = self.v_exp = None
            _check(lib().ema_kvcache_init(ctypes.byref(self.desc), _ptr(self.k), _ptr(self.v), batch, n_kv_heads,
                                          capacity, head_dim), "ema_kvcache_init")
        elif dtype == "fp8":
            eshape = (batch, n_kv_heads, capacity, head_dim // 64)
            rshape = (batch, n_kv_heads, capacity, head_dim + n_rot)
            self.k = k if k is not None else torch.zeros(rshape, dtype=torch.uint8, device=device)
            self.v = v if v is not None else torch.zeros(rshape, dtype=torch.uint8, device=device)
            self.k_exp = k_exp if k_exp is not None else torch.zeros(eshape, dtype=torch.int8, device=device)
            self.v_exp = v_exp if v_exp is not None else torch.zeros(eshape, dtype=torch.int8, device=device)
            _check(lib().ema_kvcache_init_fp8(ctypes.byref(self.desc), _ptr(self.k), _ptr(self.v), _ptr(self.k_exp),
                                              _ptr(self.v_exp), batch, n_kv_heads, capacity, head_dim, n_rot),
                   "ema_kvcache_init_fp8")
        elif dtype == "int4":
            mshape = (batch, n_kv_heads, capacity, head_dim // 64)
            self.k = k if k is not None else torch.zeros(shape[:3] + (head_dim // 8,), dtype=torch.int32, device=device)
            self.v = v if v is not None else torch.zeros(shape[:3] + (head_dim // 8,), dtype=torch.int32, device=device)
            self.k_exp = self.v_exp = None
            self.k_scales, self.k_biases, self.v_scales, self.v_biases = (
                t if t is not None else torch.zeros(mshape, dtype=torch.bfloat16, device=device)
                for t in (k_scales, k_biases, v_scales, v_biases))
            _check(lib().ema_kvcache_init_int4(ctypes.byref(self.desc), _ptr(self.k), _ptr(self.v),
                                               _ptr(self.k_scales), _ptr(self.k_biases), _ptr(self.v_scales),
                                               _ptr(self.v_biases), batch, n_kv_heads, capacity, head_dim),
                   "ema_kvcache_init_int4")
        else:
            raise ValueError(f"unknown cache dtype {dtype!r} (bf16, fp8 or int4)")
        if n_rot and dtype != "fp8":
            raise ValueError("n_rot is an fp8 cache parameter")
        self.rotating = bool(rotating)
        if self.rotating:
            self.desc.flags = EMA_KV_ROTATING
        self.offsets = [0] * batch

    @property
    def capacity(self) -> int:
        return self.desc.capacity

    def len(self) -> int:
        n = max(self.offsets) if self.offsets else 0
        return min(n, self.capacity) if self.rotating else n

    def is_empty(self) -> bool:
        return self.len() == 0

    def reset(self) -> None:
        self.offsets = [0] * len(self.offsets)

    def memory_bytes(self) -> int:
        out = ctypes.c_uint64()
        _check(lib().ema_kvcache_memory_bytes(ctypes.byref(self.desc), ctypes.byref(out)), "ema_kvcache_memory_bytes")
        return out.value


def quantize_int4(src: StaticCache, dst: StaticCache, n_rows: int, src_row: int = 0, dst_row: int = 0,
                  stream=None) -> None:
    """Rows [src_row, src_row + n_rows) of the bf16 cache ``src`` quantised into rows
    [dst_row, ...) of the int4 cache ``dst`` (convert_kv_to_int4,
    crates/serve/src/engine_ext.rs:158-210)."""
    _check(lib().ema_kvcache_quantize_int4(_stream(stream), ctypes.byref(src.desc), src_row, ctypes.byref(dst.desc),
                                           dst_row, n_rows), "ema_kvcache_quantize_int4")


def kvcache_convert(src: StaticCache, dst: StaticCache, n_rows: int, src_row: int = 0, dst_row: int = 0,
                    stream=None) -> None:
    """Rows [src_row, src_row + n_rows) of ``src`` converted into rows [dst_row, ...) of
    ``dst``: bf16 -> FP8 (Fp8Cache::append's quantisation, crates/kvcache/src/fp8.rs:47-68),
    FP8 -> bf16 (the decoded values Fp8Cache::get returns) or bf16 -> int4."""
    _check(lib().ema_kvcache_convert(_stream(stream), ctypes.byref(src.desc), src_row, ctypes.byref(dst.desc),
                                     dst_row, n_rows), "ema_kvcache_convert")


def position_write(slot, value: int, stream=None) -> None:
    """Stream-ordered write of ``value`` into the device int32 tensor element ``slot``."""
    _check(lib().ema_position_write(_stream(stream), _ptr(slot), int(value)), "ema_position_write")


def pre_attention(qkv, q_norm_w, k_norm_w, eps, theta, offsets, n_heads, cache: StaticCache, flags=0,
                  q_out=None, stream=None, prefill_workspace=None, max_kv_len=None):
    """qkv [B,T,(Hq+2Hkv)*D] bf16; offsets int32 device [B]. Returns q_out [B,Hq,T,D].

    With prefill_workspace (an FP8 cache: the workspace of prefill_attention for max_kv_len,
    default the capacity), ema_pre_attention_ws also writes the stored rows, decoded, into
    its bf16 copy; pass rows_decoded=True to prefill_attention with the same workspace."""
    import torch

    B, T, F = qkv.shape
    D = cache.desc.head_dim
    Hkv = cache.desc.n_kv_heads
    if q_out is None:
        q_out = torch.empty((B, n_heads, T, D), dtype=torch.bfloat16, device=qkv.device)
    if prefill_workspace is not None:
        if max_kv_len is None:
            max_kv_len = cache.capacity
        _check(lib().ema_pre_attention_ws(_stream(stream), _ptr(qkv), _ptr(q_norm_w), _ptr(k_norm_w), eps, theta,
                                          _ptr(offsets), B, T, n_heads, Hkv, D, flags, _ptr(q_out),
                                          ctypes.byref(cache.desc), max_kv_len, _ptr(prefill_workspace),
                                          prefill_workspace.numel()), "ema_pre_attention_ws")
        return q_out
    _check(lib().ema_pre_attention(_stream(stream), _ptr(qkv), _ptr(q_norm_w), _ptr(k_norm_w), eps, theta,
                                   _ptr(offsets), B, T, n_heads, Hkv, D, flags, _ptr(q_out),
                                   ctypes.byref(cache.desc)), "ema_pre_attention")
    return q_out


def decode_workspace_size(batch, n_heads, n_kv_heads, head_dim, max_len) -> int:
    out = ctypes.c_uint64()
    _check(lib().ema_decode_workspace_size(batch, n_heads, n_kv_heads, head_dim, max_len, ctypes.byref(out)),
           "ema_decode_workspace_size")
    return out.value


def decode_workspace(batch, n_heads, n_kv_heads, head_dim, max_len, device="cuda", stream=None):
    """Allocate a decode workspace (reusable across calls on one stream, any shape): zero-
    filled, as the arrival counters at its start must be before the first call."""
    import torch

    n = decode_workspace_size(batch, n_heads, n_kv_heads, head_dim, max_len)
    return torch.zeros(n, dtype=torch.uint8, device=device)


def decode_attention(q, cache: StaticCache, lengths, max_len, scale=None, out=None, workspace=None, stream=None):
    """q [B,Hq,D] (or [B,Hq,1,D]) bf16; lengths int32 device [B]. Returns out [B, Hq*D]."""
    import torch

    B, Hq = q.shape[0], q.shape[1]
    D = cache.desc.head_dim
    if scale is None:
        scale = 1.0 / math.sqrt(D)
    if out is None:
        out = torch.empty((B, Hq * D), dtype=torch.bfloat16, device=q.device)
    if workspace is None:
        workspace = decode_workspace(B, Hq, cache.desc.n_kv_heads, D, max_len, device=q.device, stream=stream)
    _check(lib().ema_decode_attention(_stream(stream), _ptr(q), ctypes.byref(cache.desc), _ptr(lengths), max_len, Hq,
                                      scale, _ptr(out), _ptr(workspace), workspace.numel()), "ema_decode_attention")
    return out


def decode_step(qkv, q_norm_w, k_norm_w, eps, theta, offsets, n_heads, cache: StaticCache, max_len, scale=None,
                flags=0, out=None, workspace=None, stream=None):
    """Fused pre-attention (one token per sequence) + decode attention.

    qkv [B,(Hq+2Hkv)*D] (or [B,1,...]) bf16; offsets int32 device [B]. Returns out [B, Hq*D]."""
    import torch

    B = qkv.shape[0]
    D = cache.desc.head_dim
    if scale is None:
        scale = 1.0 / math.sqrt(D)
    if out is None:
        out = torch.empty((B, n_heads * D), dtype=torch.bfloat16, device=qkv.device)
    if workspace is None:
        workspace = decode_workspace(B, n_heads, cache.desc.n_kv_heads, D, max_len, device=qkv.device)
    _check(lib().ema_decode_step(_stream(stream), _ptr(qkv), _ptr(q_norm_w), _ptr(k_norm_w), eps, theta,
                                 _ptr(offsets), max_len, n_heads, flags, scale, ctypes.byref(cache.desc), _ptr(out),
                                 _ptr(workspace), workspace.numel()), "ema_decode_step")
    return out


def decode_step_noalloc(qkv, q_norm_w, k_norm_w, eps, theta, offsets, n_heads, cache: StaticCache, max_len, out,
                        scale=None, flags=0, stream=None):
    """ema_decode_step over the library's static per-device scratch: no workspace and no
    device allocation in the call (out is the caller's [B, Hq*D] bf16 buffer)."""
    D = cache.desc.head_dim
    if scale is None:
        scale = 1.0 / math.sqrt(D)
    _check(lib().ema_decode_step_noalloc(_stream(stream), _ptr(qkv), _ptr(q_norm_w), _ptr(k_norm_w), eps, theta,
                                         _ptr(offsets), max_len, n_heads, flags, scale, ctypes.byref(cache.desc),
                                         _ptr(out)), "ema_decode_step_noalloc")
    return out


def prefill_workspace_size(cache: StaticCache, max_kv_len: int) -> int:
    out = ctypes.c_uint64()
    _check(lib().ema_prefill_workspace_size(ctypes.byref(cache.desc), max_kv_len, ctypes.byref(out)),
           "ema_prefill_workspace_size")
    return out.value


def prefill_attention(q, cache: StaticCache, q_offsets, scale=None, causal=True, chunk_only=False, out=None,
                      stream=None, max_kv_len=None, workspace=None, rows_decoded=False):
    """q [B,Hq,T,D] bf16; q_offsets int32 device [B]. Returns out [B,T,Hq*D].

    An FP8 cache goes through ema_prefill_attention_ws: its attended rows (at most
    max_kv_len per sequence, default the capacity) are decoded into a bf16 workspace.
    rows_decoded: the chunk's rows are in that workspace already (pre_attention with
    prefill_workspace, EMA_PREFILL_ROWS_DECODED)."""
    import torch

    B, Hq, T, D = q.shape
    if scale is None:
        scale = 1.0 / math.sqrt(D)
    if out is None:
        out = torch.empty((B, T, Hq * D), dtype=torch.bfloat16, device=q.device)
    flags = (EMA_PREFILL_CAUSAL if causal else 0) | (EMA_PREFILL_CHUNK_ONLY if chunk_only else 0)
    flags |= EMA_PREFILL_ROWS_DECODED if rows_decoded else 0
    if cache.dtype == "bf16" and workspace is None:
        _check(lib().ema_prefill_attention(_stream(stream), _ptr(q), ctypes.byref(cache.desc), _ptr(q_offsets), T,
                                           Hq, scale, flags, _ptr(out)), "ema_prefill_attention")
        return out
    if max_kv_len is None:
        max_kv_len = cache.capacity
    if workspace is None:
        workspace = torch.empty(max(prefill_workspace_size(cache, max_kv_len), 16), dtype=torch.uint8,
                                device=q.device)
    _check(lib().ema_prefill_attention_ws(_stream(stream), _ptr(q), ctypes.byref(cache.desc), _ptr(q_offsets), T,
                                          Hq, scale, flags, _ptr(out), max_kv_len, _ptr(workspace),
                                          workspace.numel()), "ema_prefill_attention_ws")
    return out


def gdn_scan_workspace_size(B, T, Hk, Hv, Dk, Dv) -> int:
    """Bytes of the workspace with which gdn_scan runs T tokens in one segment
    (ema_gdn_scan_workspace_size)."""
    n = ctypes.c_uint64(0)
    _check(lib().ema_gdn_scan_workspace_size(B, T, Hk, Hv, Dk, Dv, ctypes.byref(n)), "ema_gdn_scan_workspace_size")
    return n.value


def gdn_workspace(B, T, Hk, Hv, Dk, Dv, device="cuda"):
    """A workspace tensor for gdn_scan (no initialisation needed)."""
    import torch

    return torch.empty(gdn_scan_workspace_size(B, T, Hk, Hv, Dk, Dv), dtype=torch.uint8, device=device)


def gdn_scan(q, k, v, g, beta, state, y=None, stream=None, workspace=None):
    """Gated DeltaNet recurrent scan (ema_gdn_scan): q, k [B,T,Hk,Dk], v [B,T,Hv,Dv] in bf16,
    f16 or f32; g, beta [B,T,Hv] f32 (inputs that are not contiguous, such as pieces of a convolution's
    rows, are copied first); state [B,Hv,Dv,Dk] f32, contiguous, updated in place. Returns
    y [B,T,Hv,Dv] in the activation dtype. With a workspace (a uint8 tensor, e.g. from
    gdn_workspace) bf16 scans of 32+ tokens run in WY form (ema_gdn_scan_ws)."""
    op = "ema_gdn_scan"
    torch = _torch or _load_torch()
    dtype, dev, f32 = q.dtype, q.get_device(), torch.float32
    code = _act_code(op, q)
    if q.dim() != 4 or v.dim() != 4:
        raise EmaError(EMA_ERR_SHAPE, op, f"q must be [B,T,Hk,Dk] and v [B,T,Hv,Dv], not {tuple(q.shape)}, {tuple(v.shape)}")
    B, T, Hk, Dk = q.shape
    _, _, Hv, Dv = v.shape
    values, gates = (B, T, Hv, Dv), (B, T, Hv)
    if y is None:
        y = _empty(stream, values, dtype, q.device) if stream is not None else torch.empty(values, dtype=dtype, device=q.device)
    if not (k.dtype is dtype and k.shape == q.shape and k.get_device() == dev and k.is_contiguous() and q.is_contiguous()
            and v.dtype is dtype and v.shape == values and v.get_device() == dev and v.is_contiguous()
            and g.dtype is f32 and g.shape == gates and g.get_device() == dev and g.is_contiguous()
            and beta.dtype is f32 and beta.shape == gates and beta.get_device() == dev and beta.is_contiguous()
            and y.dtype is dtype and y.shape == values and y.get_device() == dev and y.is_contiguous()
            and state.dtype is f32 and state.shape == (B, Hv, Dv, Dk) and state.get_device() == dev and state.is_contiguous()
            and (workspace is None or (workspace.get_device() == dev and workspace.is_contiguous()))):
        for name, t, kind, shape in (("k", k, dtype, (B, T, Hk, Dk)), ("v", v, dtype, values), ("g", g, f32, gates),
                                     ("beta", beta, f32, gates)):
            if t.shape != shape or t.dtype is not kind or t.get_device() != dev:
                raise EmaError(EMA_ERR_SHAPE, op, f"{name} must be a {kind} tensor {shape} on {q.device}, not {t.dtype} "
                                                  f"{tuple(t.shape)} on {t.device}")
        _want(op, "y", y, dtype, values, dev)
        _want(op, "state", state, f32, (B, Hv, Dv, Dk), dev)
        if workspace is not None:
            _want(op, "workspace", workspace, workspace.dtype, workspace.shape, dev)
        with _on(stream):
            q, k, v, g, beta = (t.contiguous() for t in (q, k, v, g, beta))
    if dev < 0:
        _not_on_gpu(op)
    args = (torch._C._cuda_getCurrentRawStream(dev) if stream is None else stream.cuda_stream, q.data_ptr(), k.data_ptr(),
            v.data_ptr(), g.data_ptr(), beta.data_ptr(), state.data_ptr(), y.data_ptr(), B, T, Hk, Hv, Dk, Dv, code)
    call = _lib.ema_gdn_scan
    if workspace is not None:
        call, op = _lib.ema_gdn_scan_ws, "ema_gdn_scan_ws"
        args += workspace.data_ptr(), workspace.numel() * workspace.element_size()
    rc = call(*args) if torch._C._cuda_getDevice() == dev else _elsewhere(dev, call, *args)
    if rc:
        _check(rc, op)
    return y


def quantized_matmul(x, w, scales, biases, group_size=64, bits=4, out=None, stream=None):
    """MLX quantized_matmul(x, w, scales, biases, transpose=True, group_size, bits, "affine")
    (ema_quantized_matmul; the reference's qmatmul, crates/ops/src/quant.rs:57-76): x [..., K]
    bf16 or f16 with a contiguous last axis; w [N, K*bits/32] int32/uint32 words of MLX's
    packing; scales, biases [N, K/group_size] in x's dtype. Returns y [..., N] in x's dtype.
    `out` may be a 2-D view whose rows are wider than N (e.g. the q, k or v columns of a
    q|k|v buffer)."""
    import torch

    dtypes = {torch.bfloat16: EMA_DTYPE_BF16, torch.float16: EMA_DTYPE_F16}
    if x.dtype not in dtypes:
        raise EmaError(EMA_ERR_INVALID_ARG, "ema_quantized_matmul", f"unsupported activation dtype {x.dtype}")
    K = x.shape[-1]
    x2 = x.reshape(-1, K)
    M, N = x2.shape[0], w.shape[0]
    if w.shape[1] * 32 // bits != K:
        raise EmaError(EMA_ERR_SHAPE, "ema_quantized_matmul", f"w {tuple(w.shape)} does not pack K={K} at {bits} bits")
    if out is None:
        y2 = torch.empty((M, N), dtype=x.dtype, device=x.device)
    else:
        y2 = out
        if y2.dim() != 2 or y2.shape[0] != M or y2.shape[1] != N or y2.stride(1) != 1:
            raise EmaError(EMA_ERR_SHAPE, "ema_quantized_matmul", "out must be a [M, N] view with unit column stride")
    _check(lib().ema_quantized_matmul(_stream(stream), _ptr(x2), x2.stride(0), _ptr(w), _ptr(scales), _ptr(biases),
                                      _ptr(y2), y2.stride(0), M, N, K, group_size, bits, dtypes[x.dtype]),
           "ema_quantized_matmul")
    return y2.reshape(x.shape[:-1] + (N,)) if out is None else y2


class PagedCache:
    """Pool of K/V pages shared by many sequences: [n_pages, Hkv, page_size, D], bf16 or FP8
    (E4M3 codes with ``k_exp``/``v_exp`` int8 [n_pages, Hkv, page_size, D/64] exponents, as
    StaticCache's), page_size a power of two of at least 16.

    A page table int32 [B, cols] names each sequence's pages in order: position p lies in slot
    p % page_size of page table[b, p // page_size]. Entries outside [0, n_pages) are never
    followed: nothing is written there and their positions read as zero rows.

    bf16 ``k``/``v`` may be views with any page, head and position strides (multiples of 8
    elements, D contiguous, both alike), e.g. ``pool.transpose(1, 2)`` of a
    [n_pages, page_size, Hkv, D] tensor.
    """

    def __init__(self, n_pages: int, n_kv_heads: int, page_size: int, head_dim: int, device="cuda", k=None, v=None,
                 dtype="bf16", k_exp=None, v_exp=None):
        import torch

        op = "PagedCache"
        shape = (n_pages, n_kv_heads, page_size, head_dim)
        if dtype not in ("bf16", "fp8"):
            raise ValueError(f"unknown page dtype {dtype!r} (bf16 or fp8)")
        want = torch.bfloat16 if dtype == "bf16" else torch.uint8
        self.k = k if k is not None else torch.zeros(shape, dtype=want, device=device)
        self.v = v if v is not None else torch.zeros(shape, dtype=want, device=device)
        for name, t in (("k", self.k), ("v", self.v)):
            if t.dtype != want or tuple(t.shape) != shape or t.stride(3) != 1:
                raise EmaError(EMA_ERR_SHAPE, op, f"{name} must be {want} {shape}, its last axis contiguous")
        if self.k.stride() != self.v.stride() or self.k.device != self.v.device:
            raise EmaError(EMA_ERR_SHAPE, op, "k and v differ in strides or device")
        self.desc = KvCacheDesc()
        self.dtype = dtype
        self.k_exp = self.v_exp = None
        if dtype == "bf16":
            _check(lib().ema_kvcache_init(ctypes.byref(self.desc), _ptr(self.k), _ptr(self.v), *shape),
                   "ema_kvcache_init")
        else:
            # (on the codes' device, whose index is all that the calls compare with)
            eshape, dev = shape[:3] + (head_dim // 64,), self.k.device
            self.k_exp = k_exp if k_exp is not None else torch.zeros(eshape, dtype=torch.int8, device=dev)
            self.v_exp = v_exp if v_exp is not None else torch.zeros(eshape, dtype=torch.int8, device=dev)
            for name, t in (("k_exp", self.k_exp), ("v_exp", self.v_exp)):
                if t.dtype != torch.int8 or tuple(t.shape) != eshape or not t.is_contiguous():
                    raise EmaError(EMA_ERR_SHAPE, op, f"{name} must be contiguous int8 {eshape}")
                if t.device != dev:
                    raise EmaError(EMA_ERR_INVALID_ARG, op, f"{name} is on {t.device}, the codes on {dev}")
            _check(lib().ema_kvcache_init_fp8(ctypes.byref(self.desc), _ptr(self.k), _ptr(self.v), _ptr(self.k_exp),
                                              _ptr(self.v_exp), *shape, 0), "ema_kvcache_init_fp8")
        self.desc.stride_batch, self.desc.stride_head, self.desc.stride_pos = self.k.stride()[:3]
        self.desc_ref = ctypes.byref(self.desc)
        self.device_index = self.k.get_device()

    @property
    def n_pages(self) -> int:
        return self.desc.batch

    @property
    def page_size(self) -> int:
        return self.desc.capacity

    def memory_bytes(self) -> int:
        out = ctypes.c_uint64()
        _check(lib().ema_kvcache_memory_bytes(ctypes.byref(self.desc), ctypes.byref(out)), "ema_kvcache_memory_bytes")
        return out.value


def _want(op: str, name: str, t, dtype, shape, device: int) -> None:
    """A contiguous tensor of the given dtype and shape on the given device (an index; -1: CPU)."""
    if t.shape != shape or t.dtype is not dtype or not t.is_contiguous():
        raise EmaError(EMA_ERR_SHAPE, op, f"{name} must be a contiguous {dtype} tensor {tuple(shape)}, not "
                                          f"{t.dtype} {tuple(t.shape)} with strides {t.stride()}")
    if t.get_device() != device:
        raise EmaError(EMA_ERR_INVALID_ARG, op, f"{name} is on {t.device}, not on device {device}")


def _refuse(op: str, device: int, *wanted) -> None:
    """Raises for the first of (name, tensor, dtype, shape) that is not as wanted."""
    for name, t, dtype, shape in wanted:
        if t is not None:
            _want(op, name, t, dtype, shape, device)
    raise EmaError(EMA_ERR_SHAPE, op, "arguments that do not belong together")


def _no_tensor(op: str, needed: dict, optional: dict) -> None:
    """Raises for the first argument that is no tensor; an optional one may be None."""
    import torch

    for name, t in (needed | optional).items():
        if not isinstance(t, torch.Tensor) and not (t is None and name in optional):
            raise EmaError(EMA_ERR_INVALID_ARG, op, f"{name} must be a tensor, not {type(t).__name__}")


def _elsewhere(device: int, call, *args) -> int:
    """call(*args) with the pool's device, which is not the current one, made current."""
    import torch

    if device < 0:
        raise EmaError(EMA_ERR_INVALID_ARG, call.__name__, "the pages are not on a GPU")
    with torch.cuda.device(device):
        return call(*args)


def _on(stream):
    """What a call allocates for itself belongs to the stream that it is given: filled and reused in
    that stream's order, not in the current one's."""
    import contextlib

    import torch

    return contextlib.nullcontext() if stream is None else torch.cuda.stream(stream)


def paged_append(qkv, q_norm_w, k_norm_w, eps, theta, offsets, n_heads, cache: PagedCache, table, q_starts=None,
                 flags=0, q_out=None, prefix_len=None, stream=None):
    """Norm, rotation and append of a ragged batch (ema_paged_append): qkv [n, (Hq+2Hkv)*D] bf16,
    offsets int32 [B] (position of each sequence's first row), table int32 [B, cols], q_starts
    int32 [B+1] (None: n / B rows each); prefix_len int32 [1]: a shared prefix's positions, which
    the rotation counts before the sequences' own. Returns q_out [n, Hq, D]."""
    import torch

    # one expression for what is right (2 us for the five to seven tensors of a call: the smallest
    # calls are bound by the host), the tensor to name looked for only when it is not
    op, bf, i32, dev = "ema_paged_append", torch.bfloat16, torch.int32, cache.device_index
    D, F = cache.desc.head_dim, n_heads + 2 * cache.desc.n_kv_heads
    try:
        B, cols = table.shape if table.dim() == 2 else (-1, -1)
        n = qkv.shape[0] if qkv.dim() else -1
        if q_out is None and n >= 0:
            with _on(stream):
                q_out = torch.empty((n, n_heads, D), dtype=bf, device=qkv.device)
        if not (table.dtype is i32 and table.is_contiguous() and table.get_device() == dev
                and offsets.dtype is i32 and offsets.shape == (B,) and offsets.is_contiguous() and offsets.get_device() == dev
                and qkv.dtype is bf and qkv.shape == (n, F * D) and qkv.is_contiguous() and qkv.get_device() == dev
                and q_out.dtype is bf and q_out.shape == (n, n_heads, D) and q_out.is_contiguous() and q_out.get_device() == dev
                and (q_norm_w is None or (q_norm_w.dtype is bf and q_norm_w.shape == (D,) and q_norm_w.is_contiguous()
                                          and q_norm_w.get_device() == dev))
                and (k_norm_w is None or (k_norm_w.dtype is bf and k_norm_w.shape == (D,) and k_norm_w.is_contiguous()
                                          and k_norm_w.get_device() == dev))
                and (q_starts is None or (q_starts.dtype is i32 and q_starts.shape == (B + 1,) and q_starts.is_contiguous()
                                          and q_starts.get_device() == dev))
                and (prefix_len is None or (prefix_len.dtype is i32 and prefix_len.shape == (1,)
                                            and prefix_len.get_device() == dev))):
            _refuse(op, dev, ("table", table, i32, (B, cols)), ("offsets", offsets, i32, (B,)),
                    ("qkv", qkv, bf, (n, F * D)), ("q_out", q_out, bf, (n, n_heads, D)), ("q_norm_w", q_norm_w, bf, (D,)),
                    ("k_norm_w", k_norm_w, bf, (D,)), ("q_starts", q_starts, i32, (B + 1,)),
                    ("prefix_len", prefix_len, i32, (1,)))
    except AttributeError:
        _no_tensor(op, dict(table=table, qkv=qkv, offsets=offsets),
                   dict(q_norm_w=q_norm_w, k_norm_w=k_norm_w, q_starts=q_starts, prefix_len=prefix_len, q_out=q_out))
        raise
    args = (torch._C._cuda_getCurrentRawStream(dev) if stream is None and dev >= 0 else _stream(stream), qkv.data_ptr(),
            _ptr(q_norm_w), _ptr(k_norm_w), eps, theta, _ptr(q_starts), offsets.data_ptr(), _ptr(prefix_len), B, n,
            n_heads, flags, q_out.data_ptr(), cache.desc_ref, table.data_ptr(), cols)
    call = lib().ema_paged_append
    rc = call(*args) if torch._C._cuda_getDevice() == dev else _elsewhere(dev, call, *args)
    if rc:
        _check(rc, op)
    return q_out


def paged_workspace_size(batch, n_rows, n_heads, n_kv_heads, head_dim, max_q, max_len, max_prefix=0) -> int:
    out = ctypes.c_uint64()
    _check(lib().ema_paged_workspace_size(batch, n_rows, n_heads, n_kv_heads, head_dim, max_q, max_len, max_prefix,
                                          ctypes.byref(out)), "ema_paged_workspace_size")
    return out.value


def paged_workspace(batch, n_rows, n_heads, n_kv_heads, head_dim, max_q, max_len, max_prefix=0, device="cuda"):
    """A workspace for paged_attention and (with max_prefix) prefix_attention: zero-filled, as the
    arrival counters at its start must be before the first call; reusable on one stream."""
    import torch

    n = paged_workspace_size(batch, n_rows, n_heads, n_kv_heads, head_dim, max_q, max_len, max_prefix)
    return torch.zeros(n, dtype=torch.uint8, device=device)


def _paged_args(op, q, cache, table, lengths, q_starts, max_q, max_len, scale, out, workspace, stream, shared=False,
                max_prefix=0, prefix_table=None, prefix_len=None):
    """Checks the tensors of an attention call (see paged_append), with shared those of a prefix too, and
    returns (stream, B, n, Hq, cols, max_q, scale, out, workspace)."""
    import torch

    bf, i32, dev = torch.bfloat16, torch.int32, cache.device_index
    D = cache.desc.head_dim
    try:
        B, cols = table.shape if table.dim() == 2 else (-1, -1)
        n, Hq = q.shape[:2] if q.dim() == 3 else (-1, -1)
        if q_starts is None:
            max_q = -(-n // B) if B > 0 else 0
        elif max_q is None:
            max_q = n
        if out is None and n >= 0:
            with _on(stream):
                out = torch.empty((n, Hq * D), dtype=bf, device=q.device)
        if not (table.dtype is i32 and table.is_contiguous() and table.get_device() == dev
                and lengths.dtype is i32 and lengths.shape == (B,) and lengths.is_contiguous() and lengths.get_device() == dev
                and q.dtype is bf and q.shape == (n, Hq, D) and q.is_contiguous() and q.get_device() == dev
                and out.dtype is bf and out.shape == (n, Hq * D) and out.is_contiguous() and out.get_device() == dev
                and (q_starts is None or (q_starts.dtype is i32 and q_starts.shape == (B + 1,) and q_starts.is_contiguous()
                                          and q_starts.get_device() == dev))
                and (workspace is None or (workspace.dtype is torch.uint8 and workspace.is_contiguous()
                                           and workspace.get_device() == dev))
                and (not shared or (prefix_table.dtype is i32 and prefix_table.dim() == 1
                                    and prefix_table.is_contiguous() and prefix_table.get_device() == dev
                                    and prefix_len.dtype is i32 and prefix_len.shape == (1,)
                                    and prefix_len.get_device() == dev))):
            _refuse(op, dev, ("table", table, i32, (B, cols)), ("lengths", lengths, i32, (B,)), ("q", q, bf, (n, Hq, D)),
                    ("out", out, bf, (n, Hq * D)), ("q_starts", q_starts, i32, (B + 1,)),
                    ("workspace", workspace, torch.uint8, workspace.shape if workspace is not None else ()),
                    ("prefix_table", prefix_table, i32, (prefix_table.numel(),) if shared else ()),
                    ("prefix_len", prefix_len, i32, (1,)))
    except AttributeError:
        _no_tensor(op, dict(table=table, lengths=lengths, q=q,
                            **(dict(prefix_table=prefix_table, prefix_len=prefix_len) if shared else {})),
                   dict(q_starts=q_starts, out=out, workspace=workspace))
        raise
    if workspace is None:
        with _on(stream):
            workspace = paged_workspace(B, n, Hq, cache.desc.n_kv_heads, D, max_q, max_len, max_prefix, device=q.device)
    raw = torch._C._cuda_getCurrentRawStream(dev) if stream is None and dev >= 0 else _stream(stream)
    return raw, B, n, Hq, cols, max_q, 1.0 / math.sqrt(D) if scale is None else scale, out, workspace


def _paged_call(op: str, cache, call, *args) -> None:
    import torch

    dev = cache.device_index
    rc = call(*args) if torch._C._cuda_getDevice() == dev else _elsewhere(dev, call, *args)
    if rc:
        _check(rc, op)


def paged_attention(q, cache: PagedCache, table, lengths, max_len, q_starts=None, max_q=None, causal=True, scale=None,
                    out=None, workspace=None, stream=None):
    """Attention of a ragged batch over its pages (ema_paged_attention): q [n, Hq, D] bf16, lengths
    int32 [B] (positions held, the call's rows included), table int32 [B, cols]; max_len and
    max_q are host bounds of the lengths and of a sequence's rows. Returns out [n, Hq * D]."""
    op = "ema_paged_attention"
    raw, B, n, Hq, cols, max_q, scale, out, workspace = _paged_args(op, q, cache, table, lengths, q_starts, max_q,
                                                                    max_len, scale, out, workspace, stream)
    _paged_call(op, cache, lib().ema_paged_attention, raw, q.data_ptr(), cache.desc_ref, table.data_ptr(), cols,
                _ptr(q_starts), lengths.data_ptr(), B, n, max_q, max_len, Hq, scale, EMA_PREFILL_CAUSAL if causal else 0,
                out.data_ptr(), workspace.data_ptr(), workspace.numel())
    return out


def prefix_attention(q, cache: PagedCache, prefix_table, prefix_len, max_prefix, table, lengths, max_len,
                     q_starts=None, max_q=None, scale=None, out=None, workspace=None, stream=None):
    """Causal attention where every sequence's own pages continue one shared prefix
    (ema_prefix_attention): prefix_table int32 [cols], prefix_len int32 [1] (its positions,
    max_prefix a host bound); table and lengths are of the sequences' own positions, the rest as
    in paged_attention. The prefix is held once, and a long one read once per 128 packed rows of a kv
    head (FP8: 32). Returns out [n, Hq * D]."""
    op = "ema_prefix_attention"
    raw, B, n, Hq, cols, max_q, scale, out, workspace = _paged_args(op, q, cache, table, lengths, q_starts, max_q,
                                                                    max_len, scale, out, workspace, stream, True,
                                                                    max_prefix, prefix_table, prefix_len)
    _paged_call(op, cache, lib().ema_prefix_attention, raw, q.data_ptr(), cache.desc_ref, prefix_table.data_ptr(),
                prefix_table.numel(), prefix_len.data_ptr(), max_prefix, table.data_ptr(), cols, _ptr(q_starts),
                lengths.data_ptr(), B, n, max_q, max_len, Hq, scale, out.data_ptr(), workspace.data_ptr(),
                workspace.numel())
    return out


# ---- around the recurrent scans: convolution, state space scan, norms


# Each call decides in one expression whether its tensors are right (2 us for the eight tensors of a
# convolution: the smallest calls are bound by the host), and looks for the one to name only when they
# are not.
_torch = None
_act_codes: dict = {}


def _load_torch():
    global _torch
    import torch

    _act_codes.update({torch.bfloat16: EMA_DTYPE_BF16, torch.float16: EMA_DTYPE_F16, torch.float32: EMA_DTYPE_F32})
    _torch = torch
    lib()
    return torch


def _act_code(op: str, t):
    """EMA_DTYPE_* of an activation tensor."""
    _torch or _load_torch()
    code = _act_codes.get(t.dtype)
    if code is None:
        raise EmaError(EMA_ERR_INVALID_ARG, op, f"unsupported activation dtype {t.dtype}")
    return code


def _want_rows(op: str, name: str, t, dtype, shape, device: int) -> None:
    """A [n, ...] tensor of the given dtype and shape whose rows are contiguous."""
    if t.shape != shape or t.dtype is not dtype:
        raise EmaError(EMA_ERR_SHAPE, op, f"{name} must be a {dtype} tensor {tuple(shape)}, not {t.dtype} {tuple(t.shape)}")
    if t.get_device() != device:
        raise EmaError(EMA_ERR_INVALID_ARG, op, f"{name} is on {t.device}, not on device {device}")
    if not _rows_whole(t):
        raise EmaError(EMA_ERR_SHAPE, op, f"a row of {name} must be contiguous, not strided {t.stride()}")


def _rows_whole(t) -> bool:
    width = 1
    for size, stride in zip(reversed(t.shape[1:]), reversed(t.stride()[1:])):
        if stride != width and size != 1:
            return False
        width *= size
    return True


def _name_batch(op: str, dev: int, batch, starts, offsets, slots) -> None:
    """Raises for the first of the int32 tensors that describe the sequences that is not right."""
    for name, t, size in (("starts", starts, batch + 1), ("offsets", offsets, batch), ("slots", slots, batch)):
        if t is not None:
            _want(op, name, t, _torch.int32, (size,), dev)


def _empty(stream, shape, dtype, device):
    with _on(stream):
        return _torch.empty(shape, dtype=dtype, device=device)


def _not_on_gpu(op: str):
    raise EmaError(EMA_ERR_INVALID_ARG, op, "the tensors are not on a GPU")


def causal_conv(x, weight, bias=None, state=None, starts=None, offsets=None, slots=None, batch=None, max_rows=None,
                silu=True, out=None, stream=None):
    """Short causal convolution of each channel over its sequence's time (ema_causal_conv): x [n, C] (rows may
    be pieces of wider ones) in bf16, f16 or f32, weight [C, W] and bias [C] in the same type, W 2 to 4; state
    [n_slots, W-1, C], the inputs kept between calls, updated in place (None: start from zeros, keep nothing).
    starts int32 [B+1] (None: n / B rows each), offsets int32 [B] (position of the first row: at 0 a sequence
    starts from zeros), slots int32 [B] (None: slot b). Returns out [n, C]."""
    op = "ema_causal_conv"
    torch = _torch or _load_torch()
    i32 = torch.int32
    try:
        dtype, dev = x.dtype, x.get_device()
        (n, C), (ldx, sx) = x.shape, x.stride()
        W = weight.shape[1]
        if batch is None:
            batch = (starts.shape[0] - 1 if starts is not None else offsets.shape[0] if offsets is not None
                     else slots.shape[0] if slots is not None else state.shape[0] if state is not None else 1)
        if out is None:
            out = _empty(stream, (n, C), dtype, x.device)
        ldy, sy = out.stride()
        n_slots = 0 if state is None else state.shape[0]
        if not (dtype in _act_codes and (sx == 1 or C == 1) and (sy == 1 or C == 1)
                and out.dtype is dtype and out.shape == (n, C) and out.get_device() == dev
                and weight.dtype is dtype and weight.shape == (C, W) and weight.is_contiguous() and weight.get_device() == dev
                and (bias is None or (bias.dtype is dtype and bias.shape == (C,) and bias.is_contiguous()
                                      and bias.get_device() == dev))
                and (state is None or (state.dtype is dtype and state.shape == (n_slots, W - 1, C)
                                       and state.is_contiguous() and state.get_device() == dev))
                and (starts is None or (starts.dtype is i32 and starts.shape == (batch + 1,) and starts.is_contiguous()
                                        and starts.get_device() == dev))
                and (offsets is None or (offsets.dtype is i32 and offsets.shape == (batch,) and offsets.is_contiguous()
                                         and offsets.get_device() == dev))
                and (slots is None or (slots.dtype is i32 and slots.shape == (batch,) and slots.is_contiguous()
                                       and slots.get_device() == dev))):
            _act_code(op, x)
            _want_rows(op, "x", x, dtype, (n, C), dev)
            _want_rows(op, "out", out, dtype, (n, C), dev)
            _want(op, "weight", weight, dtype, (C, W), dev)
            for name, t, shape in (("bias", bias, (C,)), ("state", state, (n_slots, W - 1, C))):
                if t is not None:
                    _want(op, name, t, dtype, shape, dev)
            _name_batch(op, dev, batch, starts, offsets, slots)
    except (AttributeError, ValueError, IndexError):
        _no_tensor(op, dict(x=x, weight=weight),
                   dict(bias=bias, state=state, starts=starts, offsets=offsets, slots=slots, out=out))
        if x.dim() != 2 or weight.dim() != 2 or (out is not None and out.dim() != 2):
            raise EmaError(EMA_ERR_SHAPE, op, f"x must be [n, C] and weight [C, W], not {tuple(x.shape)}, {tuple(weight.shape)}")
        raise
    if dev < 0:
        _not_on_gpu(op)
    args = (torch._C._cuda_getCurrentRawStream(dev) if stream is None else stream.cuda_stream, x.data_ptr(), ldx if n > 1 else C, weight.data_ptr(),
            None if bias is None else bias.data_ptr(), None if starts is None else starts.data_ptr(),
            None if offsets is None else offsets.data_ptr(), None if slots is None else slots.data_ptr(), batch, n,
            n if max_rows is None else max_rows, C, W, EMA_CONV_SILU if silu else 0,
            None if state is None else state.data_ptr(), n_slots, out.data_ptr(), ldy if n > 1 else C,
            _act_codes[dtype])
    call = _lib.ema_causal_conv
    rc = call(*args) if torch._C._cuda_getDevice() == dev else _elsewhere(dev, call, *args)
    if rc:
        _check(rc, op)
    return out


def ssm_workspace_size(batch, n_rows, max_rows, n_heads, head_dim, d_state, n_groups, dtype=None) -> int:
    """Bytes with which ssm_scan splits every call of at most these bounds in time as it likes best (0: it splits
    none); dtype a torch type, bf16 by default."""
    _torch or _load_torch()
    out = ctypes.c_uint64()
    code = EMA_DTYPE_BF16 if dtype is None else _act_codes.get(dtype, 0)
    _check(lib().ema_ssm_workspace_size(batch, n_rows, max_rows, n_heads, head_dim, d_state, n_groups, code,
                                        ctypes.byref(out)), "ema_ssm_workspace_size")
    return out.value


def ssm_workspace(batch, n_rows, max_rows, n_heads, head_dim, d_state, n_groups, dtype=None, device="cuda"):
    """A workspace for ssm_scan (no initialisation needed), reusable on one stream."""
    size = ssm_workspace_size(batch, n_rows, max_rows, n_heads, head_dim, d_state, n_groups, dtype)
    return _torch.empty(size, dtype=_torch.uint8, device=device)


def ssm_scan(x, dt, B, C, A, state, D=None, dt_bias=None, starts=None, offsets=None, slots=None, batch=None,
             max_rows=None, softplus=True, dt_limit=(0.0, math.inf), out=None, workspace=None, stream=None):
    """Selective state space scan, one decay per head (ema_ssm_scan): x [n, H, P], dt [n, H], B and C [n, G, N]
    in bf16, f16 or f32 (rows may be pieces of wider ones); A (at most 0), D, dt_bias f32 [H]; state f32
    [n_slots, H, P, N], updated in place; starts, offsets, slots as in causal_conv; max_rows a host bound of a
    sequence's rows, by which the kernels are chosen: without starts n / B, with them n unless given, so give it
    for a ragged step of few rows each. workspace: a uint8 tensor (ssm_workspace) that long sequences are split over;
    None allocates one. Returns out [n, H, P]."""
    op = "ema_ssm_scan"
    torch = _torch or _load_torch()
    i32, f32 = torch.int32, torch.float32
    try:
        dtype, dev = x.dtype, x.get_device()
        (n, H, P), (ldx, sh, sp) = x.shape, x.stride()
        _, G, N = B.shape
        (ldb, sbg, sbn), (ldc, scg, scn), (lddt, sdt) = B.stride(), C.stride(), dt.stride()
        n_slots = state.shape[0]
        if batch is None:
            batch = (starts.shape[0] - 1 if starts is not None else offsets.shape[0] if offsets is not None
                     else slots.shape[0] if slots is not None else n_slots)
        if starts is None and batch > 0:
            max_rows = n // batch
        elif max_rows is None:
            max_rows = n
        if out is None:
            out = _empty(stream, (n, H, P), dtype, x.device)
        ldy, yh, yp = out.stride()
        if not (dtype in _act_codes and (sp == 1 or P == 1) and (sh == P or H == 1) and (yp == 1 or P == 1)
                and (yh == P or H == 1) and (sbn == 1 or N == 1) and (sbg == N or G == 1) and (scn == 1 or N == 1)
                and (scg == N or G == 1) and (sdt == 1 or H == 1)
                and out.dtype is dtype and out.shape == (n, H, P) and out.get_device() == dev
                and B.dtype is dtype and B.shape == (n, G, N) and B.get_device() == dev
                and C.dtype is dtype and C.shape == (n, G, N) and C.get_device() == dev
                and dt.dtype is dtype and dt.shape == (n, H) and dt.get_device() == dev
                and A.dtype is f32 and A.shape == (H,) and A.is_contiguous() and A.get_device() == dev
                and state.dtype is f32 and state.shape == (n_slots, H, P, N) and state.is_contiguous()
                and state.get_device() == dev
                and (D is None or (D.dtype is f32 and D.shape == (H,) and D.is_contiguous() and D.get_device() == dev))
                and (dt_bias is None or (dt_bias.dtype is f32 and dt_bias.shape == (H,) and dt_bias.is_contiguous()
                                         and dt_bias.get_device() == dev))
                and (starts is None or (starts.dtype is i32 and starts.shape == (batch + 1,) and starts.is_contiguous()
                                        and starts.get_device() == dev))
                and (offsets is None or (offsets.dtype is i32 and offsets.shape == (batch,) and offsets.is_contiguous()
                                         and offsets.get_device() == dev))
                and (slots is None or (slots.dtype is i32 and slots.shape == (batch,) and slots.is_contiguous()
                                       and slots.get_device() == dev))
                and (workspace is None or (workspace.dtype is torch.uint8 and workspace.is_contiguous()
                                           and workspace.get_device() == dev))):
            _act_code(op, x)
            for name, t, shape in (("x", x, (n, H, P)), ("out", out, (n, H, P)), ("B", B, (n, G, N)), ("C", C, (n, G, N)),
                                   ("dt", dt, (n, H))):
                _want_rows(op, name, t, dtype, shape, dev)
            for name, t, shape in (("A", A, (H,)), ("D", D, (H,)), ("dt_bias", dt_bias, (H,)),
                                   ("state", state, (n_slots, H, P, N))):
                if t is not None or name == "A":
                    _want(op, name, t, f32, shape, dev)
            if workspace is not None:
                _want(op, "workspace", workspace, torch.uint8, workspace.shape, dev)
            _name_batch(op, dev, batch, starts, offsets, slots)
    except (AttributeError, ValueError, IndexError):
        _no_tensor(op, dict(x=x, dt=dt, B=B, C=C, A=A, state=state),
                   dict(D=D, dt_bias=dt_bias, starts=starts, offsets=offsets, slots=slots, out=out, workspace=workspace))
        for name, t, dims in (("x", x, 3), ("dt", dt, 2), ("B", B, 3), ("C", C, 3), ("out", out, 3)):
            if t is not None and t.dim() != dims:
                raise EmaError(EMA_ERR_SHAPE, op, f"{name} must have {dims} dimensions, not {tuple(t.shape)}")
        raise
    if workspace is None and dev >= 0 and n:
        size = ssm_workspace_size(batch, n, max_rows, H, P, N, G, dtype)
        workspace = _empty(stream, (size,), torch.uint8, x.device)
    size = 0 if workspace is None else workspace.numel()
    if dev < 0:
        _not_on_gpu(op)
    args = (torch._C._cuda_getCurrentRawStream(dev) if stream is None else stream.cuda_stream, x.data_ptr(), ldx if n > 1 else H * P, dt.data_ptr(),
            lddt if n > 1 else H, B.data_ptr(), ldb if n > 1 else G * N, C.data_ptr(), ldc if n > 1 else G * N,
            A.data_ptr(), None if D is None else D.data_ptr(), None if dt_bias is None else dt_bias.data_ptr(),
            dt_limit[0], dt_limit[1], None if starts is None else starts.data_ptr(),
            None if offsets is None else offsets.data_ptr(), None if slots is None else slots.data_ptr(), batch, n,
            max_rows, H, P, G, N, EMA_SSM_SOFTPLUS if softplus else 0, state.data_ptr(), n_slots, out.data_ptr(),
            ldy if n > 1 else H * P, _act_codes[dtype], workspace.data_ptr() if size else None, size)
    call = _lib.ema_ssm_scan
    rc = call(*args) if torch._C._cuda_getDevice() == dev else _elsewhere(dev, call, *args)
    if rc:
        _check(rc, op)
    return out


def gated_norm(x, gate, weight, eps, group=None, gate_first=False, sigmoid=False, unit_offset=False, out=None,
               stream=None):
    """RMSNorm of each `group` values (default: all) of the rows x [n, dim], gated (ema_gated_norm): norm(x) * w *
    act(gate), or norm(x * act(gate)) * w with gate_first; act is silu, or sigmoid. gate [n, dim] or None;
    weight [dim], [group] (one for all groups) or None; unit_offset: 1 + w multiplies. Rows of x, gate and out
    may be pieces of wider ones; out may be x or gate. Returns out [n, dim]."""
    op = "ema_gated_norm"
    torch = _torch or _load_torch()
    try:
        dtype, dev = x.dtype, x.get_device()
        (n, dim), (ldx, sx) = x.shape, x.stride()
        if group is None:
            group = dim
        if out is None:
            out = _empty(stream, (n, dim), dtype, x.device)
        ldy, sy = out.stride()
        ldg, sg = (0, 1) if gate is None else gate.stride()
        flags = ((EMA_NORM_GATE_FIRST if gate_first else 0) | (EMA_NORM_GATE_SIGMOID if sigmoid else 0)
                 | (EMA_NORM_UNIT_OFFSET if unit_offset else 0))
        width = dim
        if weight is not None and group != dim and weight.shape == (group,):
            flags |= EMA_NORM_SHARED_WEIGHT
            width = group
        if not (dtype in _act_codes and (sx == 1 or dim == 1) and (sy == 1 or dim == 1) and (sg == 1 or dim == 1)
                and out.dtype is dtype and out.shape == (n, dim) and out.get_device() == dev
                and (gate is None or (gate.dtype is dtype and gate.shape == (n, dim) and gate.get_device() == dev))
                and (weight is None or (weight.dtype is dtype and weight.shape == (width,) and weight.is_contiguous()
                                        and weight.get_device() == dev))):
            _act_code(op, x)
            for name, t in (("x", x), ("out", out), ("gate", gate)):
                if t is not None:
                    _want_rows(op, name, t, dtype, (n, dim), dev)
            if weight is not None:
                _want(op, "weight", weight, dtype, (width,), dev)
    except (AttributeError, ValueError):
        _no_tensor(op, dict(x=x), dict(gate=gate, weight=weight, out=out))
        for name, t in (("x", x), ("gate", gate), ("out", out)):
            if t is not None and t.dim() != 2:
                raise EmaError(EMA_ERR_SHAPE, op, f"{name} must be [n, dim], not {tuple(t.shape)}")
        raise
    if dev < 0:
        _not_on_gpu(op)
    args = (torch._C._cuda_getCurrentRawStream(dev) if stream is None else stream.cuda_stream, x.data_ptr(), ldx if n > 1 else dim,
            None if gate is None else gate.data_ptr(), ldg if n > 1 else dim,
            None if weight is None else weight.data_ptr(), eps, n, dim, group, flags, out.data_ptr(),
            ldy if n > 1 else dim, _act_codes[dtype])
    call = _lib.ema_gated_norm
    rc = call(*args) if torch._C._cuda_getDevice() == dev else _elsewhere(dev, call, *args)
    if rc:
        _check(rc, op)
    return out


def residual_norm(branch, residual, pre_weight, eps, post_weight=None, gate=None, scale=1.0, unit_offset=False,
                  out=None, stream=None):
    """The norm after one block and the one before the next (ema_residual_norm): residual += scale * gate *
    norm(branch) * post_weight in place (post_weight None: the branch as it is), then returns out =
    norm(residual) * pre_weight (of the sum before it is rounded). branch [n, dim] in bf16, f16 or f32, residual
    [n, dim] in the same type or f32; gate [n, dim], [dim] (one for all rows) or None; pre_weight None: the
    residual stream alone (returns None). Rows may be pieces of wider ones; out may be branch."""
    op = "ema_residual_norm"
    torch = _torch or _load_torch()
    f32 = torch.float32
    try:
        dtype, dev, rtype = branch.dtype, branch.get_device(), residual.dtype
        (n, dim), (ldx, sx), (ldr, sr) = branch.shape, branch.stride(), residual.stride()
        if out is None and pre_weight is not None:
            out = _empty(stream, (n, dim), dtype, branch.device)
        ldo, so = (0, 1) if out is None else out.stride()
        one = gate is not None and gate.dim() == 1  # a row for all
        ldg, sg = (0, 1) if gate is None or one else gate.stride()
        if not (dtype in _act_codes and (rtype is dtype or rtype is f32) and (sx == 1 or dim == 1)
                and (sr == 1 or dim == 1) and (so == 1 or dim == 1) and (sg == 1 or dim == 1)
                and residual.shape == (n, dim) and residual.get_device() == dev
                and (out is None or (out.dtype is dtype and out.shape == (n, dim) and out.get_device() == dev))
                and (gate is None or (gate.dtype is dtype and gate.shape == ((dim,) if one else (n, dim))
                                      and (not one or gate.is_contiguous()) and gate.get_device() == dev))
                and (pre_weight is None or (pre_weight.dtype is dtype and pre_weight.shape == (dim,)
                                            and pre_weight.is_contiguous() and pre_weight.get_device() == dev))
                and (post_weight is None or (post_weight.dtype is dtype and post_weight.shape == (dim,)
                                             and post_weight.is_contiguous() and post_weight.get_device() == dev))):
            _act_code(op, branch)
            _want_rows(op, "branch", branch, dtype, (n, dim), dev)
            _want_rows(op, "residual", residual, f32 if rtype is f32 else dtype, (n, dim), dev)
            if out is not None:
                _want_rows(op, "out", out, dtype, (n, dim), dev)
            if gate is not None:
                (_want if one else _want_rows)(op, "gate", gate, dtype, (dim,) if one else (n, dim), dev)
            for name, w in (("pre_weight", pre_weight), ("post_weight", post_weight)):
                if w is not None:
                    _want(op, name, w, dtype, (dim,), dev)
    except (AttributeError, ValueError):
        _no_tensor(op, dict(branch=branch, residual=residual),
                   dict(pre_weight=pre_weight, post_weight=post_weight, gate=gate, out=out))
        for name, t in (("branch", branch), ("residual", residual), ("gate", gate), ("out", out)):
            if t is not None and t.dim() != 2 and not (name == "gate" and t.dim() == 1):
                raise EmaError(EMA_ERR_SHAPE, op, f"{name} must be [n, dim], not {tuple(t.shape)}")
        raise
    if n <= 1:
        ldx = ldr = ldo = dim
        ldg = 0
    if dev < 0:
        _not_on_gpu(op)
    args = (torch._C._cuda_getCurrentRawStream(dev) if stream is None else stream.cuda_stream, branch.data_ptr(), ldx,
            None if post_weight is None else post_weight.data_ptr(), None if gate is None else gate.data_ptr(), ldg,
            scale, residual.data_ptr(), ldr, EMA_DTYPE_F32 if rtype is f32 else _act_codes[dtype],
            None if pre_weight is None else pre_weight.data_ptr(), eps, n, dim,
            EMA_NORM_UNIT_OFFSET if unit_offset else 0, None if out is None else out.data_ptr(), ldo,
            _act_codes[dtype])
    call = _lib.ema_residual_norm
    rc = call(*args) if torch._C._cuda_getDevice() == dev else _elsewhere(dev, call, *args)
    if rc:
        _check(rc, op)
    return out
