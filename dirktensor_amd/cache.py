"""A quantised key/value cache and the attention that reads it, on the HIP path: every call goes to
libdirktensor_amd.so; nothing here computes.

    KVCache(slots, capacity, n_heads, format="int8" | "fp8" | "bf16" | "fp4")
        append(K, V)              quantises rows as they are written behind what the slots hold
        read(starts, count)       the rows as the values they stand for
        truncate(lengths)         shortens slots (0: free for another sequence)
    cached_attention(Q, cache, scale, prefix=None) -> FlashAttentionResult
        attention of the newest tokens over a cache, optionally behind a prefix shared by the whole batch (the
        cached form of flash_attention_forward, FlashAttention.h:15-21)

A step of generation appends the new tokens' keys and values and attends with their queries; several answers to one
prompt hold the prompt once, in a cache of one slot that is passed as ``prefix``.
"""

from __future__ import annotations

import ctypes
from typing import Optional

import numpy as np

from . import _capi as C
from ._workspace import kept_workspace, new_workspace
from .attention import Context, FlashAttentionResult, _is_torch, _mode_of, _stream_of, default_context, torch

_FORMATS = {"int8": C.DT_KV_INT8, "fp8": C.DT_KV_FP8, "bf16": C.DT_KV_BF16, "fp4": C.DT_KV_FP4}


def _address(a: np.ndarray) -> int:
    """Where a contiguous array's values lie (``a.ctypes`` builds an object for that)."""
    try:
        return ctypes.addressof(ctypes.c_char.from_buffer(a))
    except (TypeError, ValueError):  # read-only or empty
        return a.ctypes.data


def _per_row(x, B: int, name: str):
    """A per-row argument as B int32 values in host memory and their address (None: NULL)."""
    if x is None:
        return None, None
    if type(x) is np.ndarray and x.dtype == np.int32 and x.shape == (B,) and x.flags.c_contiguous:
        return x, _address(x)
    a = np.asarray(x.cpu() if _is_torch(x) else x)
    if a.dtype.kind not in "iu" or a.shape != (B,):
        raise ValueError(f"{name} must be {B} whole numbers, got {a.dtype} of shape {a.shape}")
    if a.size and (a.max() > 0x7FFFFFFF or a.min() < -0x80000000):
        raise ValueError(f"{name} holds a number beyond 32 bits")
    a = np.ascontiguousarray(a, dtype=np.int32)
    return a, _address(a)


def _rows_of(x):
    """[B, T, H, 128] as rows of one token stride: the tensor itself where its strides allow that, else a copy."""
    B, T, H, D = x.shape
    if x.is_contiguous() and x.data_ptr() % 16 == 0:
        return x, H * D
    if x.stride(3) == 1 and x.stride(2) == D or (H == 1 and x.stride(3) == 1):
        ld = x.stride(1) if T > 1 else (x.stride(0) if B > 1 else H * D)
        if ((B == 1 or x.stride(0) == T * ld) and ld >= H * D and ld * x.element_size() % 16 == 0
                and x.data_ptr() % 16 == 0):
            return x, ld
    x = x.contiguous()
    if x.data_ptr() % 16:
        x = x.clone()
    return x, H * D


class KVCache:
    """Keys and values of ``slots`` sequences of at most ``capacity`` tokens, ``n_heads`` heads of 128 values each,
    held in ``format``: "int8" (one scale a token and head), "fp8" (e4m3, scaled by a power of two), "bf16" or
    "fp4" (e2m1, each 32 values scaled by a power of two; half the bytes of the 8-bit formats).

    A row with an infinity or a NaN reads back as NaN and gives NaN to the queries that see it. The lengths live on the
    host and move when a call is made; calls on one cache must be ordered on their streams, except calls that only
    read. A call captured into a graph repeats the positions it was captured with.
    """

    def __init__(self, slots: int, capacity: int, n_heads: int = C.N_HEADS, *, format: str = "int8",
                 ctx: Optional[Context] = None):
        self.handle = None
        if format not in _FORMATS:
            raise ValueError(f"unknown cache format {format!r}: expected one of {sorted(_FORMATS)}")
        self.ctx = ctx or default_context(torch.cuda.current_device() if torch is not None and torch.cuda.is_available() else 0)
        self.slots, self.capacity, self.n_heads, self.format = int(slots), int(capacity), int(n_heads), format
        h = ctypes.c_void_p()
        C.call("dt_kv_cache_create", self.ctx.handle, self.slots, self.capacity, self.n_heads, C.HEAD_DIM,
               _FORMATS[format], ctypes.byref(h))
        self.handle = h
        self._device = torch.device("cuda", self.ctx.device) if torch is not None else None

    def close(self) -> None:
        if getattr(self, "handle", None):
            C.lib().dt_kv_cache_destroy(self.handle)
            self.handle = None

    def __del__(self):  # pragma: no cover - interpreter teardown order
        try:
            self.close()
        except Exception:
            pass

    def _live(self):
        if not self.handle:
            raise RuntimeError("the cache is closed")
        if not self.ctx.handle:
            raise RuntimeError("the cache's context is closed")
        return self.handle

    @property
    def lengths(self) -> np.ndarray:
        """The tokens held by each slot."""
        out = np.empty(self.slots, np.int32)
        C.call("dt_kv_cache_lengths", self._live(), out.ctypes.data)
        return out

    def truncate(self, lengths, *, slots=None) -> None:
        """Shortens the slots (None: the first len(lengths)) to ``lengths``, at most what they hold."""
        B = len(lengths)
        n, n_p = _per_row(lengths, B, "lengths")
        s, s_p = _per_row(slots, B, "slots")
        C.call("dt_kv_cache_truncate", self._live(), B, s_p, n_p)

    def _check_device(self, *tensors) -> None:
        for t in tensors:
            if not t.is_cuda:
                raise ValueError("torch inputs must be on a ROCm device; use numpy arrays for host memory")
            if t.device.index != self.ctx.device:
                raise ValueError(f"a tensor is on {t.device}, the cache on cuda:{self.ctx.device}")

    def append(self, K, V, *, slots=None, counts=None) -> None:
        """Writes the rows of K and V [B, T, n_heads, 128] (both fp32 or both bf16; torch device tensors, views of a
        projection's output among them, or numpy arrays) behind what the B slots hold: slots[b], distinct, or 0 .. B-1.
        With ``counts`` batch row b appends its first counts[b] tokens. Raises DTError where a slot has no room."""
        shape = K.shape
        if shape != V.shape or len(shape) != 4 or shape[2] != self.n_heads or shape[3] != C.HEAD_DIM:
            raise ValueError(f"K and V must share a shape [B, T, {self.n_heads}, {C.HEAD_DIM}], got {tuple(shape)}, "
                             f"{tuple(V.shape)}")
        if _is_torch(K) != _is_torch(V) or K.dtype != V.dtype:
            raise TypeError("K and V must be of one kind and dtype")
        B, T = shape[0], shape[1]
        dtype = _mode_of(K, None)
        s, s_p = _per_row(slots, B, "slots")
        n, n_p = _per_row(counts, B, "counts")
        if _is_torch(K):
            self._check_device(K, V)
            (K, ldk), (V, ldv) = _rows_of(K), _rows_of(V)
            C.call("dt_kv_cache_append", self._live(), K.data_ptr(), V.data_ptr(), B, T, ldk, ldv, s_p, n_p, dtype,
                   C.DT_MEM_DEVICE, _stream_of(K))
            return
        K, V = np.ascontiguousarray(K), np.ascontiguousarray(V)
        ld = self.n_heads * C.HEAD_DIM
        C.call("dt_kv_cache_append", self._live(), K.ctypes.data, V.ctypes.data, B, T, ld, ld, s_p, n_p, dtype,
               C.DT_MEM_HOST, None)

    def read(self, starts, count: int, *, slots=None, mode: str = "bf16", host: bool = False):
        """``count`` tokens from position starts[b] on of the slots (None: the first len(starts)), as K and V
        [B, count, n_heads, 128] of what the cache holds, in bf16 or fp32 by ``mode``: torch tensors on the cache's
        device, or with ``host`` numpy arrays (bf16 as uint16 bits)."""
        B, T = len(starts), int(count)
        dtype = _mode_of(None, mode)
        st, st_p = _per_row(starts, B, "starts")
        s, s_p = _per_row(slots, B, "slots")
        if B < 1 or T < 1:
            raise ValueError(f"nothing to read: {B} slots, {T} tokens")
        shape = (B, T, self.n_heads, C.HEAD_DIM)
        if host:
            K, V = (np.empty(shape, np.uint16 if dtype == C.DT_BF16 else np.float32) for _ in range(2))
            C.call("dt_kv_cache_read", self._live(), K.ctypes.data, V.ctypes.data, B, T, s_p, st_p, dtype,
                   C.DT_MEM_HOST, None)
            return K, V
        K = torch.empty(shape, dtype=torch.bfloat16 if dtype == C.DT_BF16 else torch.float32, device=self._device)
        V = torch.empty_like(K)
        C.call("dt_kv_cache_read", self._live(), K.data_ptr(), V.data_ptr(), B, T, s_p, st_p, dtype, C.DT_MEM_DEVICE,
               _stream_of(K))
        return K, V


def cached_attention(Q, cache: KVCache, scale: float, causal: bool = True, *, slots=None, counts=None,
                     prefix: Optional[KVCache] = None, prefix_slot: int = 0) -> FlashAttentionResult:
    """Attention of the newest tokens over what ``cache`` holds.

    Q: [B, T, H, 128], bf16 or fp32 (exact mode), a torch device tensor or a numpy array; H a multiple of the cache's
    heads, consecutive query heads sharing one. The tokens' own keys and values are appended first: token t of batch
    row b, whose slot holds L tokens, is at position L - counts[b] + t (counts: all T by default) and sees the keys up
    to it, or all L without ``causal``. Rows t >= counts[b], and rows that see no key, are the empty row (output 0,
    m = -inf, l = 0). ``slots`` names the slot of each batch row (0 .. B-1 by default; one may serve several).

    ``prefix``: a cache of the same format and heads whose slot ``prefix_slot`` holds tokens that come before every
    sequence of the batch (a shared prompt); every query sees all of them and they are read once for all.
    """
    if len(Q.shape) != 4:
        raise ValueError(f"expected [B, T, H, {C.HEAD_DIM}] queries, got {tuple(Q.shape)}")
    B, T, H, D = Q.shape
    dtype = _mode_of(Q, None)
    s, s_p = _per_row(slots, B, "slots")
    n, n_p = _per_row(counts, B, "counts")
    pre = prefix._live() if prefix is not None else None
    if _is_torch(Q):
        cache._check_device(Q)
        Q, ldq = _rows_of(Q)
        stream = _stream_of(Q)
        O = Q.new_empty((B, T, H, D))
        m = Q.new_empty((B, T, H), dtype=torch.float32)
        l = torch.empty_like(m)
        handle, q_p, o_p, m_p, l_p = cache._live(), Q.data_ptr(), O.data_ptr(), m.data_ptr(), l.data_ptr()

        def attend(ws_p, nbytes):
            return C.lib().dt_cached_attn_fwd(handle, q_p, o_p, m_p, l_p, B, T, H, D, ldq, float(scale), int(bool(causal)),
                                              s_p, n_p, pre, int(prefix_slot), ws_p, nbytes, dtype, C.DT_MEM_DEVICE, stream)

        kept = kept_workspace(cache.ctx.device, stream)
        if kept is not None:
            rc = attend(kept[0], kept[1])
            if rc == C.DT_OK:
                return FlashAttentionResult(O, m, l)
            if rc != C.DT_ERR_INVALID_ARG:
                C.check(rc)
        # none yet, too small, or another argument that is refused, again then
        need = ctypes.c_int64()
        C.call("dt_cached_attn_workspace", handle, B, T, H, D, s_p, n_p, pre, int(prefix_slot), dtype, ctypes.byref(need))
        ws = new_workspace(Q, cache.ctx.device, stream, need.value) if kept is None or need.value > kept[1] else kept
        C.check(attend(ws[0], ws[1]))
        return FlashAttentionResult(O, m, l)
    Qh = np.ascontiguousarray(Q)
    O = np.empty_like(Qh)
    m = np.empty((B, T, H), np.float32)
    l = np.empty((B, T, H), np.float32)
    C.call("dt_cached_attn_fwd", cache._live(), Qh.ctypes.data, O.ctypes.data, m.ctypes.data, l.ctypes.data, B, T, H, D,
           H * D, float(scale), int(bool(causal)), s_p, n_p, pre, int(prefix_slot), None, 0, dtype, C.DT_MEM_HOST, None)
    return FlashAttentionResult(O, m, l)
