"""Rotary positions of queries and keys, with or without each head's norm, on the HIP path: every call goes to
libdirktensor_amd.so; nothing here computes.

    Rotary(dims, theta, layout, scaling)      which values of a head turn, and how far a position turns them
    rotary(Q, K, rot, positions=...)          the rotation at any positions (apply_rope, OlmoAttention.cpp:111-146)
    rotary_backward(dQ, dK, rot, ...)         its gradient
    head_norm_rotary(Q, K, wq, wk, rot, ...)  RMSNorm of each head and the rotation in one pass
    head_norm_rotary_backward(...)            its gradients, those of the norm weights among them

A step of generation rotates the newest tokens at the positions where the cache continues (``starts=cache.lengths``)
and appends the keys.
"""

from __future__ import annotations

import ctypes
from dataclasses import dataclass
from typing import Optional

import numpy as np

from . import _capi as C
from ._workspace import kept_workspace, new_workspace
from .attention import Context, _is_torch, _mode_of, _stream_of, default_context, torch
from .cache import _per_row, _rows_of

_LAYOUTS = {"half": C.DT_ROTARY_HALF, "interleaved": C.DT_ROTARY_INTERLEAVED}
_SCALINGS = {None: C.DT_ROTARY_UNSCALED, "linear": C.DT_ROTARY_LINEAR, "theta": C.DT_ROTARY_THETA, "ramp": C.DT_ROTARY_RAMP}


class Rotary:
    """How positions turn a head's values: the first ``dims`` of 128 (a multiple of 16), in pairs (d, d + dims/2) for the
    layout "half" or (2i, 2i + 1) for "interleaved", pair i by theta^(-2i/dims) radians a position; the results are
    multiplied by ``magnitude``.

    scaling, for contexts longer than the trained one, by ``factor``:
        "linear"  every frequency divided by the factor
        "theta"   theta times factor^(dims / (dims - 2)): the slowest pair is divided by the factor, the fastest stays
        "ramp"    a pair that makes ``high`` turns or more over ``original_length`` stays, one that makes ``low`` or
                  fewer is divided by the factor, between them a share of both, linear in the turns
    ``frequencies`` ([dims/2], radians a position) takes the place of all of these."""

    def __init__(self, dims: int = C.HEAD_DIM, theta: float = 500000.0, layout: str = "half", scaling: Optional[str] = None,
                 factor: float = 1.0, original_length: float = C.MAX_SEQ_LEN, low: float = 1.0, high: float = 32.0,
                 magnitude: float = 1.0, frequencies=None):
        if layout not in _LAYOUTS:
            raise ValueError(f"unknown layout {layout!r}: expected one of {sorted(_LAYOUTS)}")
        if scaling not in _SCALINGS:
            raise ValueError(f"unknown scaling {scaling!r}: expected None, 'linear', 'theta' or 'ramp'")
        self._c = C.DTRotary()
        self._p = ctypes.addressof(self._c)
        C.call("dt_rotary_init", self._p, int(dims), _LAYOUTS[layout], float(theta), _SCALINGS[scaling], float(factor),
               float(original_length), float(low), float(high), float(magnitude))
        if frequencies is not None:
            f = np.asarray(frequencies, dtype=np.float64)
            if f.shape != (self._c.dims // 2,) or not np.isfinite(f).all():
                raise ValueError(f"frequencies must be {self._c.dims // 2} finite numbers")
            self._c.frequency[:len(f)] = f.tolist()
        self.layout = layout

    @property
    def dims(self) -> int:
        return self._c.dims

    @property
    def magnitude(self) -> float:
        return self._c.magnitude

    @property
    def frequencies(self) -> np.ndarray:
        """Radians a position of each pair."""
        return np.array(self._c.frequency[:self._c.dims // 2])


@dataclass
class HeadNormRotaryGradients:
    """d_Q [B, T, H, 128] and d_K [B, T, Hk, 128] in the inputs' dtype, d_q_weight and d_k_weight [128] fp32 (those of K are
    None without it)."""

    d_Q: object
    d_K: object
    d_q_weight: object
    d_k_weight: object


def _check_rows(Q, K, names=("Q", "K")):
    """[B, T, heads, 128] tensors of one kind, dtype and place; K may be None. (B, T, H, Hk)"""
    q = Q.shape
    if len(q) != 4 or q[3] != C.HEAD_DIM:
        raise ValueError(f"{names[0]} must be [B, T, H, {C.HEAD_DIM}], got {tuple(q)}")
    B, T, H = q[0], q[1], q[2]
    if K is None:
        return B, T, H, 0
    k = K.shape
    if len(k) != 4 or k[3] != C.HEAD_DIM or k[0] != B or k[1] != T:
        raise ValueError(f"{names[1]} must be [{B}, {T}, heads, {C.HEAD_DIM}], got {tuple(k)}")
    if _is_torch(Q) != _is_torch(K) or Q.dtype != K.dtype or (_is_torch(Q) and Q.device != K.device):
        raise TypeError(f"{names[0]} and {names[1]} must be of one kind, dtype and device")
    return B, T, H, k[2]


def _context_of(Q, ctx):
    if not _is_torch(Q):
        return ctx or default_context(0)
    if not Q.is_cuda:
        raise ValueError("torch inputs must be on a ROCm device; use numpy arrays for host memory")
    ctx = ctx or default_context(Q.device.index or 0)
    if Q.device.index != ctx.device:
        raise ValueError(f"a tensor is on {Q.device}, the context on cuda:{ctx.device}")
    return ctx


def _positions_of(positions, starts, B, T, like):
    """(what to hold, the positions' address, their bytes, the starts' address)"""
    if positions is None:
        if starts is None:
            return None, None, 0, None
        s, s_p = _per_row(starts, B, "starts")
        return s, None, 0, s_p
    if starts is not None:
        raise ValueError("positions and starts exclude each other")
    if tuple(positions.shape) != (B, T):
        raise ValueError(f"positions have shape {tuple(positions.shape)}, expected {(B, T)}")
    if _is_torch(like):
        if not _is_torch(positions) or positions.device != like.device:
            raise ValueError("positions must be where the rows are")
        if positions.dtype not in (torch.int32, torch.int64):
            raise TypeError(f"unsupported position dtype {positions.dtype}: int32 or int64")
        p = positions.contiguous()
        return p, p.data_ptr(), p.element_size(), None
    p = np.asarray(positions.cpu() if _is_torch(positions) else positions)
    if p.dtype not in (np.int32, np.int64):
        raise TypeError(f"unsupported position dtype {p.dtype}: int32 or int64")
    p = np.ascontiguousarray(p)
    return p, p.ctypes.data, p.itemsize, None


def _inputs(x, host):
    """A tensor's rows as the library takes them: (what to hold, address, token stride)"""
    if x is None:
        return None, None, 0
    if host:
        a = np.ascontiguousarray(x)
        return a, a.ctypes.data, a.shape[2] * C.HEAD_DIM
    if x.is_contiguous():  # (as _rows_of has it)
        p = x.data_ptr()
        if p % 16 == 0:
            return x, p, x.shape[2] * C.HEAD_DIM
    r, ld = _rows_of(x)
    return r, r.data_ptr(), ld


def _rows_and_result(x, host, inplace):
    """The same, and where the result goes: (what to hold, address, token stride, the result, its address, its token stride)"""
    if x is None:
        return None, None, 0, None, None, 0
    r, p, ld = _inputs(x, host)
    if inplace:
        if r is not x or (host and not x.flags.writeable):
            raise ValueError("in place needs writable rows of 128 contiguous values, 16-byte aligned, with one stride between tokens")
        if not host and x.requires_grad and torch.is_grad_enabled():
            raise ValueError("in place, a tensor that requires a gradient is only overwritten under torch.no_grad()")
        return r, p, ld, x, p, ld
    if host:
        o = np.empty(x.shape, x.dtype)
        return r, p, ld, o, o.ctypes.data, o.shape[2] * C.HEAD_DIM
    o = torch.empty_like(r) if r is x and x.is_contiguous() else x.new_empty(x.shape)
    return r, p, ld, o, o.data_ptr(), x.shape[2] * C.HEAD_DIM


def _overwritten(*tensors):
    """What torch's own operators do behind a write: a graph that saved such a tensor raises when it meets the new values."""
    torch.autograd.graph.increment_version([t for t in tensors if t is not None])


_needs: dict = {}  # bytes by (B, T, H, Hk): they follow from these alone


def _workspace_bytes(B: int, T: int, H: int, Hk: int) -> int:
    n = _needs.get((B, T, H, Hk))
    if n is None:
        out = ctypes.c_int64()
        C.call("dt_head_norm_rotary_bwd_workspace", B, T, H, Hk, ctypes.byref(out))
        if len(_needs) >= 4096:
            _needs.clear()
        n = _needs[(B, T, H, Hk)] = out.value
    return n


def _weight(w, like, name):
    if _is_torch(like):
        if not _is_torch(w) or w.dtype != torch.float32 or w.dim() != 1 or w.numel() != C.HEAD_DIM or w.device != like.device:
            raise ValueError(f"{name} must be a [{C.HEAD_DIM}] fp32 tensor where the rows are")
        if not w.is_contiguous() or w.data_ptr() % 16:
            w = w.clone(memory_format=torch.contiguous_format)
        return w, w.data_ptr()
    w = np.ascontiguousarray(w)
    if w.dtype != np.float32 or w.shape != (C.HEAD_DIM,):
        raise ValueError(f"{name} must be a [{C.HEAD_DIM}] fp32 array")
    return w, w.ctypes.data


def _rotate(Q, K, rot, positions, starts, inplace, ctx, backward):
    B, T, H, Hk = _check_rows(Q, K, ("d_Q", "d_K") if backward else ("Q", "K"))
    ctx = _context_of(Q, ctx)
    dtype, host = _mode_of(Q, None), not _is_torch(Q)
    _held, pos_p, pos_bytes, starts_p = _positions_of(positions, starts, B, T, Q)
    _q, q_p, ldq, out_q, oq_p, ldoq = _rows_and_result(Q, host, inplace)
    _k, k_p, ldk, out_k, ok_p, ldok = _rows_and_result(K, host, inplace)
    mem, stream = (C.DT_MEM_HOST, None) if host else (C.DT_MEM_DEVICE, _stream_of(Q))
    C.check(C.lib().dt_rotary_fwd(ctx.handle, q_p, k_p, oq_p, ok_p, B, T, H, Hk, C.HEAD_DIM, ldq, ldk, ldoq, ldok, pos_p, pos_bytes,
                                  starts_p, rot._p, backward, dtype, mem, stream))
    if inplace and not host:
        _overwritten(Q, K)
    return out_q, out_k


def rotary(Q, K, rot: Rotary, *, positions=None, starts=None, inplace: bool = False, ctx: Optional[Context] = None):
    """Q [B, T, H, 128] and K [B, T, Hk, 128] (or None) rotated to their positions, as (Q', K'): bf16 or fp32, torch device
    tensors, views of a projection's output among them, or numpy arrays.

    Token (b, t) is at ``positions`` [B, T] (int32 or int64, where the rows are), or at starts[b] + t for ``starts`` of B whole
    numbers on the host (such as a cache's lengths; a captured call repeats them), or at t. With ``inplace`` Q and K are
    overwritten (torch is told, as by its own operators; tensors that require a gradient are refused where gradients are
    recorded)."""
    return _rotate(Q, K, rot, positions, starts, inplace, ctx, 0)


def rotary_backward(d_Q, d_K, rot: Rotary, *, positions=None, starts=None, inplace: bool = False, ctx: Optional[Context] = None):
    """The gradients of rotary's inputs from those of its outputs, at the same positions."""
    return _rotate(d_Q, d_K, rot, positions, starts, inplace, ctx, 1)


def head_norm_rotary(Q, K, q_weight, k_weight, rot: Rotary, *, positions=None, starts=None, eps: float = 1e-6,
                     inplace: bool = False, ctx: Optional[Context] = None):
    """RMSNorm of each head, x / sqrt(mean x^2 + eps) * weight with q_weight and k_weight [128] in fp32, and the rotation, as
    (Q', K'). Everything else as in ``rotary``; K None: k_weight is ignored. (qk_norm_rope's norm spans all heads.)"""
    B, T, H, Hk = _check_rows(Q, K)
    ctx = _context_of(Q, ctx)
    dtype, host = _mode_of(Q, None), not _is_torch(Q)
    _held, pos_p, pos_bytes, starts_p = _positions_of(positions, starts, B, T, Q)
    _wq, wq_p = _weight(q_weight, Q, "q_weight")
    _wk, wk_p = _weight(k_weight, Q, "k_weight") if Hk else (None, None)
    _q, q_p, ldq, out_q, oq_p, ldoq = _rows_and_result(Q, host, inplace)
    _k, k_p, ldk, out_k, ok_p, ldok = _rows_and_result(K, host, inplace)
    mem, stream = (C.DT_MEM_HOST, None) if host else (C.DT_MEM_DEVICE, _stream_of(Q))
    C.check(C.lib().dt_head_norm_rotary_fwd(ctx.handle, q_p, k_p, wq_p, wk_p, oq_p, ok_p, B, T, H, Hk, C.HEAD_DIM, ldq, ldk, ldoq, ldok,
                                            pos_p, pos_bytes, starts_p, rot._p, float(eps), dtype, mem, stream))
    if inplace and not host:
        _overwritten(Q, K)
    return out_q, out_k


def head_norm_rotary_backward(d_Q, d_K, Q, K, q_weight, k_weight, rot: Rotary, *, positions=None, starts=None, eps: float = 1e-6,
                              ctx: Optional[Context] = None) -> HeadNormRotaryGradients:
    """The gradients of head_norm_rotary's inputs and weights from those of its outputs, at the same positions."""
    B, T, H, Hk = _check_rows(d_Q, d_K, ("d_Q", "d_K"))
    if (K is None) != (d_K is None):
        raise ValueError("K and d_K must both be given, or neither")
    if tuple(Q.shape) != tuple(d_Q.shape) or _check_rows(Q, K)[3] != Hk:
        raise ValueError("Q and K must have their gradients' shapes")
    if _is_torch(Q) != _is_torch(d_Q) or Q.dtype != d_Q.dtype or (_is_torch(Q) and Q.device != d_Q.device):
        raise TypeError("the gradients must be of the inputs' kind, dtype and device")
    ctx = _context_of(Q, ctx)
    dtype, host = _mode_of(Q, None), not _is_torch(Q)
    _held, pos_p, pos_bytes, starts_p = _positions_of(positions, starts, B, T, Q)
    _wq, wq_p = _weight(q_weight, Q, "q_weight")
    _wk, wk_p = _weight(k_weight, Q, "k_weight") if Hk else (None, None)
    _gq, gq_p, ldgq = _inputs(d_Q, host)
    _gk, gk_p, ldgk = _inputs(d_K, host)
    _q, q_p, ldq, out_q, oq_p, ldoq = _rows_and_result(Q, host, False)
    _k, k_p, ldk, out_k, ok_p, ldok = _rows_and_result(K, host, False)
    n = 2 if Hk else 1
    if host:
        dw = np.empty((n, C.HEAD_DIM), np.float32)
        dw_p, ws, mem, stream = dw.ctypes.data, (None, 0), C.DT_MEM_HOST, None
        d_w = list(dw)
    else:
        dw = Q.new_empty((n, C.HEAD_DIM), dtype=torch.float32)
        dw_p, mem, stream = dw.data_ptr(), C.DT_MEM_DEVICE, _stream_of(Q)
        d_w = dw.unbind(0)
        need = _workspace_bytes(B, T, H, Hk)
        ws = kept_workspace(ctx.device, stream)
        if ws is None or ws[1] < need:
            ws = new_workspace(Q, ctx.device, stream, need)
    C.check(C.lib().dt_head_norm_rotary_bwd(ctx.handle, gq_p, gk_p, q_p, k_p, wq_p, wk_p, oq_p, ok_p, dw_p,
                                            dw_p + 4 * C.HEAD_DIM if Hk else None, B, T, H, Hk, C.HEAD_DIM, ldgq, ldgk, ldq, ldk, ldoq,
                                            ldok, pos_p, pos_bytes, starts_p, rot._p, float(eps), ws[0], ws[1], dtype, mem, stream))
    return HeadNormRotaryGradients(out_q, out_k, d_w[0], d_w[1] if Hk else None)
