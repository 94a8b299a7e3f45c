"""Drafted tokens verified against a model's probabilities, on the HIP path: every call goes to libdirktensor_amd.so;
nothing here computes.

    verify_drafts(logits, drafts, uniforms, draft_logits=None) -> VerifiedDrafts
        how many drafts of each sequence are accepted, and the token that follows them

A program drafts K tokens a sequence, runs the model over them (appending their keys and values to the cache), verifies
them, and truncates the cache to what was accepted.
"""

from __future__ import annotations

import ctypes
from dataclasses import dataclass
from typing import Optional

import numpy as np

from . import _capi as C
from ._workspace import kept_workspace, new_workspace
from .attention import Context, _is_torch, _mode_of, _stream_of, torch
from .cache import _per_row
from .logprobs import _check_logits


@dataclass
class VerifiedDrafts:
    """accepted [B] int32: how many drafts were accepted; tokens [B, K + 1] int32: these, the token that follows, then -1;
    logprob [B, K + 1] fp32: the tokens' log probabilities, then 0."""

    accepted: object
    tokens: object
    logprob: object


def _logit_rows(x):
    """[B, T, V] logits with contiguous rows: (the tensor itself, or a copy; batch stride, row stride)"""
    if x.is_contiguous():
        return x, x.shape[1] * x.shape[2], x.shape[2]
    if (x.stride(2) == 1 or x.shape[2] == 1) and x.stride(0) >= 0 and x.stride(1) >= 0:
        return x, x.stride(0), x.stride(1)
    x = x.contiguous()
    return x, x.stride(0), x.stride(1)


_needs: dict = {}  # bytes by (B, K, V, draft logits, greedy): they follow from these alone


def _workspace_bytes(B, K, V, drafts, temperature) -> int:
    key = (B, K, V, drafts, temperature == 0.0)
    n = _needs.get(key)
    if n is None:
        out = ctypes.c_int64()
        C.call("dt_verify_drafts_workspace", B, K, V, drafts, temperature, ctypes.byref(out))
        if len(_needs) >= 4096:
            _needs.clear()
        n = _needs[key] = out.value
    return n


def verify_drafts(logits, drafts, uniforms, *, draft_logits=None, temperature: float = 1.0, counts=None,
                  ctx: Optional[Context] = None) -> VerifiedDrafts:
    """Which drafted tokens the model accepts, and the token that follows them.

    logits [B, K + 1, V] (bf16 or fp32; torch device tensors, strided views with contiguous rows among them, or numpy
    arrays): row i gives the token behind the first i drafts. drafts [B, K], int32 or int64 (K = 0: a token is drawn).
    uniforms [B, K + 1], fp32 in [0, 1): one for each draft, the last for the token that follows (None is allowed at
    temperature 0). draft_logits [B, K, V], of the logits' dtype: what the drafts were drawn from, at the same
    temperature; None for drafts that nothing was drawn for (each counts as drawn with probability 1). counts: how many drafts each
    batch row has (host; the rows behind them are not read).

    With p and q the softmax of logits and draft logits over the temperature, draft i is accepted, if those before it were, while
    uniform * q(draft) < p(draft). The token that follows is drawn from max(p - q, 0) where a draft was refused, otherwise from
    the last row's p: what is emitted is distributed as p. At temperature 0 it is the largest logit's token, and drafts that are it
    are accepted. A row with a NaN or +inf, or with nothing but -inf, gives token -1 and log probability NaN."""
    ctx = _check_logits(logits, ctx)
    shape = logits.shape
    if len(shape) != 3 or shape[1] < 1:
        raise ValueError(f"logits must be [B, K + 1, V], got {tuple(shape)}")
    B, K, V = shape[0], shape[1] - 1, shape[2]
    dtype, on_device, temperature = _mode_of(logits, None), _is_torch(logits), float(temperature)
    if tuple(drafts.shape) != (B, K):
        raise ValueError(f"drafts have shape {tuple(drafts.shape)}, expected {(B, K)}")
    if uniforms is not None and tuple(uniforms.shape) != (B, K + 1):
        raise ValueError(f"uniforms have shape {tuple(uniforms.shape)}, expected {(B, K + 1)}")
    if draft_logits is not None:
        if tuple(draft_logits.shape) != (B, K, V) or draft_logits.dtype != logits.dtype:
            raise ValueError(f"draft_logits must be {(B, K, V)} of the logits' dtype, got {draft_logits.dtype} {tuple(draft_logits.shape)}")
    for name, t in (("drafts", drafts), ("uniforms", uniforms), ("draft_logits", draft_logits)):
        if t is not None and (_is_torch(t) != on_device or (on_device and t.device != logits.device)):
            raise ValueError(f"{name} must be where the logits are")
    n, n_p = _per_row(counts, B, "counts")
    has = draft_logits is not None and K > 0
    if on_device:
        if drafts.dtype not in (torch.int32, torch.int64):
            raise TypeError(f"unsupported token dtype {drafts.dtype}: int32 or int64")
        if uniforms is not None and uniforms.dtype != torch.float32:
            raise TypeError(f"unsupported dtype of uniforms {uniforms.dtype}: float32")
        d = drafts.contiguous()
        u = uniforms.contiguous() if uniforms is not None else None
        x, ldb, ldt = _logit_rows(logits)
        y, ldb_y, ldt_y = _logit_rows(draft_logits) if has else (None, 0, 0)
        stream = _stream_of(x)
        need = _workspace_bytes(B, K, V, has, temperature)
        ws = kept_workspace(ctx.device, stream)
        if ws is None or ws[1] < need:
            ws = new_workspace(x, ctx.device, stream, need)
        accepted = x.new_empty((B,), dtype=torch.int32)
        tokens = x.new_empty((B, K + 1), dtype=torch.int32)
        logprob = torch.empty_like(tokens, dtype=torch.float32)
        C.call("dt_verify_drafts", ctx.handle, x.data_ptr(), d.data_ptr() or None, u.data_ptr() if u is not None else None,
               y.data_ptr() if has else None, B, K, V, ldb, ldt, ldb_y, ldt_y, d.element_size(), n_p, temperature,
               accepted.data_ptr(), tokens.data_ptr(), logprob.data_ptr(), ws[0], ws[1], dtype, C.DT_MEM_DEVICE, stream)
        return VerifiedDrafts(accepted, tokens, logprob)
    d = np.ascontiguousarray(drafts)
    if d.dtype not in (np.int32, np.int64):
        raise TypeError(f"unsupported token dtype {d.dtype}: int32 or int64")
    u = np.ascontiguousarray(uniforms) if uniforms is not None else None
    if u is not None and u.dtype != np.float32:
        raise TypeError(f"unsupported dtype of uniforms {u.dtype}: float32")
    x = np.ascontiguousarray(logits)
    y = np.ascontiguousarray(draft_logits) if has else None
    accepted, tokens, logprob = np.empty(B, np.int32), np.empty((B, K + 1), np.int32), np.empty((B, K + 1), np.float32)
    C.call("dt_verify_drafts", ctx.handle, x.ctypes.data, d.ctypes.data if K else None, u.ctypes.data if u is not None else None,
           y.ctypes.data if has else None, B, K, V, (K + 1) * V, V, K * V, V, d.itemsize, n_p, temperature, accepted.ctypes.data,
           tokens.ctypes.data, logprob.ctypes.data, None, 0, dtype, C.DT_MEM_HOST, None)
    return VerifiedDrafts(accepted, tokens, logprob)
