"""Scores of given tokens and their gradient, on the HIP path (beside ce_loss, which gives their mean over a batch): every
call goes to libdirktensor_amd.so; nothing here computes.

    token_logprobs(logits, tokens, top_k=0) -> TokenLogprobs
        log probabilities of the tokens, the rows' entropies and their top_k most likely tokens
    token_logprobs_backward(d_logprob, logits, tokens, result, d_entropy=None) -> d_logits
"""

from __future__ import annotations

import ctypes
from dataclasses import dataclass
from typing import Optional

import numpy as np

from . import _capi as C
from ._workspace import kept_workspace, new_workspace
from .attention import Context, _is_torch, _mode_of, _stream_of, default_context, torch


@dataclass
class TokenLogprobs:
    """logprob, entropy (nats), softmax_m (row maximum) and softmax_l (sum exp(x - m)) [...], fp32; with top_k > 0 top_index
    (int32) and top_logprob [..., top_k], descending, the lower index first of equals. ``ignore_index`` is the call's."""

    logprob: object
    entropy: object
    softmax_m: object
    softmax_l: object
    top_index: object = None
    top_logprob: object = None
    ignore_index: Optional[int] = None


def _two_strides(shape, strides):
    """Leading dimensions as B x T of two strides: (B, T, ldb, ldt), or None where they are none."""
    dims = [(n, s) for n, s in zip(shape, strides) if n != 1]
    merged = []
    for n, s in dims:
        if merged and merged[-1][1] == n * s:
            merged[-1] = (merged[-1][0] * n, s)
        else:
            merged.append((n, s))
    if len(merged) > 2:
        return None
    while len(merged) < 2:
        merged.insert(0, (1, 0))
    (B, ldb), (T, ldt) = merged
    return B, T, ldb, ldt


def _check_tokens(tokens, lead, like):
    if tokens.shape != lead:
        raise ValueError(f"tokens have shape {tuple(tokens.shape)}, expected {tuple(lead)}")
    if _is_torch(like):
        if not _is_torch(tokens) or tokens.device != like.device:
            raise ValueError("tokens must be a torch tensor on the logits' device")
        if tokens.dtype not in (torch.int32, torch.int64):
            raise TypeError(f"unsupported token dtype {tokens.dtype}: int32 or int64")
        t = tokens.contiguous()
        return t, t.data_ptr(), 4 if t.dtype == torch.int32 else 8
    t = np.asarray(tokens.cpu() if _is_torch(tokens) else tokens)
    if t.dtype not in (np.int32, np.int64):
        raise TypeError(f"unsupported token dtype {t.dtype}: int32 or int64")
    t = np.ascontiguousarray(t)
    return t, t.ctypes.data, t.itemsize


def _ignore_of(ignore_index) -> int:
    if ignore_index is None:
        return C.DT_NO_IGNORE
    i = int(ignore_index)
    if not C.DT_NO_IGNORE < i < 2**63:
        raise ValueError(f"ignore_index={i} is no token index of 64 bits, or the least one, which stands for none")
    return i


def _check_logits(logits, ctx):
    if len(logits.shape) < 1:
        raise ValueError("logits need a vocabulary dimension")
    if _is_torch(logits):
        if not logits.is_cuda:
            raise ValueError("torch inputs must be on a ROCm device; use numpy arrays for host memory")
        ctx = ctx or default_context(logits.device.index or 0)
        if logits.device.index != ctx.device:
            raise ValueError(f"logits are on {logits.device}, the context on cuda:{ctx.device}")
        return ctx
    return ctx or default_context(0)


def _rows(logits):
    """The logits' rows as the library takes them: the tensor itself where its leading dimensions have at most two strides
    (a slice [:, :-1] is one), else a copy."""
    if logits.is_contiguous():
        V = logits.shape[-1]
        return logits, (1, logits.numel() // V if V else 0, 0, V)
    if logits.stride(-1) == 1 or logits.shape[-1] == 1:
        r = _two_strides(logits.shape[:-1], logits.stride()[:-1])
        if r is not None:
            return logits, r
    logits = logits.contiguous()
    return logits, _two_strides(logits.shape[:-1], logits.stride()[:-1])


_needs: dict = {}  # bytes by (B, T, V, top_k): they follow from the sizes alone


def _workspace_bytes(B: int, T: int, V: int, k: int) -> int:
    n = _needs.get((B, T, V, k))
    if n is None:
        out = ctypes.c_int64()
        C.call("dt_token_logprobs_workspace", B, T, V, k, ctypes.byref(out))
        if len(_needs) >= 4096:
            _needs.clear()
        n = _needs[(B, T, V, k)] = out.value
    return n


def token_logprobs(logits, tokens, *, top_k: int = 0, ignore_index: Optional[int] = None,
                   ctx: Optional[Context] = None) -> TokenLogprobs:
    """Scores tokens [...] by the rows of logits [..., V] (fp32 or bf16, torch device tensors, strided views such as
    logits[:, :-1] among them, or numpy arrays). For next-token scores pass logits[:, :-1] and tokens[:, 1:].

    Positions whose token is ``ignore_index`` get logprob 0 (and no gradient from it). A token outside the vocabulary is refused
    with numpy arrays and gives NaN on the device. Logits of -inf are tokens of probability 0; a row with a NaN or +inf, or with
    nothing but -inf, gives NaN. top_k: 0 to 64."""
    ctx = _check_logits(logits, ctx)
    lead, V, k = logits.shape[:-1], logits.shape[-1], int(top_k)
    dtype = _mode_of(logits, None)
    tok, tok_p, tok_bytes = _check_tokens(tokens, lead, logits)
    ign = _ignore_of(ignore_index)
    if _is_torch(logits):
        x, (B, T, ldb, ldt) = _rows(logits)
        nbytes = _workspace_bytes(B, T, V, k)
        stream = _stream_of(x)
        ws = (None, 0)
        if nbytes:
            ws = kept_workspace(ctx.device, stream)
            if ws is None or ws[1] < nbytes:
                ws = new_workspace(x, ctx.device, stream, nbytes)
        lp, ent, m, l = x.new_empty((4, *lead), dtype=torch.float32).unbind(0)
        idx = x.new_empty((*lead, k), dtype=torch.int32) if k else None
        top = torch.empty_like(idx, dtype=torch.float32) if k else None
        C.call("dt_token_logprobs", ctx.handle, x.data_ptr(), tok_p, B, T, V, ldb, ldt, tok_bytes, ign, k, lp.data_ptr(),
               ent.data_ptr(), m.data_ptr(), l.data_ptr(), idx.data_ptr() if k else None, top.data_ptr() if k else None,
               ws[0], ws[1], dtype, C.DT_MEM_DEVICE, stream)
        return TokenLogprobs(lp, ent, m, l, idx, top, ignore_index)
    x = np.ascontiguousarray(logits)
    rows = int(np.prod(lead, dtype=np.int64))
    lp, ent, m, l = (np.empty(lead, np.float32) for _ in range(4))
    idx = np.empty((*lead, k), np.int32) if k else None
    top = np.empty((*lead, k), np.float32) if k else None
    C.call("dt_token_logprobs", ctx.handle, x.ctypes.data, tok_p, 1, rows, V, rows * V, V, tok_bytes, ign, k, lp.ctypes.data,
           ent.ctypes.data, m.ctypes.data, l.ctypes.data, idx.ctypes.data if k else None, top.ctypes.data if k else None, None,
           0, dtype, C.DT_MEM_HOST, None)
    return TokenLogprobs(lp, ent, m, l, idx, top, ignore_index)


def _span(t):
    """The addresses that a tensor's elements lie in."""
    last = sum((n - 1) * s for n, s in zip(t.shape, t.stride()))
    return t.data_ptr(), t.data_ptr() + (last + 1) * t.element_size()


def _out_rows(out, logits, x, B, T, ldb, ldt):
    """The rows of ``out`` beside those of x (the logits as they are read), split alike: (B, T, ldb, ldt, ldb_out, ldt_out)."""
    if out.shape != logits.shape or out.dtype != logits.dtype or out.device != logits.device:
        raise ValueError("out must have the logits' shape, dtype and device")
    if out.stride(-1) != 1 and out.shape[-1] != 1:
        raise ValueError("out's vocabulary dimension must be contiguous")
    same = out.data_ptr() == x.data_ptr() and out.stride() == x.stride()
    if not same and out.numel():
        (a0, a1), (b0, b1) = _span(out), _span(x)
        if a0 < b1 and b0 < a1:
            raise ValueError("out overlaps the logits without being them")
    r = _two_strides(out.shape[:-1], out.stride()[:-1])
    if r is not None and r[:2] == (B, T):
        return B, T, ldb, ldt, r[2], r[3]
    if r is not None and B == 1:  # the logits' rows have one stride: they split like out's
        return r[0], r[1], r[1] * ldt, ldt, r[2], r[3]
    if r is not None and r[0] == 1:
        return B, T, ldb, ldt, T * r[3], r[3]
    raise ValueError("out's leading dimensions must have at most two strides, split like the logits'")


def token_logprobs_backward(d_logprob, logits, tokens, result: TokenLogprobs, *, d_entropy=None, out=None,
                            ctx: Optional[Context] = None):
    """The gradient with respect to the logits, in their dtype, of d_logprob [...] and (optionally) d_entropy [...], fp32, for
    the forward's ``result`` on the same logits and tokens. ``out`` (torch): where to write it, a tensor of the logits' shape and
    dtype, or the logits themselves to overwrite them."""
    ctx = _check_logits(logits, ctx)
    lead, V = logits.shape[:-1], logits.shape[-1]
    dtype = _mode_of(logits, None)
    tok, tok_p, tok_bytes = _check_tokens(tokens, lead, logits)
    ign = _ignore_of(result.ignore_index)
    on_device = _is_torch(logits)
    per_row = dict(d_logprob=d_logprob, softmax_m=result.softmax_m, softmax_l=result.softmax_l, entropy=result.entropy)
    if d_entropy is not None:
        per_row["d_entropy"] = d_entropy
    for name, t in per_row.items():
        if t.shape != lead:
            raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {tuple(lead)}")
        if _is_torch(t) != on_device or (on_device and t.device != logits.device):
            raise ValueError(f"{name} must be where the logits are")
    if on_device:
        p = {k: t if t.dtype == torch.float32 and t.is_contiguous() else t.contiguous().float() for k, t in per_row.items()}
        x, (B, T, ldb, ldt) = _rows(logits)
        if out is None:
            out = x.new_empty(logits.shape)
            bo, to = T * V, V  # (row (b, t) is row b T + t of a dense tensor)
        else:
            B, T, ldb, ldt, bo, to = _out_rows(out, logits, x, B, T, ldb, ldt)
        C.call("dt_token_logprobs_bwd", ctx.handle, p["d_logprob"].data_ptr(),
               p["d_entropy"].data_ptr() if d_entropy is not None else None, x.data_ptr(), tok_p, p["softmax_m"].data_ptr(),
               p["softmax_l"].data_ptr(), p["entropy"].data_ptr(), B, T, V, ldb, ldt, tok_bytes, ign, out.data_ptr(), bo, to,
               dtype, C.DT_MEM_DEVICE, _stream_of(x))
        return out
    if out is not None:
        raise ValueError("out is for torch tensors")
    x = np.ascontiguousarray(logits)
    p = {k: np.ascontiguousarray(t, dtype=np.float32) for k, t in per_row.items()}
    g = np.empty_like(x)
    rows = int(np.prod(lead, dtype=np.int64))
    C.call("dt_token_logprobs_bwd", ctx.handle, p["d_logprob"].ctypes.data,
           p["d_entropy"].ctypes.data if d_entropy is not None else None, x.ctypes.data, tok_p, p["softmax_m"].ctypes.data,
           p["softmax_l"].ctypes.data, p["entropy"].ctypes.data, 1, rows, V, rows * V, V, tok_bytes, ign, g.ctypes.data,
           rows * V, V, dtype, C.DT_MEM_HOST, None)
    return g
