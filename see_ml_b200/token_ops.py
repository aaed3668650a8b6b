"""Vocabulary-row operators on torch CUDA tensors, over the C ABI: scores of given tokens
(log probability, entropy, top alternatives), distillation from a teacher's top entries, and
their gradients. The entry points are described in include/seeml_b200.h.

Logits are a [rows, vocab] tensor in f32, bf16 or f16 whose columns are contiguous; rows may be
strided. Work is enqueued on torch's current stream of the logits' device and returns at once.
These are plain functions, not autograd nodes: the gradient is a call of its own. Arguments that
do not fit raise ``BackendError``.

    s = token_scores(teacher_logits, tokens, top_k=32, temperature=T)
    r = distill_topk(student_logits, s.top_id, s.top_logprob, row_weight=mask, scale=1 / n,
                     temperature=T, tail=True, grad=True)          # r.loss, r.dlogits
"""
from __future__ import annotations

import ctypes as C
from typing import NamedTuple, Optional

import torch

from . import _lib as L

TOP_K_MAX = 128
_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_F32, _I32 = torch.float32, torch.int32


class TokenScores(NamedTuple):
    logprob: Optional[torch.Tensor]      # [rows] f32, None without labels
    entropy: Optional[torch.Tensor]      # [rows] f32
    stats: Optional[torch.Tensor]        # [rows, 2] f32: max, sum exp((x - max) / T); for token_scores_backward
    top_logprob: Optional[torch.Tensor]  # [rows, top_k] f32
    top_id: Optional[torch.Tensor]       # [rows, top_k] i32


class DistillLoss(NamedTuple):
    loss: torch.Tensor                   # [] f32
    row_loss: torch.Tensor               # [rows] f32
    saved: Optional[torch.Tensor]        # [rows, 4] f32, what distill_topk_backward reads
    dlogits: Optional[torch.Tensor]      # [rows, vocab], the logits' type


def _refuse(msg):
    raise L.BackendError("UpdateEngine: " + msg)


def _matrix(name, t):
    if not isinstance(t, torch.Tensor) or t.dim() != 2:
        _refuse(f"{name} must be a [rows, vocab] tensor")
    if not t.is_cuda:
        _refuse(f"{name} must be device memory")
    if t.dtype not in _DTYPES:
        _refuse(f"{name} must be f32, bf16 or f16 (got {t.dtype})")
    if t.shape[1] > 1 and t.stride(1) != 1:
        _refuse(f"the columns of {name} must be contiguous")
    if t.shape[0] > 1 and t.stride(0) < t.shape[1]:
        _refuse(f"the rows of {name} overlap (row stride {t.stride(0)}, {t.shape[1]} columns)")
    return t


def _stride(t):
    return t.stride(0) if t.shape[0] > 1 else max(t.stride(0), t.shape[1])


def _operand(name, t, shape, dtypes, device):
    if t is None:
        return None
    if not isinstance(t, torch.Tensor) or tuple(t.shape) != shape:
        _refuse(f"{name} must be a tensor of shape {shape}")
    if t.dtype not in dtypes:
        _refuse(f"{name} has type {t.dtype}")
    if t.device != device:
        _refuse(f"{name} lives on {t.device}, the logits on {device}")
    if not t.is_contiguous():
        _refuse(f"{name} must be contiguous")
    return t.data_ptr()


def _gradient(logits, out):
    if out is None:
        return torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
    _matrix("out", out)
    if out.shape != logits.shape or out.dtype != logits.dtype or out.device != logits.device:
        _refuse("out must have the logits' shape, type and device")
    return out


def _call(fn, desc, device):
    stream = torch._C._cuda_getCurrentRawStream(device.index)      # current_stream() without building its object
    if torch.cuda.current_device() == device.index:
        rc = fn(C.byref(desc), stream)
    else:
        with torch.cuda.device(device):
            rc = fn(C.byref(desc), stream)
    if rc:
        raise L.BackendError(L.last_error())


def token_scores(logits, labels=None, *, top_k=0, temperature=1.0, entropy=True, stats=False) -> TokenScores:
    """Log probability of `labels` (i32, negative = none), entropy and the `top_k` alternatives."""
    _matrix("logits", logits)
    rows, vocab = logits.shape
    dev = logits.device
    if not 0 <= top_k <= min(TOP_K_MAX, vocab):
        _refuse(f"top_k must be 0..{TOP_K_MAX} and at most the vocabulary (got {top_k})")
    lab = _operand("labels", labels, (rows,), (_I32,), dev)
    logprob = torch.empty(rows, dtype=_F32, device=dev) if labels is not None else None
    ent = torch.empty(rows, dtype=_F32, device=dev) if entropy else None
    st = torch.empty((rows, 2), dtype=_F32, device=dev) if stats else None
    top_lp = torch.empty((rows, top_k), dtype=_F32, device=dev) if top_k else None
    top_id = torch.empty((rows, top_k), dtype=_I32, device=dev) if top_k else None
    d = L.TokenScores(logits.data_ptr(), lab, logprob.data_ptr() if logprob is not None else None,
                      ent.data_ptr() if entropy else None, st.data_ptr() if stats else None, top_lp.data_ptr() if top_k else None,
                      top_id.data_ptr() if top_k else None, rows, vocab, _stride(logits), _DTYPES[logits.dtype], top_k,
                      temperature, 0)
    _call(L.lib().seeml_b200_token_scores_fwd, d, dev)
    return TokenScores(logprob, ent, st, top_lp, top_id)


def token_scores_backward(logits, labels, stats, entropy, dlogprob, dentropy, *, temperature=1.0, out=None):
    """Gradient of sum(dlogprob * logprob + dentropy * entropy); `out` may be the logits."""
    _matrix("logits", logits)
    rows, vocab = logits.shape
    dev = logits.device
    lab = _operand("labels", labels, (rows,), (_I32,), dev)
    st = _operand("stats", stats, (rows, 2), (_F32,), dev)
    ent = _operand("entropy", entropy, (rows,), (_F32,), dev)
    dlp = _operand("dlogprob", dlogprob, (rows,), (_F32,), dev)
    dent = _operand("dentropy", dentropy, (rows,), (_F32,), dev)
    g = _gradient(logits, out)
    d = L.TokenScoresGrad(logits.data_ptr(), lab, st, ent, dlp, dent, g.data_ptr(), rows, vocab, _stride(logits),
                          _stride(g), _DTYPES[logits.dtype], temperature)
    _call(L.lib().seeml_b200_token_scores_bwd, d, dev)
    return g


def distill_topk(logits, teacher_id, teacher_logprob, *, row_weight=None, scale=1.0, temperature=1.0, tail=False,
                 grad=False, saved=False, out=None) -> DistillLoss:
    """Loss against a teacher's top entries, with its gradient (`grad`, into `out` when given, which
    may be the logits) or with what `distill_topk_backward` needs (`saved`)."""
    _matrix("logits", logits)
    rows, vocab = logits.shape
    dev = logits.device
    if not isinstance(teacher_id, torch.Tensor) or teacher_id.dim() != 2:
        _refuse("teacher_id must be a [rows, entries] tensor")
    k = teacher_id.shape[1]
    tid = _operand("teacher_id", teacher_id, (rows, k), (_I32,), dev)
    tlp = _operand("teacher_logprob", teacher_logprob, (rows, k), _DTYPES, dev)
    if tlp is None:
        _refuse("teacher_logprob is missing")
    w = _operand("row_weight", row_weight, (rows,), (_F32,), dev)
    row_loss = torch.empty(rows, dtype=_F32, device=dev)
    loss = torch.empty((), dtype=_F32, device=dev)
    keep = torch.empty((rows, 4), dtype=_F32, device=dev) if saved else None
    g = _gradient(logits, out) if grad or out is not None else None
    d = L.DistillTopk(logits.data_ptr(), tid, tlp, w, row_loss.data_ptr(), loss.data_ptr(),
                      keep.data_ptr() if saved else None, g.data_ptr() if g is not None else None, rows, vocab,
                      _stride(logits), _stride(g) if g is not None else vocab, _DTYPES[logits.dtype],
                      _DTYPES[teacher_logprob.dtype], k, int(bool(tail)), temperature, scale)
    _call(L.lib().seeml_b200_distill_topk_fwd, d, dev)
    return DistillLoss(loss, row_loss, keep, g)


def distill_topk_backward(logits, teacher_id, teacher_logprob, saved, drow_loss, *, temperature=1.0, tail=False, out=None):
    """Gradient of sum(drow_loss * row_loss) from the forward call's `saved`; `out` may be the logits."""
    _matrix("logits", logits)
    rows, vocab = logits.shape
    dev = logits.device
    if not isinstance(teacher_id, torch.Tensor) or teacher_id.dim() != 2:
        _refuse("teacher_id must be a [rows, entries] tensor")
    k = teacher_id.shape[1]
    tid = _operand("teacher_id", teacher_id, (rows, k), (_I32,), dev)
    tlp = _operand("teacher_logprob", teacher_logprob, (rows, k), _DTYPES, dev)
    if tlp is None:
        _refuse("teacher_logprob is missing")
    sv = _operand("saved", saved, (rows, 4), (_F32,), dev)
    up = _operand("drow_loss", drow_loss, (rows,), (_F32,), dev)
    g = _gradient(logits, out)
    d = L.DistillTopkGrad(logits.data_ptr(), tid, tlp, sv, up, g.data_ptr(), rows, vocab, _stride(logits), _stride(g),
                          _DTYPES[logits.dtype], _DTYPES[teacher_logprob.dtype], k, int(bool(tail)), temperature, 0)
    _call(L.lib().seeml_b200_distill_topk_bwd, d, dev)
    return g
