"""Vocabulary-row operators on torch CUDA tensors, over the C ABI: scores of given tokens
(log probability, entropy, top alternatives), distillation from a teacher's top entries, and
their gradients. The entry points are described in include/seeml_b200.h.

Logits are a [rows, vocab] tensor in f32, bf16 or f16 whose columns are contiguous; rows may be
strided. Work is enqueued on torch's current stream of the logits' device and returns at once.
These are plain functions, not autograd nodes: the gradient is a call of its own, also of logits
that require one (hand it on with ``logits.backward(dlogits)``). Writing into `out` counts as an
in-place modification of it, which autograd refuses to overlook when a node has kept the tensor.
Arguments that do not fit raise ``BackendError``.

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
    """Checks a matrix of logits; returns (rows, columns, row stride, dtype code, device index)."""
    if not isinstance(t, torch.Tensor) or t.dim() != 2:
        _refuse(f"{name} must be a [rows, vocab] tensor")
    if not t.is_cuda:
        _refuse(f"{name} must be device memory")
    code = _DTYPES.get(t.dtype)
    if code is None:
        _refuse(f"{name} must be f32, bf16 or f16 (got {t.dtype})")
    rows, cols = t.shape
    pitch, step = t.stride()
    if cols > 1 and step != 1:
        _refuse(f"the columns of {name} must be contiguous")
    if pitch < cols:
        if rows > 1:
            _refuse(f"the rows of {name} overlap (row stride {pitch}, {cols} columns)")
        pitch = cols
    return rows, cols, pitch, code, t.get_device()


def _operand(name, t, shape, dtypes, device):
    if t is None:
        return None
    if not isinstance(t, torch.Tensor) or t.shape != shape:
        _refuse(f"{name} must be a tensor of shape {shape}")
    if t.dtype not in dtypes:
        _refuse(f"{name} has type {t.dtype}")
    if t.get_device() != device:
        _refuse(f"{name} lives on {t.device}, the logits on device {device}")
    if not t.is_contiguous():
        _refuse(f"{name} must be contiguous")
    return t.data_ptr()


def _gradient(logits, out):
    """The gradient's tensor and its row stride."""
    if out is None:
        rows, vocab = logits.shape
        return logits.new_empty(rows, vocab), vocab
    pitch = _matrix("out", out)[2]
    if out.shape != logits.shape or out.dtype != logits.dtype or out.device != logits.device:
        _refuse("out must have the logits' shape, type and device")
    return out, pitch


def _call(fn, desc, device, out=None):
    stream = torch._C._cuda_getCurrentRawStream(device)      # current_stream() without building its object
    if torch._C._cuda_getDevice() == device:
        rc = fn(C.byref(desc), stream)
    else:
        with torch.cuda.device(device):
            rc = fn(C.byref(desc), stream)
    if rc:
        raise L.BackendError(L.last_error())
    if out is not None:
        torch.autograd.graph.increment_version(out)


def _teacher(teacher_id, teacher_logprob, rows, device):
    """Checks a teacher's entries; returns (entries, token pointer, value pointer, dtype code)."""
    if not isinstance(teacher_id, torch.Tensor) or teacher_id.dim() != 2:
        _refuse("teacher_id must be a [rows, entries] tensor")
    if teacher_logprob is None:
        _refuse("teacher_logprob is missing")
    k = teacher_id.shape[1]
    tid = _operand("teacher_id", teacher_id, (rows, k), (_I32,), device)
    tlp = _operand("teacher_logprob", teacher_logprob, (rows, k), _DTYPES, device)
    return k, tid, tlp, _DTYPES[teacher_logprob.dtype]


def token_scores(logits, labels=None, *, top_k=0, temperature=1.0, entropy=True, stats=False) -> TokenScores:
    """Log probability of `labels` (i32, negative = none), entropy and the `top_k` alternatives."""
    rows, vocab, pitch, code, dev = _matrix("logits", logits)
    if not 0 <= top_k <= min(TOP_K_MAX, vocab):
        _refuse(f"top_k must be 0..{TOP_K_MAX} and at most the vocabulary (got {top_k})")
    lab = _operand("labels", labels, (rows,), (_I32,), dev)
    where = logits.device
    logprob = torch.empty(rows, dtype=_F32, device=where) if lab is not None else None
    ent = torch.empty(rows, dtype=_F32, device=where) if entropy else None
    st = torch.empty(rows, 2, dtype=_F32, device=where) if stats else None
    top_lp = torch.empty(rows, top_k, dtype=_F32, device=where) if top_k else None
    top_id = torch.empty(rows, top_k, dtype=_I32, device=where) if top_k else None
    d = L.TokenScores(logits.data_ptr(), lab, logprob.data_ptr() if lab is not None else None,
                      ent.data_ptr() if entropy else None, st.data_ptr() if stats else None,
                      top_lp.data_ptr() if top_k else None, top_id.data_ptr() if top_k else None, rows, vocab, pitch, code,
                      top_k, temperature, 0)
    _call(L.lib().seeml_b200_token_scores_fwd, d, dev)
    return TokenScores(logprob, ent, st, top_lp, top_id)


def token_scores_backward(logits, labels, stats, entropy, dlogprob, dentropy, *, temperature=1.0, out=None):
    """Gradient of sum(dlogprob * logprob + dentropy * entropy); `out` may be the logits."""
    rows, vocab, pitch, code, dev = _matrix("logits", logits)
    lab = _operand("labels", labels, (rows,), (_I32,), dev)
    st = _operand("stats", stats, (rows, 2), (_F32,), dev)
    ent = _operand("entropy", entropy, (rows,), (_F32,), dev)
    dlp = _operand("dlogprob", dlogprob, (rows,), (_F32,), dev)
    dent = _operand("dentropy", dentropy, (rows,), (_F32,), dev)
    g, g_pitch = _gradient(logits, out)
    d = L.TokenScoresGrad(logits.data_ptr(), lab, st, ent, dlp, dent, g.data_ptr(), rows, vocab, pitch, g_pitch, code,
                          temperature)
    _call(L.lib().seeml_b200_token_scores_bwd, d, dev, out)
    return g


def distill_topk(logits, teacher_id, teacher_logprob, *, row_weight=None, scale=1.0, temperature=1.0, tail=False,
                 grad=False, saved=False, out=None) -> DistillLoss:
    """Loss against a teacher's top entries, with its gradient (`grad`, into `out` when given, which
    may be the logits) or with what `distill_topk_backward` needs (`saved`)."""
    rows, vocab, pitch, code, dev = _matrix("logits", logits)
    k, tid, tlp, tcode = _teacher(teacher_id, teacher_logprob, rows, dev)
    w = _operand("row_weight", row_weight, (rows,), (_F32,), dev)
    where = logits.device
    row_loss = torch.empty(rows, dtype=_F32, device=where)
    loss = row_loss.new_empty(())
    keep = torch.empty(rows, 4, dtype=_F32, device=where) if saved else None
    g, g_pitch = _gradient(logits, out) if grad or out is not None else (None, vocab)
    d = L.DistillTopk(logits.data_ptr(), tid, tlp, w, row_loss.data_ptr(), loss.data_ptr(),
                      keep.data_ptr() if saved else None, g.data_ptr() if g is not None else None, rows, vocab, pitch,
                      g_pitch, code, tcode, k, 1 if tail else 0, temperature, scale)
    _call(L.lib().seeml_b200_distill_topk_fwd, d, dev, out)
    return DistillLoss(loss, row_loss, keep, g)


def distill_topk_backward(logits, teacher_id, teacher_logprob, saved, drow_loss, *, temperature=1.0, tail=False, out=None):
    """Gradient of sum(drow_loss * row_loss) from the forward call's `saved`; `out` may be the logits."""
    rows, vocab, pitch, code, dev = _matrix("logits", logits)
    k, tid, tlp, tcode = _teacher(teacher_id, teacher_logprob, rows, dev)
    sv = _operand("saved", saved, (rows, 4), (_F32,), dev)
    up = _operand("drow_loss", drow_loss, (rows,), (_F32,), dev)
    g, g_pitch = _gradient(logits, out)
    d = L.DistillTopkGrad(logits.data_ptr(), tid, tlp, sv, up, g.data_ptr(), rows, vocab, pitch, g_pitch, code, tcode, k,
                          1 if tail else 0, temperature, 0)
    _call(L.lib().seeml_b200_distill_topk_bwd, d, dev, out)
    return g
