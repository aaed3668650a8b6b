"""Vocabulary-row operators written from their definitions in 64 bits (CPU), with the rounding
bounds that the f32 kernels are held to.

u = 2^-24 (half an f32 step). Bounds, for rows of V logits:
  delta   relative error of a row's exponential sum: an exponent (x - m) / T carries three
          roundings, so exp is off by 3 |y| u (y = (x - m) / T; weighted by p, sum p |y| <= ln V <= 14)
          plus 4 u for the exponential itself; a thread adds at most V / 128 terms in f32, u each.
          V / 128 + 64 covers 3 * 14 + 4 + the few partial sums.
  an element's exponential: 3 |y| u + 4 u, and 6 u for the factors it is multiplied with."""
import math

import numpy as np
import torch

U = 2.0 ** -24


def delta(V):
    return (V / 128 + 64) * U


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def floor_of(dtype):
    """Half a step at the bottom of the type's range, where steps stop shrinking."""
    return 2.0 ** -25 if dtype == torch.float16 else 2.0 ** -126


def scores(x, labels, k, T):
    """x: [rows, V] f64. Returns logprob, entropy, top_logprob, top_id."""
    rows, V = x.shape
    out_lp, out_h = np.zeros(rows), np.zeros(rows)
    tlp, tid = np.zeros((rows, k)), np.zeros((rows, k), np.int64)
    for r in range(rows):
        v = x[r]
        bad = np.isnan(v).any() or np.isposinf(v).any()
        empty = not bad and np.isneginf(v).all()
        if bad:
            lp = np.full(V, np.nan)
            out_h[r] = np.nan
        elif empty:
            lp = np.full(V, -np.inf)
        else:
            y = (v - v.max()) / T
            lp = y - math.log(np.exp(y).sum())
            p = np.exp(lp)
            out_h[r] = -np.sum(np.where(p > 0, p * np.where(p > 0, lp, 0.0), 0.0))
        if labels is not None and labels[r] >= 0:
            out_lp[r] = lp[labels[r]] if labels[r] < V else np.nan
        if k:
            key = np.where(np.isnan(v), np.inf, v)
            order = np.lexsort((np.arange(V), -key, ~np.isnan(v)))[:k]
            tid[r], tlp[r] = order, lp[order]
    return out_lp, out_h, tlp, tid


def scores_grad(x, labels, gl, gh, T):
    """Gradient and its bound's scale, [rows, V] each (finite rows with some unmasked token)."""
    m = x.max(1, keepdims=True)
    y = (x - m) / T
    lse = np.log(np.exp(y).sum(1, keepdims=True))
    lp = y - lse
    p = np.exp(lp)
    plp = np.where(p > 0, p * np.where(p > 0, lp, 0.0), 0.0)
    H = -plp.sum(1, keepdims=True)
    gl = np.where(labels >= 0, gl, 0.0)[:, None]
    gh = gh[:, None]
    g = -gl * p - gh * (plp + p * H)
    there = labels >= 0
    g[there, labels[there]] += gl[there, 0]
    V = x.shape[1]
    size = p * (np.abs(gl) + np.abs(gh) * (np.abs(np.where(p > 0, lp, 0.0)) + np.abs(H)))
    rel = delta(V) * 2 + (3 * np.where(p > 0, -y, 0.0) + 16) * U
    # the entropy that the gradient reads is itself rounded; the label's own 1 - p is not a difference
    err = size * rel + np.abs(gh) * p * (2 + math.log(V)) * 2 * delta(V)
    err[there, labels[there]] += 4 * U * np.abs(gl[there, 0])
    return g / T, err / T


def distill(x, ids, vals, T, tail):
    """Row losses and d row_loss / dx with their bounds, for rows whose entries are valid."""
    rows, V = x.shape
    loss, loss_err = np.zeros(rows), np.zeros(rows)
    grad, grad_err = np.zeros((rows, V)), np.zeros((rows, V))
    for r in range(rows):
        keep = ids[r] >= 0
        i, v = ids[r][keep], vals[r][keep]
        target = np.zeros(V)
        if tail:
            q = np.exp(v)
            rest = max(0.0, 1.0 - q.sum())
        else:
            top = v.max() if v.size else -np.inf
            q = np.exp(v - top) / np.exp(v - top).sum() if np.isfinite(top) else np.zeros(v.size)
            rest = 0.0
        np.add.at(target, i, q)
        named = np.zeros(V, bool)
        named[i] = True
        if np.isneginf(x[r]).all():
            loss[r] = np.inf if q.sum() > 0 else 0.0
            continue
        y = (x[r] - x[r].max()) / T
        log_sum = math.log(np.exp(y).sum())
        lp = y - log_sum
        p = np.exp(lp)
        unnamed = np.where(named, -np.inf, y)
        if np.isneginf(unnamed).all():
            rest, share = 0.0, np.zeros(V)
            lp_rest = 0.0
        else:
            top = unnamed.max()
            e = np.exp(unnamed - top)
            lp_rest = top + math.log(e.sum()) - log_sum
            share = e / e.sum()
        Q = q.sum() + rest
        with np.errstate(divide="ignore", invalid="ignore"):
            terms = np.where(q > 0, q * (np.log(q) - lp[i]), 0.0)
        loss[r] = terms.sum() + (rest * (math.log(rest) - lp_rest) if rest > 0 else 0.0)
        loss_err[r] = Q * 2 * delta(V) + abs(loss[r]) * U if np.isfinite(loss[r]) else 0.0
        grad[r] = (p * Q - target - rest * share) / T
        rel = 2 * delta(V) + (3 * np.where(p > 0, -y, 0.0) + 16) * U
        grad_err[r] = ((p * Q + rest * share) * rel + target * 4 * U) / T
    return loss, loss_err, grad, grad_err
