"""Distributions over a vocabulary in 64 bits: the definitions that the kernels of
dizo_amd.token_loss are held to. Rows of logits (n, v) as float64 arrays."""
from __future__ import annotations

import numpy as np


def log_softmax(x: np.ndarray) -> np.ndarray:
    """NaN for a row with NaN or +inf, and for one with nothing above -inf."""
    x = np.asarray(x, dtype=np.float64)
    out = np.full(x.shape, np.nan)
    for r in range(x.shape[0]):
        m = x[r].max(initial=-np.inf)
        if np.isfinite(m):
            y = x[r] - m
            out[r] = y - np.log(np.exp(y).sum())
    return out


def entropy(logq: np.ndarray) -> np.ndarray:
    q = np.exp(logq)
    return -np.where(q > 0, q * np.where(q > 0, logq, 0.0), np.where(np.isnan(q), np.nan, 0.0)).sum(-1)


def token_logprobs(x, tokens, top=0, ignore=-100):
    """(logprobs, entropy, top_logprobs, top_tokens) of rows x and their tokens."""
    n, v = x.shape
    logq = log_softmax(x)
    lp, ent = np.zeros(n), np.zeros(n)
    tlp, ttok = np.full((n, top), -np.inf), np.full((n, top), -1, dtype=np.int64)
    h = entropy(logq)
    for r in range(n):
        t = int(tokens[r])
        if t == ignore:
            continue
        lp[r] = logq[r, t] if 0 <= t < v else np.nan
        ent[r] = h[r]
        if top:
            if np.isnan(logq[r]).any():
                tlp[r] = np.nan
            else:
                ttok[r] = np.argsort(-x[r], kind="stable")[:top]
                tlp[r] = logq[r][ttok[r]]
    return lp, ent, tlp, ttok


def token_logprobs_grad(x, tokens, weights, entropy_weights, ignore=-100):
    """Gradient of sum(weights logprobs) + sum(entropy_weights entropy) with respect to x."""
    n, v = x.shape
    logq = log_softmax(x)
    q, h = np.exp(logq), entropy(logq)
    out = np.zeros((n, v))
    for r in range(n):
        t = int(tokens[r])
        if t == ignore:
            continue
        if not 0 <= t < v:
            out[r] = np.nan
            continue
        out[r] = -weights[r] * q[r] - entropy_weights[r] * np.where(q[r] > 0, q[r] * (np.where(q[r] > 0, logq[r], 0) + h[r]), q[r])
        out[r, t] += weights[r]
    return out


def teacher_weights(values, tokens, v, temperature, normalize):
    """(w, log w) of a row's entries; NaN where they make no distribution."""
    there = tokens != -1
    t = np.where(there, np.asarray(values, dtype=np.float64), -np.inf) / (temperature if normalize else 1.0)
    bad = (there & ((tokens < 0) | (tokens >= v) | ~(t < np.inf))).any()
    if normalize:
        with np.errstate(invalid="ignore", divide="ignore"):
            m = t.max()
            logw = t - m - np.log(np.exp(t - m).sum())
        bad = bad or not np.isfinite(m)
    else:
        logw = t
    if bad:
        return np.full(t.shape, np.nan), np.full(t.shape, np.nan)
    return np.exp(logw), logw


def topk_distill(x, values, tokens, temperature=1.0, normalize=True, weights=None):
    """loss (n,), and with weights the gradient of sum(weights loss) with respect to x."""
    n, v = x.shape
    logq = log_softmax(np.asarray(x, dtype=np.float64) / temperature)
    loss, grad = np.zeros(n), np.zeros((n, v))
    for r in range(n):
        at = np.asarray(tokens[r])
        if (at == -1).all():
            continue
        w, logw = teacher_weights(values[r], at, v, temperature, normalize)
        if np.isnan(w).any() or np.isnan(logq[r]).any():
            loss[r], grad[r] = np.nan, np.nan
            continue
        live = w > 0
        loss[r] = temperature**2 * (w[live] * (logw[live] - logq[r][at[live]])).sum()
        grad[r] = np.exp(logq[r]) * w.sum()
        np.subtract.at(grad[r], at[live], w[live])
        grad[r] *= temperature
    return (loss, None) if weights is None else (loss, grad * np.asarray(weights)[:, None])
