"""64-bit restatements of the 4-bit linear layer and of the top-logit distillation loss, from their definitions, on the CPU.
Test infrastructure only."""
import math

import numpy as np


def unpack(q, k):
    """uint8 [out, ceil(k/2)] -> integer codes [out, k]."""
    q = np.asarray(q, dtype=np.int64)
    codes = np.empty((q.shape[0], 2 * q.shape[1]), dtype=np.int64)
    codes[:, 0::2], codes[:, 1::2] = q % 16, q // 16
    return codes[:, :k]


def weights(q, scales, zeros, group, k):
    """float64 [out, k]."""
    codes = unpack(q, k)
    s = np.asarray(scales, dtype=np.float64)
    z = np.full(s.shape, 8.0) if zeros is None else np.asarray(zeros, dtype=np.float64)
    g = np.arange(k) // group
    return (codes - z[:, g]) * s[:, g]


def linear(x, w, bias=None, relu=False):
    y = np.asarray(x, dtype=np.float64) @ w.T
    if bias is not None:
        y = y + np.asarray(bias, dtype=np.float64)
    return np.maximum(y, 0.0) if relu else y


def input_grad(gy, w, gate=None):
    g = np.asarray(gy, dtype=np.float64) @ w
    return g if gate is None else np.where(np.asarray(gate, dtype=np.float64) > 0, g, 0.0)


def _lse(v):
    if not len(v):
        return -math.inf
    m = v.max()
    if not np.isfinite(m):
        return m
    return m + math.log(np.exp(v - m).sum())


def distill_row(z, index, value, tau, lse=None):
    """(loss, gradient [V]) of one row; z, value float64 arrays, index integers (-1 = empty)."""
    z = np.asarray(z, dtype=np.float64)
    v = len(z)
    index = np.asarray(index)
    if ((index < -1) | (index >= v)).any():
        return math.nan, np.full(v, math.nan)
    live = index >= 0
    t = np.asarray(value, dtype=np.float64)[live] / tau
    idx = index[live]
    if not len(idx) or (lse is None and (t == -math.inf).all()):
        return 0.0, np.zeros(v)
    u = z / tau
    log_q = u - _lse(u)
    p = np.zeros(v)
    np.add.at(p, idx, np.exp(t - (_lse(t) if lse is None else float(lse))))
    named = np.zeros(v, dtype=bool)
    named[idx] = True
    terms = p[named] > 0
    loss = float((p[named][terms] * (np.log(p[named][terms]) - log_q[named][terms])).sum())
    target = p                                     # loss = constant - sum_i target_i log q_i: gradient sum(target) q - target
    if lse is not None:
        rest = max(0.0, 1.0 - float(np.exp(t - float(lse)).sum()))
        log_qr = _lse(log_q[~named])
        if rest > 0 and np.isfinite(log_qr):
            loss += rest * (math.log(rest) - log_qr)
            target = p + np.where(named, 0.0, rest * np.exp(log_q - log_qr))
    return tau * tau * loss, tau * (target.sum() * np.exp(log_q) - target)


def distill(z, index, value, tau, lse=None, grad_loss=None):
    """(loss [N], gradient [N, V]); one teacher row serves all rows."""
    n = len(z)
    loss, grad = np.empty(n), np.empty(np.shape(z))
    for i in range(n):
        j = i if len(index) == n else 0
        loss[i], grad[i] = distill_row(z[i], index[j], value[j], tau, None if lse is None else lse[j])
        if grad_loss is not None:
            grad[i] *= float(grad_loss[i])
    return loss, grad
