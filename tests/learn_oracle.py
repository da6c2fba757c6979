"""Plain 64-bit numpy implementations of the language-model training operators (group norm,
router, expert sort/dispatch/combine, distillation), written from their definitions for the
tests of the kernels and of the host layer."""
import math

import numpy as np

f64 = np.float64


def _erf(x):
    return np.vectorize(math.erf, otypes=[f64])(x)


def act(v, name):
    if name == "relu":
        return np.where(v > 0, v, 0.0)
    if name == "silu":
        return v / (1 + np.exp(-v))
    if name == "gelu":
        return v * 0.5 * (1 + _erf(v / math.sqrt(2)))
    return v


def act_slope(v, name):
    if name == "relu":
        return (v > 0).astype(f64)
    if name == "silu":
        s = 1 / (1 + np.exp(-v))
        return s * (1 + v * (1 - s))
    if name == "gelu":
        return 0.5 * (1 + _erf(v / math.sqrt(2))) + v * np.exp(-v * v / 2) / math.sqrt(2 * math.pi)
    return np.ones_like(v)


def group_norm(x, gamma, beta, groups, eps, name, dy=None):
    """x [B, L, C]. Returns y, mean, rstd, and with dy also dx, dgamma, dbeta."""
    x = x.astype(f64)
    b, n, c = x.shape
    gamma = np.ones(c) if gamma is None else gamma.astype(f64)
    beta = np.zeros(c) if beta is None else beta.astype(f64)
    g = x.reshape(b, n, groups, c // groups)
    mean = g.mean(axis=(1, 3), keepdims=True)
    var = ((g - mean) ** 2).mean(axis=(1, 3), keepdims=True)
    with np.errstate(divide="ignore", invalid="ignore"):
        rstd = 1 / np.sqrt(var + eps)
        xh = ((g - mean) * rstd).reshape(b, n, c)
    v = xh * gamma + beta
    res = [act(v, name), mean.reshape(b, groups), rstd.reshape(b, groups)]
    if dy is None:
        return res
    dv = dy.astype(f64) * act_slope(v, name)
    a = (dv * gamma).reshape(g.shape)
    xg = xh.reshape(g.shape)
    dx = rstd * (a - a.mean(axis=(1, 3), keepdims=True) - xg * (a * xg).mean(axis=(1, 3), keepdims=True))
    return res + [dx.reshape(x.shape), (dv * xh).sum(axis=(0, 1)), dv.sum(axis=(0, 1))]


def route(logits, k, renorm, dw=None):
    z = logits.astype(f64)
    t, e = z.shape
    # NaN first, then larger first, then the lower expert
    rank = np.lexsort((np.broadcast_to(np.arange(e), z.shape), -np.where(np.isnan(z), 0, z), ~np.isnan(z)), axis=1)
    ids = rank[:, :k].astype(np.int64)
    picked = np.take_along_axis(z, ids, 1)
    ids = np.where(picked == -np.inf, -1, ids)
    w = np.zeros((t, k))
    dl = np.zeros((t, e))
    for i in range(t):
        held = ids[i] >= 0
        if not held.any():
            continue
        with np.errstate(invalid="ignore", over="ignore"):
            over = picked[i][held] if renorm else z[i]
            ex = np.exp(over - picked[i][0])
            w[i, held] = np.exp(picked[i][held] - picked[i][0]) / ex.sum()
        if dw is not None:
            dot = (w[i] * dw[i])[held].sum()
            if renorm:
                dl[i, ids[i][held]] = w[i][held] * (dw[i][held] - dot)
            else:
                up = np.zeros(e)
                up[ids[i][held]] = dw[i][held]
                dl[i] = ex / ex.sum() * (up - dot)
    return (w, ids) if dw is None else (w, ids, dl)


def expert_sort(ids, experts, capacity):
    """slot, src, counts, offsets, written choice by choice."""
    flat = ids.reshape(-1)
    counts = np.zeros(experts, np.int64)
    for e in flat:
        if 0 <= e < experts:
            counts[e] += 1
    offsets = np.arange(experts + 1) * capacity if capacity else np.concatenate([[0], np.cumsum(counts)])
    rows = experts * capacity if capacity else flat.size
    slot, src, used = np.full(flat.size, -1), np.full(rows, -1), np.zeros(experts, np.int64)
    for i, e in enumerate(flat):
        if 0 <= e < experts:
            if not capacity or used[e] < capacity:
                slot[i] = offsets[e] + used[e]
                src[slot[i]] = i
            used[e] += 1
    return slot.reshape(ids.shape), src, counts, offsets


def dispatch(x, slot, rows):
    out = np.zeros((rows, x.shape[1]), f64)
    for t in range(slot.shape[0]):
        for r in slot[t]:
            if r >= 0:
                out[r] = x[t]
    return out


def combine(rows, weights, slot, dout=None):
    t, k = slot.shape
    w = np.ones((t, k)) if weights is None else weights.astype(f64)
    rows = rows.astype(f64)
    out = np.zeros((t, rows.shape[1]))
    dw, drows = np.zeros((t, k)), np.zeros_like(rows)
    for i in range(t):
        for j in range(k):
            r = slot[i, j]
            if r >= 0:
                out[i] += w[i, j] * rows[r]
                if dout is not None:
                    dw[i, j] = dout[i].astype(f64) @ rows[r]
                    drows[r] = w[i, j] * dout[i]
    return out if dout is None else (out, drows, dw)


def distill(z, ids, teacher, tau, teacher_lse=None, dloss=None):
    """loss [R] and, with dloss, dz [R, V]."""
    r, v = z.shape
    z64 = z.astype(f64)
    loss, dz = np.zeros(r), np.zeros((r, v))
    with np.errstate(divide="ignore", invalid="ignore", over="ignore"):
        for i in range(r):
            held = (ids[i] >= 0) & (ids[i] < v)
            at, t = ids[i][held], teacher[i][held].astype(f64)
            if not held.any() or (teacher_lse is None and np.all(t == -np.inf)):
                continue
            m = z64[i].max()
            logq = (z64[i] - m) / tau - np.log(np.exp((z64[i] - m) / tau).sum())
            if teacher_lse is None:
                logp = (t - t.max()) / tau - np.log(np.exp((t - t.max()) / tau).sum())
            else:
                logp = t / tau - f64(teacher_lse[i])
            p = np.exp(logp)
            loss[i] = sum(a * (b - logq[c]) for a, b, c in zip(p, logp, at) if a != 0)
            outside = np.ones(v, bool)
            outside[at] = False
            pt = 0.0
            if teacher_lse is not None:
                pt = max(0.0, 1 - p.sum())
                if pt > 0:
                    zo = z64[i][outside]
                    mo = zo.max() if zo.size else 0.0  # no column outside: log 0
                    log_sum = np.log(np.exp((z64[i] - m) / tau).sum())
                    log_tail = (mo - m) / tau + np.log(np.exp((zo - mo) / tau).sum()) - log_sum
                    loss[i] += pt * (np.log(pt) - log_tail)
            loss[i] *= tau * tau
            if dloss is not None:
                q = np.exp(logq)
                g = (p.sum() + pt) * q
                np.subtract.at(g, at, p)
                if pt > 0 and outside.any():
                    g[outside] -= pt * np.exp(logq[outside] - log_tail)
                dz[i] = tau * f64(dloss[i]) * g
    return loss if dloss is None else (loss, dz)
