"""The policy-head operators written out in float64 numpy, row by row: what tests/test_ops.py and tests/test_gpu_ops.py
compare with.  Nothing here uses the library."""
import math

import numpy as np

HALF_STEP = {"float32": 2.0**-24, "float16": 2.0**-11, "bfloat16": 2.0**-8}  # of a value, half the type's step


def layer_norm(x, weight, bias, eps):
    x = np.asarray(x, np.float64)
    mean = x.mean(1, keepdims=True)
    rstd = 1 / np.sqrt(((x - mean) ** 2).mean(1, keepdims=True) + eps)
    h = (x - mean) * rstd
    return h * (1 if weight is None else weight) + (0 if bias is None else bias), h, rstd


def layer_norm_backward(x, weight, dy, eps):
    """dx, dweight, dbias"""
    _, h, rstd = layer_norm(x, None, None, eps)
    dy = np.asarray(dy, np.float64)
    g = dy if weight is None else dy * weight
    dx = rstd * (g - g.mean(1, keepdims=True) - h * (g * h).mean(1, keepdims=True))
    return dx, (dy * h).sum(0), dy.sum(0)


def sample_row(z, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, mask=None):
    z = np.asarray(z, np.float64)
    at = np.arange(len(z)) if mask is None else np.flatnonzero(mask)
    if any(math.isnan(v) for v in (u, temperature, top_p, min_p)) or np.isnan(z[at]).any():
        return -1
    at = at[z[at] > -np.inf]
    if len(at) == 0:
        return -1
    at = at[np.argsort(-z[at], kind="stable")]
    if temperature <= 0:
        return int(at[0])
    top = z[at[0]]
    with np.errstate(invalid="ignore", over="ignore", divide="ignore"):
        x = np.where(z[at] == top, 0.0, np.nan_to_num((z[at] - top) / temperature, nan=-np.inf, neginf=-np.inf))
    w = np.exp(x.astype(np.longdouble))
    if top_k > 0:
        w = w[:top_k]
    if top_p < 1:
        before = np.concatenate([[0], np.cumsum(w)[:-1]])
        # the share of the weight is a float64 product: of n equal weights, top_p = 0.8 keeps 0.8 n where that is whole.
        # (0.8 as a float64 is 4e-17 more than 0.8; in wider arithmetic than the operator states it would keep one more.)
        keep = before < float(top_p) * float(w.sum())
        keep[0] = True
        w = w[keep]
    w = w[w >= min(min_p, 1.0)]
    c = np.cumsum(w)
    return int(at[min(int((c <= u * c[-1]).sum()), int((w > 2.0**-46).sum()) - 1)])


def sample(z, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, mask=None):
    n = len(z)
    sets = [np.broadcast_to(np.asarray(s, np.float64), (n,)) for s in (temperature, top_k, top_p, min_p)]
    return np.array([sample_row(z[i], float(u[i]), sets[0][i], int(sets[1][i]), sets[2][i], sets[3][i],
                                None if mask is None else mask[i]) for i in range(n)], np.int64)


def distill(z, index, teacher, temperature, grad=None):
    """loss [rows], and with grad the gradient of the logits"""
    z, teacher, T = np.asarray(z, np.float64), np.asarray(teacher, np.float64), temperature
    loss, dz = np.zeros(len(z)), np.zeros(z.shape)
    for i in range(len(z)):
        there = (index[i] >= 0) & (teacher[i] > -np.inf)
        if (index[i] >= z.shape[1]).any():
            loss[i], dz[i] = np.nan, np.nan
            continue
        if not there.any():
            continue
        at, t = index[i][there], teacher[i][there] / T
        logp = t - t.max() - np.log(np.exp(t - t.max()).sum())
        x = z[i] / T
        logq = x - x.max() - np.log(np.exp(x - x.max()).sum())
        loss[i] = T * T * (np.exp(logp) * (logp - logq[at])).sum()
        if grad is not None:
            d = np.exp(logq)
            np.subtract.at(d, at, np.exp(logp))
            dz[i] = grad[i] * T * d
    return loss if grad is None else (loss, dz)
