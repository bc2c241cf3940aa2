"""Checks of the policy-head operators that run on either backend (tests/test_ops.py: CPU, tests/test_gpu_ops.py: GPU),
against the float64 statements of ops_reference.py.

Tolerances are bounds by arithmetic: the result's own rounding (half a step of its type) plus what float32 arithmetic
can lose on the way, a count of roundings times 2^-24 of the magnitudes that are added up."""
import numpy as np
import torch

import ops_reference as ref
from factory_marl_amd import ops

E32 = 2.0**-24
TINY = {"float32": 2.0**-149, "float16": 2.0**-25, "bfloat16": 2.0**-134}  # half the smallest step (float32: all of it)
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def name(t):
    return str(t.dtype).replace("torch.", "")


def np64(t):
    return t.detach().double().cpu().numpy()


def within(got, want, slack):
    """got (a tensor) is want rounded to got's type, give or take slack (absolute)"""
    g = np64(got)
    assert g.shape == want.shape, (g.shape, want.shape)
    bound = ref.HALF_STEP[name(got)] * (np.abs(want) + slack) + slack + TINY[name(got)]
    off = np.abs(g - want)
    bad = ~((off <= bound) | (np.isnan(g) & np.isnan(want)) | (g == want))
    assert not bad.any(), (int(bad.sum()), g[bad][:4], want[bad][:4], np.broadcast_to(bound, g.shape)[bad][:4])


# ------------------------------------------------------------------ layer norm
def norm_inputs(rows, cols, dtype, param, device, seed=0, offset=1.0):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(rows, cols, generator=g) * 1.5 + offset * torch.randn(rows, 1, generator=g)).to(dtype).to(device)
    w = (1 + 0.3 * torch.randn(cols, generator=g)).to(param).to(device)
    b = (0.3 * torch.randn(cols, generator=g)).to(param).to(device)
    dy = torch.randn(rows, cols, generator=g).to(dtype).to(device)
    return x, w, b, dy


def check_norm(x, w, b, dy, eps=1e-5):
    """forward and every gradient.  Roundings counted: a row's sums are taken over at most cols / 64 + 16 partial sums
    in sequence, the rest is a handful of operations; a column's over rows / 64 + 16 (a sequence within a stretch of
    rows, then one over the stretches)."""
    leaves = [t.clone().requires_grad_() if t is not None else None for t in (x, w, b)]
    y = ops.layer_norm(*leaves, eps=eps)
    assert y.dtype == x.dtype and y.shape == x.shape
    y0 = ops.layer_norm(x, w, b, eps=eps)
    assert torch.equal(y0, y.detach())
    X, W, B, D = (None if t is None else np64(t).reshape(-1, t.shape[-1]) if t is x or t is dy else np64(t) for t in (x, w, b, dy))
    want, h, rstd = ref.layer_norm(X, W, B, eps)
    n, v = X.shape
    aw = np.ones(v) if W is None else np.abs(W)
    size = (np.abs(X).mean(1, keepdims=True) + np.abs(X)) * rstd  # what x - mean is the difference of
    k = v / 64 + 32
    dh = k * E32 * (size + np.abs(h))  # error of h: of mean, of the difference, of rstd (relative)
    within(y.reshape(n, v), want, dh * aw + 4 * E32 * (np.abs(want) + (0 if B is None else np.abs(B))))
    grads = torch.autograd.grad(y, [t for t in leaves if t is not None], dy)
    dx, dw, db = ref.layer_norm_backward(X, W, D, eps)
    g = np.abs(D) * aw
    mg, mgh = g.mean(1, keepdims=True), (g * np.abs(h)).mean(1, keepdims=True)
    slack = rstd * (k * E32 * (g + mg + np.abs(h) * mgh) + dh * mgh + np.abs(h) * (g * dh).mean(1, keepdims=True))
    within(grads[0].reshape(n, v), dx, 2 * slack)
    kr = n / 64 + 32
    if w is not None:
        within(grads[1], dw, (np.abs(D) * dh).sum(0) + kr * E32 * np.abs(D * h).sum(0))
    if b is not None:
        within(grads[-1], db, kr * E32 * np.abs(D).sum(0))
    return y, grads


# ------------------------------------------------------------------ drawing categories
def check_sample(z, u, mask=None, **settings):
    got = ops.sample_logits(z, u, mask=mask, **settings)
    assert got.dtype == torch.int64 and got.shape == z.shape[:-1]
    v = z.shape[-1]
    sets = {k: (np64(s).reshape(-1) if torch.is_tensor(s) else s) for k, s in settings.items()}
    m = None if mask is None else np.broadcast_to(mask.cpu().numpy(), tuple(z.shape)).reshape(-1, v)
    want = ref.sample(np64(z).reshape(-1, v), np64(u).reshape(-1), mask=m, **sets)
    g = got.cpu().numpy().reshape(-1)
    bad = np.flatnonzero(g != want)
    assert len(bad) == 0, (len(bad), bad[:4], g[bad][:4], want[bad][:4], settings)
    return got


# ------------------------------------------------------------------ distillation
def distill_inputs(rows, cols, k, dtype, device, seed=0, padded=False, index=torch.int64):
    g = torch.Generator().manual_seed(seed)
    z = (torch.randn(rows, cols, generator=g) * 2).to(dtype)
    at = torch.stack([torch.randperm(cols, generator=g)[:k] for _ in range(rows)]) if rows else torch.zeros(0, k, dtype=torch.int64)
    t = torch.randn(rows, k, generator=g) * 3
    if padded and rows:
        at[torch.arange(k) >= torch.randint(0, k + 1, (rows, 1), generator=g)] = -1
    return z.to(device), at.to(index).to(device), t.to(device), torch.randn(rows, generator=g).to(device)


def check_distill(z, index, teacher, grad, temperature=1.0):
    """loss and gradient.  q = exp((z - largest) / T) / sum: the exponent is off by 3 roundings of itself, the sum by
    cols / 64 + 16; p likewise over k"""
    leaf = z.clone().requires_grad_()
    loss = ops.distill_loss(leaf, index, teacher, temperature=temperature)
    assert loss.dtype == torch.float32 and loss.shape == z.shape[:-1]
    assert torch.equal(ops.distill_loss(z, index, teacher, temperature=temperature).nan_to_num(7e7), loss.detach().nan_to_num(7e7))
    v, k = z.shape[-1], index.shape[-1]
    Z, A, T, G = np64(z).reshape(-1, v), index.cpu().numpy().reshape(-1, k), np64(teacher).reshape(-1, k), np64(grad).reshape(-1)
    want, dz = ref.distill(Z, A, T, temperature, G)
    with np.errstate(invalid="ignore"):
        fin = np.where(np.isfinite(Z), Z, 0)
        span = (np.abs(fin).max(1) * 2 / temperature)[:, None]
        tspan = np.where(np.isfinite(T), np.abs(T), 0).max(1) * 2 / temperature
        count = (v + k) / 64 + 64
        rel = E32 * (4 * span + 4 * tspan[:, None] + count)  # relative error of q and of p
        # loss = T^2 sum p (log p - log q): errors of p weigh the logs' size, errors of log sum come through whole
        logs = 4 * span[:, 0] + 4 * tspan + np.log(v * k + 1) + 1
        within(loss.reshape(-1), want, temperature**2 * rel[:, 0] * logs)
        got = torch.autograd.grad(loss, leaf, grad)[0]
        assert got.dtype == z.dtype and got.shape == z.shape
        x = fin / temperature
        q = np.exp(x - x.max(1, keepdims=True))
        q /= q.sum(1, keepdims=True)
        p = np.abs(dz / np.where(G == 0, 1, G * temperature)[:, None] - q) + q  # at least what is subtracted
        within(got.reshape(-1, v), dz, np.nan_to_num(np.abs(G)[:, None] * temperature * rel * (q + p) * 2, nan=0.0))
    return loss, got
