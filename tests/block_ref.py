"""64-bit statements of the recurrent-block operators and the error bounds of their tests.

The statements are vectorised over batch and channels and walk the sequence step by step,
forward and backward, from the operators' formulas (numpy, fp64).

Bounds.  A kernel computes in fp32 and rounds once.  Its result therefore differs from the
exact one by at most the unit roundoff of the stored type (2^-24, 2^-11 and 2^-8 for fp32,
fp16 and bf16) relative to the value, plus the error of the fp32 computation.  That error:
an approximate exponential or reciprocal is within 2^-21 relative, and a recurrence whose
weights sum to one (a + c = 1) keeps errors relative to its largest term; roundings of
independent steps over a memory of n steps grow like sqrt(n) 2^-24, below 2^-19 for the
n <= 1000 or so of these gates.  2^-18 of the largest value leaves room for the handful of
factors of a gradient.  Sums over rows (bias and weight gradients) are bounded relative to
the sum of the magnitudes.
"""

from __future__ import annotations

import numpy as np
import torch

UNIT = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 2.0 ** -126, torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -126}
COMPUTED = 2.0 ** -18


def wide(t):
    return None if t is None else t.detach().to("cpu", torch.float64).numpy()


def check(got, want, what, scale=None):
    """got within its type's rounding and the fp32 computation's error of want."""
    assert tuple(got.shape) == tuple(want.shape), what
    g = wide(got)
    assert np.isfinite(g).all() == np.isfinite(want).all(), what
    if not want.size:
        return
    top = np.abs(want).max() if scale is None else scale
    err = np.abs(g - want) - UNIT[got.dtype] * np.abs(want) - COMPUTED * top - TINY[got.dtype]
    assert err.max() <= 0.0, f"{what}: off by {np.abs(g - want).max()} at a scale of {top} ({err.max()} over the bound)"


def sigmoid(v):
    return 1.0 / (1.0 + np.exp(-v))


def recurrence(x, gate, z=None, bias=None, ids=None, init=None, nstates=None):
    """Returns (out, final, h, prev): prev is the state each position starts from."""
    B, D, L = x.shape
    u = gate + (bias[:, None] if bias is not None else 0.0)
    a, c = sigmoid(u), sigmoid(-u)
    n = B if ids is None else (init.shape[0] if init is not None else nstates or 0)
    final = np.zeros((n, D)) if init is None else init.copy()
    h, prev = np.zeros((B, D, L)), np.zeros((B, D, L))
    for b in range(B):
        now = np.zeros(D)
        for t in range(L):
            k = b if ids is None else ids[b, t]
            if k < 0:
                continue
            if t == 0 or (ids is not None and ids[b, t - 1] != k):
                now = init[k] if init is not None and k < n else np.zeros(D)
            prev[b, :, t] = now
            now = a[b, :, t] * now + c[b, :, t] * x[b, :, t]
            h[b, :, t] = now
            if k < n and (t == L - 1 or (ids is not None and ids[b, t + 1] != k)):
                final[k] = now
    out = h if z is None else h * z * sigmoid(z)
    if ids is not None:
        out = np.where((ids >= 0)[:, None, :], out, 0.0)
    return out, final, h, prev


def recurrence_grads(x, gate, z, bias, ids, init, dout, dfinal, nstates=None):
    """dict of dx, dgate, dz, dbias, dinit, and bias_scale (the largest sum of |dgate|)."""
    B, D, L = x.shape
    _, _, h, prev = recurrence(x, gate, z, bias, ids, init, nstates)
    u = gate + (bias[:, None] if bias is not None else 0.0)
    a, c = sigmoid(u), sigmoid(-u)
    n = B if ids is None else (init.shape[0] if init is not None else nstates or 0)
    dx, dgate, dz = np.zeros_like(x), np.zeros_like(x), np.zeros_like(x)
    dinit = np.zeros((n, D)) if dfinal is None else dfinal.copy()
    for b in range(B):
        s = np.zeros(D)
        for t in range(L - 1, -1, -1):
            k = b if ids is None else ids[b, t]
            if k < 0:
                continue
            if t == L - 1 or (ids is not None and ids[b, t + 1] != k):
                s = dfinal[k] if dfinal is not None and k < n else np.zeros(D)
            dy = dout[b, :, t]
            g = dy
            if z is not None:
                zt = z[b, :, t]
                p = sigmoid(zt)
                g = dy * zt * p
                dz[b, :, t] = dy * h[b, :, t] * p * (1.0 + zt * (1.0 - p))
            g = g + s
            dx[b, :, t] = g * c[b, :, t]
            dgate[b, :, t] = g * (prev[b, :, t] - x[b, :, t]) * a[b, :, t] * c[b, :, t]
            s = a[b, :, t] * g
            if k < n and (t == 0 or (ids is not None and ids[b, t - 1] != k)):
                dinit[k] = s
    return {"dx": dx, "dgate": dgate, "dz": dz, "dbias": dgate.sum((0, 2)), "dinit": dinit,
            "bias_scale": np.abs(dgate).sum((0, 2)).max() if x.size else 0.0}


def philox_words(seed, offset, blocks):
    """Philox4x32-10 by its definition, in Python integers: (len(blocks), 4) words."""
    low = 0xFFFFFFFF
    out = []
    for block in blocks:
        c = [block & low, (block >> 32) & low, offset & low, (offset >> 32) & low]
        k = [seed & low, (seed >> 32) & low]
        for r in range(10):
            p0, p1 = 0xD2511F53 * c[0], 0xCD9E8D57 * c[2]
            c = [(p1 >> 32) ^ c[1] ^ k[0], p1 & low, (p0 >> 32) ^ c[3] ^ k[1], p0 & low]
            k = [(k[0] + 0x9E3779B9) & low, (k[1] + 0xBB67AE85) & low]
        out.append(c)
    return out


def add_norm(x, residual, weight, keep, p, eps, stored_dtype):
    """(out, residual_out): the stream is rounded to its type before it is normalised."""
    r = np.zeros_like(x) if residual is None else residual
    r = r + (x if keep is None else np.where(keep, x / (1.0 - p), 0.0))
    stored = torch.from_numpy(r).to(stored_dtype).double().numpy()
    inv = 1.0 / np.sqrt((stored ** 2).mean(-1, keepdims=True) + eps)
    return stored * inv * weight, r


def add_norm_grads(stored, weight, keep, p, eps, dout, dres):
    inv = 1.0 / np.sqrt((stored ** 2).mean(-1, keepdims=True) + eps)
    n = stored * inv
    q = dout * weight
    dr = dres + inv * (q - n * (q * n).mean(-1, keepdims=True))
    dx = dr if keep is None else np.where(keep, dr / (1.0 - p), 0.0)
    return {"dx": dx, "dresidual": dr, "dweight": (dout * n).sum(0), "weight_scale": np.abs(dout * n).sum(0).max()}
