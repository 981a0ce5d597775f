"""64-bit statement of the selective recurrence, with a bound on the error of an fp32 kernel.

The statement walks the sequence step by step, forward and backward, from the formulas (numpy,
fp64).  Beside each value it carries the same expression of the magnitudes (H for h, G for the
gradient g of h: every product and sum of absolute values) and a first-order bound of the error
that fp32 makes of it.

An fp32 kernel takes s to 2^-21 relative (an approximate exponential and reciprocal within 2^-22,
and a handful of roundings).  a = exp(s A) is 2^v with v = s A log2(e): the hardware's 2^v is within
2^-22, the roundings of log2(e) A and of v move it by up to 2^-24 |v| ln 2 = 2^-24 |s A| each, and
the error of s by 2^-21 |s A|.  So a is within EPS (1 + |s A|) relative, EPS = 2^-20.  Each product
and sum after that rounds by 2^-24.  With b = s x B,

    E_t = a E_{t-1} + EPS ((1 + |s A|) a H_{t-1} + |b|) + 2^-23 H_t           (error of h)
    F_t = a_{t+1} F_{t+1} + EPS ((1 + |s A|) a_{t+1} G_{t+1} + |C dy|)        (error of g)

and the error of a sum of products is the sum of its factors' errors times the other factors,
plus EPS for the factors' own roundings and its additions: up to 256 states in a chain of 8 and
a tree, channels and positions in sums whose rounding is kept or that are short, all within EPS
of the sum of magnitudes.  SLACK = 2 covers what the first order leaves out.  A result is
finally rounded to its type: at most the type's unit roundoff relative.
"""

from __future__ import annotations

import numpy as np
import torch

from block_ref import TINY, UNIT, sigmoid, wide

EPS, SLACK = 2.0 ** -20, 2.0


def softplus(u):
    return np.maximum(u, 0.0) + np.log1p(np.exp(-np.abs(u)))


def _spread(t, dim):
    """(batch, groups, dstate, seqlen) -> (seqlen, batch, dim, dstate)"""
    return np.repeat(t, dim // t.shape[1], 1).transpose(3, 0, 1, 2)


def statement(v, ids=None, nstates=None, use_softplus=True):
    """v: dict of fp64 arrays x, delta, A, B, C and optionally D, z, bias, init, dout, dfinal; B and C
    with or without groups.  Returns {name: (value, bound)}: out, final and, with dout, the gradients."""
    x, delta, A = (v[k] for k in ("x", "delta", "A"))
    batch, dim, L = x.shape
    N = A.shape[1]
    grouped = v["B"].ndim == 4
    Bg, Cg = (v[k] if grouped else v[k][:, None] for k in ("B", "C"))
    groups = Bg.shape[1]
    time = lambda t: np.ascontiguousarray(t.transpose(2, 0, 1))  # noqa: E731
    x, u = time(x), time(delta)
    if v.get("bias") is not None:
        u = u + v["bias"]
    if ids is None:
        n, keys = batch, np.broadcast_to(np.arange(batch), (L, batch))
    else:
        n = v["init"].shape[0] if v.get("init") is not None else nstates or 0
        keys = ids.T
    valid = keys >= 0
    first = valid & np.concatenate([np.ones((1, batch), bool), keys[1:] != keys[:-1]])[:L]
    last = valid & np.concatenate([keys[1:] != keys[:-1], np.ones((1, batch), bool)])[:L]
    x, u = (np.where(valid[..., None], t, 0.0) for t in (x, u))
    s = softplus(u) if use_softplus else u
    Bf, Cf = (np.where(valid[..., None, None], _spread(t, dim), 0.0) for t in (Bg, Cg))
    init = v["init"] if v.get("init") is not None else np.zeros((n, dim, N))
    D = v["D"] if v.get("D") is not None else np.zeros(dim)
    a = np.exp(s[..., None] * A)
    b = (s * x)[..., None] * Bf
    rough = EPS * (1.0 + np.abs(s[..., None] * A))  # relative error of a
    shape = (L, batch, dim, N)
    h, H, E, prev, pH, pE = (np.zeros(shape) for _ in range(6))
    final, final_e = init.copy(), np.zeros_like(init)
    state = [np.zeros((dim, N))] * batch
    for bi in range(batch):
        p, P, e = np.zeros((dim, N)), np.zeros((dim, N)), np.zeros((dim, N))
        for t in range(L):
            if not valid[t, bi]:
                continue
            k = keys[t, bi]
            if first[t, bi]:
                p = init[k] if k < n else np.zeros((dim, N))
                P, e = np.abs(p), np.zeros((dim, N))
            at = a[t, bi]
            prev[t, bi], pH[t, bi], pE[t, bi] = p, P, e
            p = at * p + b[t, bi]
            e = at * e + rough[t, bi] * at * P + EPS * np.abs(b[t, bi]) + 2.0 ** -23 * (at * P + np.abs(b[t, bi]))
            P = at * P + np.abs(b[t, bi])
            h[t, bi], H[t, bi], E[t, bi] = p, P, e
            if last[t, bi] and k < n:
                final[k], final_e[k] = p, e
    del state
    y = (Cf * h).sum(-1) + D * x
    Y = (np.abs(Cf) * H).sum(-1) + np.abs(D * x)
    ye = (np.abs(Cf) * E).sum(-1) + EPS * Y
    back = lambda t: t.transpose(1, 2, 0)  # noqa: E731
    gate, slope = 1.0, None
    if v.get("z") is not None:
        z = np.where(valid[..., None], time(v["z"]), 0.0)
        p = sigmoid(z)
        gate, slope = z * p, p + z * p * (1.0 - p)
    mag = np.abs(gate)
    res = {"out": (back(y * gate), back(ye * mag + EPS * Y * mag)), "final": (final, final_e)}
    if v.get("dout") is None:
        return res
    dout = np.where(valid[..., None], time(v["dout"]), 0.0)
    if slope is not None:
        # silu' = p + z p (1 - p) may cancel: its own error is relative to its parts
        parts = p + np.abs(z) * p * (1.0 - p)
        res["dz"] = (back(dout * y * slope), back(np.abs(dout) * (ye * parts + EPS * Y * parts)))
    dy = dout * gate
    dye = EPS * np.abs(dy)
    g, G, F = np.zeros(shape), np.zeros(shape), np.zeros(shape)
    dfinal = v["dfinal"] if v.get("dfinal") is not None else np.zeros((n, dim, N))
    dinit, dinit_e = dfinal.copy(), np.zeros_like(dfinal)
    for bi in range(batch):
        c, cG, cF = (np.zeros((dim, N)) for _ in range(3))
        for t in range(L - 1, -1, -1):
            if not valid[t, bi]:
                continue
            k = keys[t, bi]
            if last[t, bi]:
                c = dfinal[k] if k < n else np.zeros((dim, N))
                cG, cF = np.abs(c), np.zeros((dim, N))
            cd = Cf[t, bi] * dy[t, bi][:, None]
            g[t, bi], G[t, bi] = c + cd, cG + np.abs(cd)
            F[t, bi] = cF + EPS * np.abs(cd) + 2.0 ** -23 * G[t, bi]
            at = a[t, bi]
            c, cG, cF = at * g[t, bi], at * G[t, bi], at * F[t, bi] + rough[t, bi] * at * G[t, bi]
            if first[t, bi] and k < n:
                dinit[k], dinit_e[k] = c, cF

    def per_group(t):  # (L, batch, dim, N) -> (batch, groups, N, L), summed over a group's channels
        t = t.reshape(L, batch, groups, dim // groups, N).sum(3).transpose(1, 2, 3, 0)
        return t if grouped else t[:, 0]

    sx, asx = (s * x)[..., None], np.abs(s * x)[..., None]
    res["dB"] = (per_group(g * sx), per_group(F * asx + 2 * EPS * G * asx))
    ady = np.abs(dy)[..., None]
    res["dC"] = (per_group(dy[..., None] * h), per_group(ady * E + 2 * EPS * ady * H))
    gb, GB = (g * Bf).sum(-1), (G * np.abs(Bf)).sum(-1)
    gbe = (F * np.abs(Bf)).sum(-1) + EPS * GB
    w, W = g * a * prev, G * a * pH
    we = F * a * pH + G * a * pE + 2 * rough * W
    res["dA"] = ((w * s[..., None]).sum((0, 1)), (we * np.abs(s)[..., None] + EPS * W * np.abs(s)[..., None]).sum((0, 1)))
    aA = np.abs(A)
    ds, DS = (w * A).sum(-1) + x * gb, (W * aA).sum(-1) + np.abs(x) * GB
    dse = (we * aA).sum(-1) + np.abs(x) * gbe + EPS * DS
    r = sigmoid(u) if use_softplus else 1.0
    du, due = ds * r, dse * r + EPS * DS * r
    res["ddelta"] = (back(du), back(due))
    res["dbias"] = (du.sum((0, 1)), (due + EPS * np.abs(du)).sum((0, 1)))
    dx, DX = s * gb + D * dy, np.abs(s) * GB + np.abs(D * dy)
    res["dx"] = (back(dx), back(np.abs(s) * gbe + EPS * DX + np.abs(D) * dye))
    res["dD"] = ((dy * x).sum((0, 1)), (2 * EPS * np.abs(dy * x)).sum((0, 1)))
    res["dinit"] = (dinit, dinit_e)
    return res


def check(got, expected, what):
    """got within its type's rounding and the fp32 computation's error of the statement's value."""
    want, bound = expected
    assert tuple(got.shape) == tuple(want.shape), what
    g = wide(got)
    assert np.isfinite(g).all() == np.isfinite(want).all(), what
    if not want.size:
        return
    err = np.abs(g - want) - UNIT[got.dtype] * np.abs(want) - (1 + UNIT[got.dtype]) * SLACK * bound - TINY[got.dtype]
    i = np.unravel_index(np.argmax(err), err.shape)
    assert err.max() <= 0.0, f"{what}: {g[i]} for {want[i]} at {i}, {err.max()} over a bound of {SLACK * bound[i]}"


def fp64(t):
    return {k: wide(x) for k, x in t.items() if x is None or isinstance(x, torch.Tensor)}
