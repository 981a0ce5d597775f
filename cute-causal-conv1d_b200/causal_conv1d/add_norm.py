"""The residual connection between two blocks: dropout, residual add and RMSNorm in one pass.

    residual_out = residual + keep x / (1 - dropout_p)
    out = residual_out / sqrt(mean(residual_out^2) + eps) * weight

The dropout mask ``keep`` is a function of a generator state and the place alone
(Philox4x32-10), recomputed by the backward and never stored.
"""

from __future__ import annotations

import torch
from causal_conv1d._abi import block as _block


def dropout_add_rms_norm_fwd_function(x, weight, residual, eps, dropout_p, rng_state, residual_in_fp32):
    """One forward pass.  Returns (out, residual_out), both with x's shape."""
    return _block.add_norm_fwd(x, weight, residual, eps, dropout_p, rng_state, residual_in_fp32)


def dropout_add_rms_norm_bwd_function(x_dtype, residual_out, weight, dout, dresidual_out, eps, dropout_p, rng_state,
                                      return_dx, return_dresidual, return_dweight):
    """One backward pass.  Returns (dx, dresidual, dweight), each None if not asked for.
    Without dropout dx and dresidual are equal, and one tensor if their dtypes are."""
    return _block.add_norm_bwd(x_dtype, residual_out, weight, dout, dresidual_out, eps, dropout_p, rng_state,
                               return_dx, return_dresidual, return_dweight)


def dropout_add_rms_norm_fn(x, weight, residual=None, eps=1e-5, dropout_p=0.0, rng_state=None,
                            residual_in_fp32=False):
    """Dropout of x, added to the residual stream, and the stream's RMSNorm.

    x: (..., dim) fp32, fp16 or bf16; weight: (dim,), any float dtype; residual: like x, in
    x's dtype or fp32 (None: the stream starts here, in x's dtype or, with
    residual_in_fp32, in fp32).  Returns (out, residual_out): out in x's dtype,
    residual_out in the stream's.  What is normalised is residual_out as stored.

    dropout_p: probability of dropping an element of x (0 outside training).  rng_state: (2,)
    int64 on x's device, a seed and an offset; the same state gives the same mask, whatever
    the strides (None draws one from the device's default generator).

    Gradients flow back to x, weight and residual.  There is no second derivative and no
    forward-mode one: both raise.
    """
    return _block.add_norm(x, weight, residual, eps, dropout_p, rng_state, residual_in_fp32)


def dropout_add_rms_norm_mask_ref(rows, dim, dropout_p, rng_state):
    """The (rows, dim) truth values of the kept elements, by Philox4x32-10 in 64-bit integer
    operations: element (row, col) takes word col % 4 of block row * ceil(dim / 4) + col // 4."""
    low = 0xFFFFFFFF
    per = -(-dim // 4)
    block = torch.arange(rows * per, device=rng_state.device, dtype=torch.int64)
    seed, offset = rng_state[0], rng_state[1]
    c0, c1, c2, c3 = block & low, block >> 32, offset & low, (offset >> 32) & low
    k0, k1 = seed & low, (seed >> 32) & low
    for _ in range(10):
        p0, p1 = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = ((p1 >> 32) & low) ^ c1 ^ k0, p1 & low, ((p0 >> 32) & low) ^ c3 ^ k1, p0 & low
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    words = torch.stack([c.expand_as(block) for c in (c0, c1, c2, c3)], -1).reshape(rows, 4 * per)[:, :dim]
    return words >= int(dropout_p * 4294967296.0)


def dropout_add_rms_norm_ref(x, weight, residual=None, eps=1e-5, dropout_p=0.0, rng_state=None,
                             residual_in_fp32=False):
    """PyTorch statement of :func:`dropout_add_rms_norm_fn` (fp32, or fp64 if x is fp64)."""
    wide = torch.float64 if x.dtype == torch.float64 else torch.float32
    dtype = residual.dtype if residual is not None else torch.float32 if residual_in_fp32 else x.dtype
    r = x.to(wide)
    if dropout_p:
        keep = dropout_add_rms_norm_mask_ref(x[..., 0].numel(), x.shape[-1], dropout_p, rng_state).view(x.shape)
        r = torch.where(keep, r * (1.0 / (1.0 - dropout_p)), torch.zeros((), dtype=wide, device=x.device))
    if residual is not None:
        r = r + residual.to(wide)
    stored = r.to(dtype)
    n = stored.to(wide) * torch.rsqrt((stored.to(wide) ** 2).mean(-1, keepdim=True) + eps)
    return (n * weight.to(wide)).to(x.dtype), stored
