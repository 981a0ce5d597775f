"""The residual connection between two blocks: dropout, residual add and RMSNorm in one pass.

    residual_out = residual + keep x / (1 - dropout_p)
    out = residual_out / sqrt(mean(residual_out^2) + eps) * weight

The dropout mask ``keep`` is a function of a generator state and the place alone
(Philox4x32-10), recomputed by the backward and never stored.
"""

from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from causal_conv1d import _abi


def _rows(t, dim):
    """t as a (rows, dim) matrix with channel stride 1."""
    if t.dim() != 2:
        t = t.reshape(-1, dim)
    return t if t.stride(1) == 1 else t.contiguous()


def dropout_add_rms_norm_fwd_function(x, weight, residual, eps, dropout_p, rng_state, residual_in_fp32):
    """One forward pass.  Returns (out, residual_out), both with x's shape."""
    if x.dim() == 0 or weight.dim() != 1 or weight.shape[0] != x.shape[-1]:
        raise ValueError("x and weight must have shapes (..., dim) and (dim,)")
    if residual is not None and residual.shape != x.shape:
        raise ValueError(f"residual must have shape {tuple(x.shape)}, got {tuple(residual.shape)}")
    if residual is not None and residual_in_fp32 and residual.dtype != torch.float32:
        raise ValueError("residual must be float32 with residual_in_fp32")
    dim = x.shape[-1]
    dtype = residual.dtype if residual is not None else torch.float32 if residual_in_fp32 else x.dtype
    out = torch.empty_like(x, memory_format=torch.contiguous_format)
    residual_out = torch.empty_like(out, dtype=dtype)
    if dim == 0:
        return out, residual_out
    flat = (out, residual_out) if out.dim() == 2 else (out.view(-1, dim), residual_out.view(-1, dim))
    _abi.add_norm_fwd(_rows(x, dim), None if residual is None else _rows(residual, dim), weight, rng_state, *flat,
                      eps, dropout_p)
    return out, residual_out


def dropout_add_rms_norm_bwd_function(x_dtype, residual_out, weight, dout, dresidual_out, eps, dropout_p, rng_state,
                                      return_dx, return_dresidual, return_dweight):
    """One backward pass.  Returns (dx, dresidual, dweight), each None if not asked for.
    Without dropout dx and dresidual are equal, and one tensor if their dtypes are."""
    shape, dim = residual_out.shape, residual_out.shape[-1]
    shared = return_dx and return_dresidual and dropout_p == 0.0 and x_dtype == residual_out.dtype

    def new(wanted, dtype):
        return torch.empty(shape, device=residual_out.device, dtype=dtype) if wanted else None

    dx = new(return_dx, x_dtype)
    dresidual = new(return_dresidual and not shared, residual_out.dtype)
    dweight = torch.empty(dim, device=residual_out.device, dtype=torch.float32) if return_dweight else None

    def rows(t):
        return None if t is None else _rows(t, dim)

    if dim:
        _abi.add_norm_bwd(x_dtype, rows(residual_out), weight, rng_state, rows(dout), rows(dresidual_out), rows(dx),
                          rows(dresidual), dweight, eps, dropout_p)
    if shared:
        dresidual = dx
    if dweight is not None and weight.dtype != torch.float32:
        dweight = dweight.to(weight.dtype)
    return dx, dresidual, dweight


class DropoutAddRMSNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, residual, eps, dropout_p, rng_state, residual_in_fp32):
        ctx.set_materialize_grads(False)
        out, residual_out = dropout_add_rms_norm_fwd_function(x, weight, residual, eps, dropout_p, rng_state,
                                                              residual_in_fp32)
        ctx.eps, ctx.dropout_p, ctx.x_dtype = eps, dropout_p, x.dtype
        ctx.save_for_backward(residual_out, weight, rng_state)
        return out, residual_out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout, dresidual_out):
        if dout is None and dresidual_out is None:
            return (None,) * 7
        residual_out, weight, rng_state = ctx.saved_tensors
        need = ctx.needs_input_grad
        dx, dresidual, dweight = dropout_add_rms_norm_bwd_function(
            ctx.x_dtype, residual_out, weight, dout, dresidual_out, ctx.eps, ctx.dropout_p, rng_state,
            need[0], need[2], need[1])
        return dx, dweight, dresidual, None, None, None, None


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
    """
    if not 0.0 <= dropout_p < 1.0:
        raise ValueError("dropout_p must be in [0, 1)")
    if dropout_p == 0.0:
        rng_state = None
    elif rng_state is None:
        rng_state = torch.randint(0, 1 << 62, (2,), device=x.device, dtype=torch.int64)
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or
                                    (residual is not None and residual.requires_grad)):
        return DropoutAddRMSNormFn.apply(x, weight, residual, eps, dropout_p, rng_state, residual_in_fp32)
    return dropout_add_rms_norm_fwd_function(x, weight, residual, eps, dropout_p, rng_state, residual_in_fp32)


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
