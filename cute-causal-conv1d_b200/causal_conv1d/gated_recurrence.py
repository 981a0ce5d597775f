"""Gated linear recurrence: what follows the causal convolution in a recurrent block.

    a_t = sigmoid(gate_t + gate_bias)
    h_t = a_t h_{t-1} + (1 - a_t) x_t
    out_t = h_t silu(z_t)                      (out = h without z)

``gated_recurrence_fn`` runs whole or packed sequences and has a backward pass;
``gated_recurrence_update`` runs a few tokens against a pool of states.  Both take the
(batch, dim, seqlen) tensors of :func:`causal_conv1d_fn` in its two layouts, compute and
carry h in fp32, and round once, on the stores.  States are fp32.
"""

from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from causal_conv1d import _abi
from causal_conv1d.cpp_functions import _like_layout


def _laid_out(x, *others):
    """x with a unit stride along dim or seqlen, and the others in x's layout."""
    s = x.stride()
    if s[1] != 1 and s[2] != 1:
        x = x.contiguous()
        s = x.stride()
    laid = [x]
    for t in others:
        if t is not None and t.stride() != s and t.dim() == 3:
            t = _like_layout(t, x)
        laid.append(t)
    return laid


def gated_recurrence_fwd_function(x, gate, z, gate_bias, seq_idx, initial_states, return_final_states,
                                  num_sequences, save_checkpoints):
    """One forward pass.  Returns (out, final_states or None, checkpoints or None)."""
    shape = x.shape
    if len(shape) != 3:
        raise ValueError(f"x must have 3 dimensions, got shape {tuple(shape)}")
    x, gate, z = _laid_out(x, gate, z)
    batch, dim, seqlen = shape
    final = None
    if return_final_states:
        if seq_idx is None:
            n = batch
        elif initial_states is not None:
            n = initial_states.shape[0]
        elif num_sequences is not None:
            n = num_sequences
        else:
            raise ValueError("num_sequences is needed to return the final states of packed sequences "
                             "that have no initial states")
        if seq_idx is None and seqlen > 0:
            final = torch.empty(n, dim, device=x.device, dtype=torch.float32)
        elif initial_states is not None:  # a sequence without positions keeps its state
            final = initial_states.detach().clone(memory_format=torch.contiguous_format)
        else:
            final = torch.zeros(n, dim, device=x.device, dtype=torch.float32)
    checkpoints = None
    if save_checkpoints:
        chunks = -(-seqlen // _abi.RECURRENCE_CHUNK)
        checkpoints = torch.empty(batch, chunks, dim, device=x.device, dtype=torch.float32)
    out = torch.empty_like(x)
    _abi.recurrence_fwd(x, gate, z, gate_bias, seq_idx, initial_states, final, checkpoints, out)
    return out, final, checkpoints


def gated_recurrence_bwd_function(x, gate, z, gate_bias, seq_idx, initial_states, checkpoints, dout, dfinal_states,
                                  return_dbias, return_dinitial_states):
    """One backward pass.  Returns (dx, dgate, dz, dbias, dinitial_states): dx, dgate and dz
    in x's dtype (dz None without z), dbias in gate_bias's dtype, dinitial_states fp32."""
    x, gate, z, dout = _laid_out(x, gate, z, dout)
    dx, dgate = torch.empty_like(x), torch.empty_like(x)
    dz = torch.empty_like(x) if z is not None else None
    dbias = dinitial = None
    if return_dbias:
        dbias = torch.empty(x.shape[1], device=x.device, dtype=torch.float32)
    if return_dinitial_states:
        if seq_idx is None and x.shape[2] > 0:
            dinitial = torch.empty(initial_states.shape, device=x.device, dtype=torch.float32)
        elif dfinal_states is not None:  # a sequence without positions hands its gradient through
            dinitial = dfinal_states.clone(memory_format=torch.contiguous_format)
        else:
            dinitial = torch.zeros(initial_states.shape, device=x.device, dtype=torch.float32)
    _abi.recurrence_bwd(x, gate, z, gate_bias, seq_idx, initial_states, checkpoints, dout, dfinal_states, dx, dgate,
                        dz, dinitial, dbias)
    if dbias is not None and gate_bias.dtype != torch.float32:
        dbias = dbias.to(gate_bias.dtype)
    return dx, dgate, dz, dbias, dinitial


class GatedRecurrenceFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gate, z, gate_bias, seq_idx, initial_states, return_final_states, num_sequences):
        ctx.set_materialize_grads(False)
        out, final, checkpoints = gated_recurrence_fwd_function(
            x, gate, z, gate_bias, seq_idx, initial_states, return_final_states, num_sequences, True)
        ctx.return_final_states = return_final_states
        ctx.save_for_backward(x, gate, z, gate_bias, seq_idx, initial_states, checkpoints)
        return (out, final) if return_final_states else out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout, dfinal_states=None):
        x, gate, z, gate_bias, seq_idx, initial_states, checkpoints = ctx.saved_tensors
        if dout is None and dfinal_states is None:
            return (None,) * 8
        if dout is None:
            dout = torch.zeros_like(x)
        need = ctx.needs_input_grad
        dx, dgate, dz, dbias, dinitial = gated_recurrence_bwd_function(
            x, gate, z, gate_bias, seq_idx, initial_states, checkpoints, dout, dfinal_states,
            gate_bias is not None and need[3], initial_states is not None and need[5])
        return dx, dgate, dz, dbias, None, dinitial, None, None


def gated_recurrence_fn(x, gate, z=None, gate_bias=None, seq_idx=None, initial_states=None,
                        return_final_states=False, num_sequences=None):
    """Gated linear recurrence over whole or packed sequences.

    x, gate, z: (batch, dim, seqlen) in one dtype (fp32, fp16, bf16), channel-last or
    contiguous; z optional.  gate_bias: (dim,), any float dtype.  initial_states:
    (batch, dim) fp32.  Returns out like x, or (out, final_states) with
    return_final_states, final_states (batch, dim) fp32.

    seq_idx: (batch, seqlen) int32 packs sequences: a run of equal ids >= 0 is one sequence,
    and its id is the row of initial_states and final_states, then (num_sequences, dim),
    that belongs to it (so an id must not be used by two runs if states are given or
    returned); num_sequences is needed only to return final states without initial ones.
    A negative id is padding: its out is 0 and nothing there is used.  A sequence without
    positions keeps its initial state.
    """
    if torch.is_grad_enabled() and any(
            t is not None and t.requires_grad for t in (x, gate, z, gate_bias, initial_states)):
        return GatedRecurrenceFn.apply(x, gate, z, gate_bias, seq_idx, initial_states, return_final_states,
                                       num_sequences)
    out, final, _ = gated_recurrence_fwd_function(x, gate, z, gate_bias, seq_idx, initial_states,
                                                  return_final_states, num_sequences, False)
    return (out, final) if return_final_states else out


def gated_recurrence_update(x, state, gate, z=None, gate_bias=None, state_indices=None):
    """One decode step (or a few tokens) of the recurrence; ``state`` is updated in place.

    x, gate, z: (batch, dim) or (batch, dim, seqlen).  state: (batch, dim) fp32, or with
    state_indices (batch,) int32 a pool (nstates, dim) of which batch row b uses row
    state_indices[b]; an index outside the pool is padding (zero output, no state
    touched), and no row may be named twice.  Returns out with x's shape.
    """
    if state_indices is not None and state_indices.dtype is not torch.int32:
        state_indices = state_indices.to(torch.int32)
    out = torch.empty_like(x)
    _abi.recurrence_update(x, gate, z, gate_bias, state, state_indices, out)
    return out


def gated_recurrence_ref(x, gate, z=None, gate_bias=None, seq_idx=None, initial_states=None,
                         return_final_states=False, num_sequences=None):
    """PyTorch statement of :func:`gated_recurrence_fn` (step by step, in fp64 if x is fp64
    and in fp32 otherwise, differentiable)."""
    wide = torch.float64 if x.dtype == torch.float64 else torch.float32
    batch, dim, seqlen = x.shape
    u = gate.to(wide)
    if gate_bias is not None:
        u = u + gate_bias.to(wide)[:, None]
    a, c = torch.sigmoid(u), torch.sigmoid(-u)
    n = batch if seq_idx is None else (initial_states.shape[0] if initial_states is not None else num_sequences or 0)
    zero = torch.zeros(dim, device=x.device, dtype=wide)
    start = [initial_states[i].to(wide) if initial_states is not None else zero for i in range(n)]
    final = list(start)
    rows = []
    for b in range(batch):
        ids = [b] * seqlen if seq_idx is None else seq_idx[b].tolist()
        h, outs = zero, []
        for t in range(seqlen):
            k = ids[t]
            if k < 0:
                outs.append(zero)
                continue
            if t == 0 or ids[t - 1] != k:
                h = start[k] if k < n else zero
            h = a[b, :, t] * h + c[b, :, t] * x[b, :, t].to(wide)
            if (t == seqlen - 1 or ids[t + 1] != k) and k < n:
                final[k] = h
            o = h
            if z is not None:
                zt = z[b, :, t].to(wide)
                o = h * (zt * torch.sigmoid(zt))
            outs.append(o)
        rows.append(torch.stack(outs, -1) if outs else x[b].to(wide))
    out = (torch.stack(rows) if rows else x).to(x.dtype)
    if not return_final_states:
        return out
    return out, (torch.stack(final) if final else torch.zeros(0, dim, device=x.device, dtype=wide))
