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
from causal_conv1d._abi import block as _block


def gated_recurrence_fwd_function(x, gate, z, gate_bias, seq_idx, initial_states, return_final_states,
                                  num_sequences, save_checkpoints):
    """One forward pass.  Returns (out, final_states or None, checkpoints or None)."""
    return _block.recurrence_fwd(x, gate, z, gate_bias, seq_idx, initial_states, return_final_states,
                                 -1 if num_sequences is None else num_sequences, save_checkpoints)


def gated_recurrence_bwd_function(x, gate, z, gate_bias, seq_idx, initial_states, checkpoints, dout, dfinal_states,
                                  return_dbias, return_dinitial_states):
    """One backward pass.  Returns (dx, dgate, dz, dbias, dinitial_states): dx, dgate and dz
    in x's dtype (dz None without z), dbias in gate_bias's dtype, dinitial_states fp32."""
    return _block.recurrence_bwd(x, gate, z, gate_bias, seq_idx, initial_states, checkpoints, dout, dfinal_states,
                                 return_dbias, return_dinitial_states)


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

    Gradients flow back to x, gate, z, gate_bias and initial_states.  There is no second
    derivative and no forward-mode one: both raise.
    """
    out, final = _block.recurrence(x, gate, z, gate_bias, seq_idx, initial_states, return_final_states,
                                   -1 if num_sequences is None else num_sequences)
    return (out, final) if return_final_states else out


def gated_recurrence_update(x, state, gate, z=None, gate_bias=None, state_indices=None):
    """One decode step (or a few tokens) of the recurrence; ``state`` is updated in place.

    x, gate, z: (batch, dim) or (batch, dim, seqlen).  state: (batch, dim) fp32, or with
    state_indices (batch,) a pool (nstates, dim) of which batch row b uses row
    state_indices[b]; an index outside the pool is padding (zero output, no state
    touched), and no row may be named twice.  The indices are int32; other signed integers
    and uint8 are converted.  Returns out with x's shape.

    It has no derivative: a backward pass that reaches out raises, a state that requires grad
    is refused outside torch.no_grad(), and the state never carries a graph.
    """
    return _block.recurrence_update(x, state, gate, z, gate_bias, state_indices)


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
