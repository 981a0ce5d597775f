"""Selective recurrence: the state-space scan that follows the causal convolution.

    s_t = softplus(delta_t + delta_bias)
    h_t[d, n] = exp(s_t[d] A[d, n]) h_{t-1}[d, n] + s_t[d] x_t[d] B_t[n]
    out_t[d] = (sum_n C_t[n] h_t[d, n] + D[d] x_t[d]) silu(z_t[d])

``selective_recurrence_fn`` runs whole or packed sequences and has a backward pass;
``selective_recurrence_update`` runs a few tokens against a pool of states.  Both take the
(batch, dim, seqlen) tensors of :func:`causal_conv1d_fn` in its two layouts, compute and carry
h in fp32, and round once, on the stores.  States are fp32.
"""

from __future__ import annotations

import torch
import torch.nn.functional as F
from causal_conv1d._abi import block as _block


def _count(num_sequences):
    return -1 if num_sequences is None else num_sequences


def selective_recurrence_fwd_function(x, delta, A, B, C, D, z, delta_bias, delta_softplus, seq_idx, initial_states,
                                      return_final_states, num_sequences, save_checkpoints):
    """One forward pass.  Returns (out, final_states or None, checkpoints or None)."""
    return _block.selective_fwd(x, delta, A, B, C, D, z, delta_bias, delta_softplus, seq_idx, initial_states,
                                return_final_states, _count(num_sequences), save_checkpoints)


def selective_recurrence_bwd_function(x, delta, A, B, C, D, z, delta_bias, delta_softplus, seq_idx, initial_states,
                                      checkpoints, dout, dfinal_states, return_dbias, return_dinitial_states):
    """One backward pass.  Returns (dx, ddelta, dA, dB, dC, dD, dz, dbias, dinitial_states):
    dD and dz are None without D and z, each gradient has its input's dtype (fp32 where the input,
    delta_bias or initial_states, is absent)."""
    return _block.selective_bwd(x, delta, A, B, C, D, z, delta_bias, delta_softplus, seq_idx, initial_states, checkpoints,
                                dout, dfinal_states, return_dbias, return_dinitial_states)


def selective_recurrence_fn(x, delta, A, B, C, D=None, z=None, delta_bias=None, delta_softplus=True, seq_idx=None,
                            initial_states=None, return_final_states=False, num_sequences=None):
    """Selective recurrence over whole or packed sequences.

    x, delta, z: (batch, dim, seqlen) in one dtype (fp32, fp16, bf16), channel-last or
    contiguous; z optional.  A: (dim, dstate), dstate up to 256; D, delta_bias: (dim,),
    optional; these three in any float dtype.  B, C: (batch, dstate, seqlen), or
    (batch, groups, dstate, seqlen) where channel d uses group d // (dim // groups), in x's
    dtype and with any strides.  Without delta_softplus the step sizes are delta + delta_bias.
    initial_states: (batch, dim, dstate) fp32.  Returns out like x, or (out, final_states) with
    return_final_states, final_states (batch, dim, dstate) fp32.

    seq_idx, num_sequences and the states of packed sequences are those of
    :func:`gated_recurrence_fn`: a run of equal ids >= 0 in seq_idx (batch, seqlen) int32 is one
    sequence, its id the row of initial_states and final_states; a negative id is padding, whose
    out is 0 and where nothing is used; a sequence without positions keeps its initial state.

    Memory of training, for each position and channel, beside the inputs: dstate / 8 bytes (dstate / 4
    up to 8 states, dstate / 2 up to 4) are kept until the backward pass, which takes about 4 bytes of
    scratch at 16 states, 16 at 32 and dstate bytes at 64 and more, of as many batch rows as 2 GB hold,
    but of one row at least.

    Gradients flow back to x, delta, A, B, C, D, z, delta_bias and initial_states; they are
    summed in a fixed order.  There is no second derivative and no forward-mode one: both raise.
    """
    out, final = _block.selective(x, delta, A, B, C, D, z, delta_bias, delta_softplus, seq_idx, initial_states,
                                  return_final_states, _count(num_sequences))
    return (out, final) if return_final_states else out


def selective_recurrence_update(x, state, delta, A, B, C, D=None, z=None, delta_bias=None, delta_softplus=True,
                                state_indices=None):
    """One decode step (or a few tokens) of the recurrence; ``state`` is updated in place.

    x, delta, z: (batch, dim) or (batch, dim, seqlen).  B, C: (batch, dstate) or
    (batch, dstate, seqlen) to match, or with groups before dstate.  state: (batch, dim, dstate)
    fp32, or with state_indices (batch,) a pool (nstates, dim, dstate) of which batch row b uses
    row state_indices[b]; an index outside the pool is padding (zero output, no state touched),
    and no row may be named twice.  The indices are int32; other signed integers and uint8 are
    converted.  No two elements of state may lie at one place, as an expanded tensor's do.  The
    rest is as in :func:`selective_recurrence_fn`.  Returns out with x's shape.

    It has no derivative: a backward pass that reaches out raises, a state that requires grad
    is refused outside torch.no_grad(), and the state never carries a graph.
    """
    return _block.selective_update(x, state, delta, A, B, C, D, z, delta_bias, delta_softplus, state_indices)


def selective_recurrence_ref(x, delta, A, B, C, D=None, z=None, delta_bias=None, delta_softplus=True, seq_idx=None,
                             initial_states=None, return_final_states=False, num_sequences=None):
    """PyTorch statement of :func:`selective_recurrence_fn` (step by step, in fp64 if x is fp64
    and in fp32 otherwise, differentiable)."""
    wide = torch.float64 if x.dtype == torch.float64 else torch.float32
    batch, dim, seqlen = x.shape
    dstate = A.shape[1]
    B, C = (t.to(wide).unsqueeze(1) if t.dim() == 3 else t.to(wide) for t in (B, C))
    B, C = (t.repeat_interleave(dim // t.shape[1], 1) for t in (B, C))  # (batch, dim, dstate, seqlen)
    s = delta.to(wide)
    if delta_bias is not None:
        s = s + delta_bias.to(wide)[:, None]
    if delta_softplus:
        s = F.softplus(s, threshold=1e9)
    n = batch if seq_idx is None else (initial_states.shape[0] if initial_states is not None else num_sequences or 0)
    zero = torch.zeros(dim, dstate, device=x.device, dtype=wide)
    start = [initial_states[i].to(wide) if initial_states is not None else zero for i in range(n)]
    final = list(start)
    rows = []
    for b in range(batch):
        ids = [b] * seqlen if seq_idx is None else seq_idx[b].tolist()
        h, outs = zero, []
        for t in range(seqlen):
            k = ids[t]
            if k < 0:
                outs.append(zero[:, 0])
                continue
            if t == 0 or ids[t - 1] != k:
                h = start[k] if k < n else zero
            st, xt = s[b, :, t, None], x[b, :, t].to(wide)
            h = torch.exp(st * A.to(wide)) * h + st * xt[:, None] * B[b, :, :, t]
            if (t == seqlen - 1 or ids[t + 1] != k) and k < n:
                final[k] = h
            y = (h * C[b, :, :, t]).sum(-1)
            if D is not None:
                y = y + D.to(wide) * xt
            if z is not None:
                zt = z[b, :, t].to(wide)
                y = y * (zt * torch.sigmoid(zt))
            outs.append(y)
        rows.append(torch.stack(outs, -1) if outs else x[b].to(wide))
    out = (torch.stack(rows) if rows else x).to(x.dtype)
    if not return_final_states:
        return out
    return out, (torch.stack(final) if final else torch.zeros(0, dim, dstate, device=x.device, dtype=wide))
