"""PyTorch operator registrations:
``torch.ops.causal_conv1d.{fwd,bwd,update,varlen_states,fwd_varlen_states}``.

The same launches as :mod:`causal_conv1d.cpp_functions`, registered as custom operators
with their mutated arguments declared (``final_states_out`` of ``fwd``, ``conv_state`` of
``update``) and shape-only fake implementations.  ``torch.compile``, FakeTensor tracing
and ``torch.library.opcheck`` can therefore see through the kernels without running
them.

* ``fwd(x, weight, bias, seq_idx, initial_states, final_states_out, silu) -> out``
* ``bwd(x, weight, bias, dout, seq_idx, initial_states, dfinal_states,
  return_dinitial_states, silu) -> (dx, dweight, dbias, dinitial_states)``.  A custom
  operator cannot return None, so ``dbias`` and ``dinitial_states`` are empty tensors
  when there is no bias or no initial-state gradient.
* ``update(x, conv_state, weight, bias, silu, cache_seqlens, conv_state_indices) -> out``
* ``varlen_states(x, cu_seqlens, state_len) -> states``
* ``fwd_varlen_states(x, weight, bias, seq_idx, cu_seqlens, state_len, silu) -> (out, states)``
* ``gated_recurrence_fwd(x, gate, z, gate_bias, seq_idx, initial_states, return_final_states,
  num_sequences, save_checkpoints) -> (out, final_states, checkpoints)``, empty where not asked for
* ``gated_recurrence_bwd(x, gate, z, gate_bias, seq_idx, initial_states, checkpoints, dout,
  dfinal_states, return_dbias, return_dinitial_states) -> (dx, dgate, dz, dbias, dinitial_states)``
* ``gated_recurrence_update(x, state, gate, z, gate_bias, state_indices) -> out``
* ``dropout_add_rms_norm_fwd(x, weight, residual, eps, dropout_p, rng_state, residual_in_fp32)
  -> (out, residual_out)``
* ``dropout_add_rms_norm_bwd(x_dtype, residual_out, weight, dout, dresidual_out, eps, dropout_p,
  rng_state) -> (dx, dresidual, dweight)``

The reference compiles its kernels with the CuTe DSL and registers no torch operators;
these registrations are this package's equivalent of the C++ extension's op table.
"""

from __future__ import annotations

import torch
from torch import Tensor

from causal_conv1d import _abi
from causal_conv1d import add_norm as _an
from causal_conv1d import cpp_functions as _cf
from causal_conv1d import gated_recurrence as _gr
from causal_conv1d.causal_conv1d_varlen import causal_conv1d_fn_varlen_states as _fwd_varlen_states
from causal_conv1d.causal_conv1d_varlen import causal_conv1d_varlen_states as _varlen_states

_EMPTY = (0,)


@torch.library.custom_op("causal_conv1d::fwd", mutates_args=("final_states_out",))
def fwd(x: Tensor, weight: Tensor, bias: Tensor | None, seq_idx: Tensor | None,
        initial_states: Tensor | None, final_states_out: Tensor | None, silu: bool) -> Tensor:
    return _cf.causal_conv1d_fwd_function(x, weight, bias, seq_idx, initial_states, final_states_out, silu)


@fwd.register_fake
def _(x, weight, bias, seq_idx, initial_states, final_states_out, silu):
    return torch.empty_like(x)


@torch.library.custom_op("causal_conv1d::bwd", mutates_args=())
def bwd(x: Tensor, weight: Tensor, bias: Tensor | None, dout: Tensor, seq_idx: Tensor | None,
        initial_states: Tensor | None, dfinal_states: Tensor | None, return_dinitial_states: bool,
        silu: bool) -> tuple[Tensor, Tensor, Tensor, Tensor]:
    dx, dw, db, di = _cf.causal_conv1d_bwd_function(x, weight, bias, dout, seq_idx, initial_states,
                                                    dfinal_states, None, return_dinitial_states, silu)
    if db is None:
        db = x.new_empty(_EMPTY, dtype=weight.dtype)
    if di is None:
        di = x.new_empty(_EMPTY)
    return dx, dw, db, di


@bwd.register_fake
def _(x, weight, bias, dout, seq_idx, initial_states, dfinal_states, return_dinitial_states, silu):
    dx = torch.empty_like(x)
    dw = torch.empty_like(weight, memory_format=torch.contiguous_format)
    db = torch.empty_like(bias) if bias is not None else x.new_empty(_EMPTY, dtype=weight.dtype)
    if initial_states is not None and return_dinitial_states:
        di = torch.empty_like(initial_states)
    else:
        di = x.new_empty(_EMPTY)
    return dx, dw, db, di


@torch.library.custom_op("causal_conv1d::update", mutates_args=("conv_state",))
def update(x: Tensor, conv_state: Tensor, weight: Tensor, bias: Tensor | None, silu: bool,
           cache_seqlens: Tensor | None, conv_state_indices: Tensor | None) -> Tensor:
    return _cf.causal_conv1d_update_function(x, conv_state, weight, bias, silu, cache_seqlens,
                                             conv_state_indices)


@update.register_fake
def _(x, conv_state, weight, bias, silu, cache_seqlens, conv_state_indices):
    return torch.empty_like(x)


@torch.library.custom_op("causal_conv1d::varlen_states", mutates_args=())
def varlen_states(x: Tensor, cu_seqlens: Tensor, state_len: int) -> Tensor:
    return _varlen_states(x, cu_seqlens, state_len)


@varlen_states.register_fake
def _(x, cu_seqlens, state_len):
    batch = cu_seqlens.shape[0] - 1
    return x.new_empty(batch, state_len, x.shape[1]).transpose(1, 2)


@torch.library.custom_op("causal_conv1d::fwd_varlen_states", mutates_args=())
def fwd_varlen_states(x: Tensor, weight: Tensor, bias: Tensor | None, seq_idx: Tensor | None,
                      cu_seqlens: Tensor, state_len: int, silu: bool) -> tuple[Tensor, Tensor]:
    return _fwd_varlen_states(x, weight, cu_seqlens, state_len, bias, seq_idx, "silu" if silu else None)


@fwd_varlen_states.register_fake
def _(x, weight, bias, seq_idx, cu_seqlens, state_len, silu):
    nseq = cu_seqlens.shape[0] - 1
    out = torch.empty_like(x) if (x.stride(2) == 1 or x.stride(1) == 1) else torch.empty_like(x.contiguous())
    return out, x.new_empty(nseq, state_len, x.shape[1]).transpose(1, 2)


# -------------------------------------------------------- recurrent-block operators
def _laid_out_like(x):
    """An empty tensor with the layout that the recurrence gives its results."""
    return torch.empty_like(x) if (x.stride(2) == 1 or x.stride(1) == 1) else torch.empty_like(x.contiguous())


@torch.library.custom_op("causal_conv1d::gated_recurrence_fwd", mutates_args=())
def gated_recurrence_fwd(x: Tensor, gate: Tensor, z: Tensor | None, gate_bias: Tensor | None, seq_idx: Tensor | None,
                         initial_states: Tensor | None, return_final_states: bool, num_sequences: int,
                         save_checkpoints: bool) -> tuple[Tensor, Tensor, Tensor]:
    out, final, checkpoints = _gr.gated_recurrence_fwd_function(
        x, gate, z, gate_bias, seq_idx, initial_states, return_final_states, num_sequences, save_checkpoints)
    empty = x.new_empty(_EMPTY, dtype=torch.float32)
    return out, empty if final is None else final, empty.clone() if checkpoints is None else checkpoints


@gated_recurrence_fwd.register_fake
def _(x, gate, z, gate_bias, seq_idx, initial_states, return_final_states, num_sequences, save_checkpoints):
    batch, dim, seqlen = x.shape
    n = batch if seq_idx is None else initial_states.shape[0] if initial_states is not None else num_sequences
    final = x.new_empty((n, dim) if return_final_states else _EMPTY, dtype=torch.float32)
    chunks = -(-seqlen // _abi.RECURRENCE_CHUNK)
    return _laid_out_like(x), final, x.new_empty((batch, chunks, dim) if save_checkpoints else _EMPTY, dtype=torch.float32)


@torch.library.custom_op("causal_conv1d::gated_recurrence_bwd", mutates_args=())
def gated_recurrence_bwd(x: Tensor, gate: Tensor, z: Tensor | None, gate_bias: Tensor | None, seq_idx: Tensor | None,
                         initial_states: Tensor | None, checkpoints: Tensor, dout: Tensor,
                         dfinal_states: Tensor | None, return_dbias: bool,
                         return_dinitial_states: bool) -> tuple[Tensor, Tensor, Tensor, Tensor, Tensor]:
    dx, dgate, dz, dbias, dinitial = _gr.gated_recurrence_bwd_function(
        x, gate, z, gate_bias, seq_idx, initial_states, checkpoints, dout, dfinal_states, return_dbias,
        return_dinitial_states)
    if dz is None:
        dz = x.new_empty(_EMPTY)
    if dbias is None:
        dbias = x.new_empty(_EMPTY, dtype=torch.float32)
    if dinitial is None:
        dinitial = x.new_empty(_EMPTY, dtype=torch.float32)
    return dx, dgate, dz, dbias, dinitial


@gated_recurrence_bwd.register_fake
def _(x, gate, z, gate_bias, seq_idx, initial_states, checkpoints, dout, dfinal_states, return_dbias,
      return_dinitial_states):
    dz = _laid_out_like(x) if z is not None else x.new_empty(_EMPTY)
    dbias = gate_bias.new_empty(x.shape[1]) if return_dbias else x.new_empty(_EMPTY, dtype=torch.float32)
    dinitial = x.new_empty(initial_states.shape if return_dinitial_states else _EMPTY, dtype=torch.float32)
    return _laid_out_like(x), _laid_out_like(x), dz, dbias, dinitial


@torch.library.custom_op("causal_conv1d::gated_recurrence_update", mutates_args=("state",))
def gated_recurrence_update(x: Tensor, state: Tensor, gate: Tensor, z: Tensor | None, gate_bias: Tensor | None,
                            state_indices: Tensor | None) -> Tensor:
    return _gr.gated_recurrence_update(x, state, gate, z, gate_bias, state_indices)


@gated_recurrence_update.register_fake
def _(x, state, gate, z, gate_bias, state_indices):
    return torch.empty_like(x)


@torch.library.custom_op("causal_conv1d::dropout_add_rms_norm_fwd", mutates_args=())
def dropout_add_rms_norm_fwd(x: Tensor, weight: Tensor, residual: Tensor | None, eps: float, dropout_p: float,
                             rng_state: Tensor | None, residual_in_fp32: bool) -> tuple[Tensor, Tensor]:
    return _an.dropout_add_rms_norm_fwd_function(x, weight, residual, eps, dropout_p, rng_state, residual_in_fp32)


@dropout_add_rms_norm_fwd.register_fake
def _(x, weight, residual, eps, dropout_p, rng_state, residual_in_fp32):
    dtype = residual.dtype if residual is not None else torch.float32 if residual_in_fp32 else x.dtype
    return x.new_empty(x.shape), x.new_empty(x.shape, dtype=dtype)


@torch.library.custom_op("causal_conv1d::dropout_add_rms_norm_bwd", mutates_args=())
def dropout_add_rms_norm_bwd(x_dtype: torch.dtype, residual_out: Tensor, weight: Tensor, dout: Tensor | None,
                             dresidual_out: Tensor | None, eps: float, dropout_p: float,
                             rng_state: Tensor | None) -> tuple[Tensor, Tensor, Tensor]:
    dx, dresidual, dweight = _an.dropout_add_rms_norm_bwd_function(
        x_dtype, residual_out, weight, dout, dresidual_out, eps, dropout_p, rng_state, True, True, True)
    return dx, dresidual.clone() if dresidual is dx else dresidual, dweight  # an operator's results may not alias


@dropout_add_rms_norm_bwd.register_fake
def _(x_dtype, residual_out, weight, dout, dresidual_out, eps, dropout_p, rng_state):
    return (residual_out.new_empty(residual_out.shape, dtype=x_dtype), residual_out.new_empty(residual_out.shape),
            weight.new_empty(weight.shape))
