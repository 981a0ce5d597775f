"""Derivatives that the recurrent-block operators do not have are refused, before anything runs."""

import pytest
import torch
import torch.autograd.forward_ad as fwAD

from causal_conv1d import dropout_add_rms_norm_fn, gated_recurrence_fn, gated_recurrence_update


def _tensors(B=2, D=24, L=20):
    x, gate, z = (torch.zeros(B, L, D).transpose(1, 2) for _ in range(3))
    return [x, gate, z, torch.zeros(D), torch.zeros(B, D)]


@pytest.mark.parametrize("grad", [True, False])
@pytest.mark.parametrize("which", range(5))
def test_recurrence_refuses_forward_mode(which, grad):
    with fwAD.dual_level(), torch.set_grad_enabled(grad):
        args = _tensors()
        args[which] = fwAD.make_dual(args[which], torch.ones_like(args[which]))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            gated_recurrence_fn(*args[:4], initial_states=args[4])


@pytest.mark.parametrize("which", range(5))
def test_update_refuses_forward_mode(which):
    with fwAD.dual_level():
        x, gate, z, bias, state = _tensors()
        args = [x[..., 0], state, gate[..., 0], z[..., 0], bias]
        args[which] = fwAD.make_dual(args[which], torch.ones_like(args[which]))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            gated_recurrence_update(*args)


@pytest.mark.parametrize("which", range(3))
def test_add_norm_refuses_forward_mode(which):
    with fwAD.dual_level():
        args = [torch.zeros(5, 16), torch.zeros(16), torch.zeros(5, 16)]
        args[which] = fwAD.make_dual(args[which], torch.ones_like(args[which]))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            dropout_add_rms_norm_fn(*args)


def test_a_level_that_is_over_refuses_nothing():
    with fwAD.dual_level():
        x = fwAD.make_dual(torch.zeros(2, 4, 3), torch.ones(2, 4, 3))
    with pytest.raises(ValueError, match="CUDA"):  # the next check
        gated_recurrence_fn(x, x)
