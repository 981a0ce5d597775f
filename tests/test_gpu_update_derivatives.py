"""gated_recurrence_update has no derivative and writes its state in place: what asks for one, or
reads a state that a graph has saved, raises."""

import pytest
import torch

from causal_conv1d import gated_recurrence_fn, gated_recurrence_update

pytestmark = pytest.mark.gpu


def _tensors(B=2, D=24, L=20):
    g = torch.Generator(device="cuda").manual_seed(0)
    x, gate, z = (torch.randn(B, L, D, generator=g, device="cuda").transpose(1, 2) for _ in range(3))
    return x, gate, z, torch.randn(D, generator=g, device="cuda"), torch.randn(B, D, generator=g, device="cuda")


@pytest.mark.parametrize("which", [0, 2, 3, 4])
def test_backward_through_the_update_raises(which):
    """It has no derivative: its result says so when one is asked for, and the values are the same."""
    x, gate, z, bias, state = _tensors()
    args = [x[..., 0], state, gate[..., 0], z[..., 0], bias]
    with torch.no_grad():
        want = gated_recurrence_update(*[a.clone() for a in args])
    args[which] = args[which].detach().requires_grad_()
    out = gated_recurrence_update(*args)
    assert torch.equal(out, want) and out.requires_grad
    with pytest.raises(RuntimeError, match="gated_recurrence_update has no derivative"):
        (out.sum() + args[which].sum()).backward()
    with torch.no_grad():
        assert not gated_recurrence_update(*args).requires_grad


def test_update_refuses_a_state_that_requires_grad():
    x, gate, z, bias, state = _tensors()
    leaf = state.clone().requires_grad_()
    for bad in (leaf, leaf * 1.0):
        with pytest.raises(RuntimeError, match="state"):
            gated_recurrence_update(x[..., 0], bad, gate[..., 0])
    with torch.no_grad():
        gated_recurrence_update(x[..., 0], leaf, gate[..., 0])
    assert not torch.equal(leaf, state)


def test_a_saved_state_that_the_update_overwrites_is_noticed():
    x, gate, z, bias, state = _tensors()
    leaf = x.detach().requires_grad_()
    out = gated_recurrence_fn(leaf, gate, z, bias, initial_states=state)
    version = state._version
    gated_recurrence_update(x[..., 0], state, gate[..., 0])
    assert state._version == version + 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()
    # a call that writes nothing counts nothing
    gated_recurrence_update(x[:0, :, 0], state[:0], gate[:0, :, 0])
    assert state._version == version + 1


def test_update_of_inference_tensors():
    x, gate, z, bias, state = _tensors()
    want = state.clone()
    gated_recurrence_update(x[..., 0], want, gate[..., 0])
    with torch.inference_mode():
        inside = state.clone()
        out = gated_recurrence_update(x[..., 0], inside, gate[..., 0])
        assert torch.equal(inside, want)
    with torch.no_grad():
        other = gated_recurrence_update(x[..., 0], inside, gate[..., 0])  # and outside
    assert out.shape == other.shape and not torch.equal(inside, want)
