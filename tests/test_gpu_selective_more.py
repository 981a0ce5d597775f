"""selective_recurrence_fn and selective_recurrence_update where a call has many states, several tokens or nothing."""

import pytest
import torch

from causal_conv1d import selective_recurrence_fn

pytestmark = pytest.mark.gpu


def test_no_channels():
    """Without channels B and C reach nothing: their gradients are zero."""
    for groups in (0, 2):
        x = torch.randn(2, 0, 5, device="cuda", requires_grad=True)
        shape = (2, groups, 4, 5) if groups else (2, 4, 5)
        B, C = (torch.randn(shape, device="cuda", requires_grad=True) for _ in range(2))
        A = -torch.ones(0, 4, device="cuda")
        for _ in range(3):
            dirty = [torch.full(shape, float("nan"), device="cuda") for _ in range(8)]  # what the allocator hands out next
            del dirty
            out = selective_recurrence_fn(x, x, A, B, C)
            for g in torch.autograd.grad(out, (B, C), torch.ones_like(out)):
                assert g.shape == shape and (g == 0).all()
