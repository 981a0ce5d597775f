"""selective_recurrence_fn and selective_recurrence_update where a call has many states, several tokens or nothing."""

import pytest
import torch

from causal_conv1d import selective_recurrence_fn, selective_recurrence_update
from test_gpu_selective import DTYPES

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


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("u", [-100.0, -80.0, -60.0, -20.0, -2.0, -1e-3, 0.0, 15.0, 40.0, 100.0])
def test_step_sizes_of_each_type(u, dtype):
    """A state that takes up one step is the step.  The exponential is within 2^-22 and the reciprocal within
    2^-23 of themselves, and five roundings follow: 2^-20 in all.  For 16-bit tensors the exponential keeps the
    rounding of its argument |u| log2(e), 2^-24, and of log2(e), 2^-26: (2^-24 + 2^-26) |u| more.  What is below
    2^-126 is zero."""
    D = 512
    delta = (u + torch.linspace(-0.5, 0.5, D, device="cuda") * max(1.0, abs(u) / 16)).view(1, D, 1).to(dtype)
    x, A = torch.ones(1, D, 1, device="cuda", dtype=dtype), torch.zeros(D, 1, device="cuda")
    bc = torch.ones(1, 1, 1, device="cuda", dtype=dtype)
    w = delta.double()[..., 0]
    want = torch.clamp(w, min=0) + torch.log1p(torch.exp(-w.abs()))
    rel = 2.0 ** -20 + (0.0 if dtype == torch.float32 else 2.0 ** -24 + 2.0 ** -26) * w.abs()
    _, final = selective_recurrence_fn(x, delta, A, bc, bc, return_final_states=True)
    state = torch.zeros(1, D, 1, device="cuda")
    selective_recurrence_update(x, state, delta, A, bc, bc)
    for got in (final, state):
        assert ((got[..., 0].double() - want).abs() <= rel * want + 2.0 ** -126).all()
