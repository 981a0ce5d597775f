"""State indices of gated_recurrence_update of other types than int32."""

import pytest
import torch

from causal_conv1d import gated_recurrence_update

pytestmark = pytest.mark.gpu


def test_indices_past_32_bits_are_outside_the_pool():
    D = 40
    g = torch.Generator(device="cuda").manual_seed(0)
    state = torch.randn(6, D, generator=g, device="cuda")
    far = [1 << 32, (1 << 32) + 5, -(1 << 32) + 1, torch.iinfo(torch.int64).min, torch.iinfo(torch.int64).max, 1 << 31, -1, 6]
    index = torch.tensor([3, *far, 0], device="cuda")
    x, gate = (torch.randn(len(index), D, generator=g, device="cuda") for _ in range(2))
    before = state.clone()
    out = gated_recurrence_update(x, state, gate, state_indices=index)
    assert not out[1:-1].any() and out[0].any() and out[-1].any()
    assert torch.equal(state[[1, 2, 4, 5]], before[[1, 2, 4, 5]])
    assert not torch.equal(state[3], before[3]) and not torch.equal(state[0], before[0])


@pytest.mark.parametrize("dtype", [torch.int8, torch.uint8, torch.int16, torch.int32, torch.int64])
def test_integer_types(dtype):
    g = torch.Generator(device="cuda").manual_seed(1)
    x, state = torch.randn(3, 8, generator=g, device="cuda"), torch.randn(5, 8, generator=g, device="cuda")
    want = state.clone()
    index = torch.tensor([4, 1, 2], device="cuda")
    expected = gated_recurrence_update(x, want, x, state_indices=index.to(torch.int32))
    assert torch.equal(gated_recurrence_update(x, state, x, state_indices=index.to(dtype)), expected)
    assert torch.equal(state, want)
