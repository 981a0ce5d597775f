"""Types of state indices that gated_recurrence_update refuses."""

import pytest
import torch

from causal_conv1d import gated_recurrence_update


@pytest.mark.parametrize("dtype", [torch.float32, torch.float64, torch.bool, torch.complex64])
def test_indices_that_are_no_integers_are_refused(dtype):
    x, state = torch.zeros(2, 8), torch.zeros(5, 8)
    with pytest.raises(TypeError, match="state_indices"):
        gated_recurrence_update(x, state, x, state_indices=torch.zeros(2).to(dtype))
    with pytest.raises(ValueError, match="CUDA"):  # the next check
        gated_recurrence_update(x, state, x, state_indices=torch.zeros(2, dtype=torch.int64))
