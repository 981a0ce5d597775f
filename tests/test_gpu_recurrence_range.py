"""gated_recurrence_fn and gated_recurrence_update at the ends of their range."""

import numpy as np
import pytest
import torch

from test_gpu_recurrence import DTYPES, LAYOUTS, _inputs, _run_and_check

pytestmark = pytest.mark.gpu


# ------------------------------------------------------- channels without a memory
@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,D,L", [(2, 70, 1), (2, 70, 33), (1, 66, 64), (2, 64, 77), (1, 64, 3001)])
def test_dfinal_reaches_the_last_position_whatever_the_bias(B, D, L, dtype, layout):
    """With a bias that lets everything go at once dx of the last position is dfinal plus the
    output's part; the last chunk is seldom whole."""
    t = _inputs(D + L, B, D, L, dtype, layout, nstates=B)
    worst = torch.tensor([-6.5e4, -1e9, torch.finfo(torch.float32).min, float("-inf"), 0.0, 6.5e4, float("inf")], device="cuda")
    t["bias"] = worst[torch.arange(D, device="cuda") % 7].contiguous()
    with np.errstate(over="ignore"):
        _run_and_check(t)
