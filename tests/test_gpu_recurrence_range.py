"""gated_recurrence_fn and gated_recurrence_update at the ends of their range: gates and biases
of any size, slow channels; compared place by place or within a channel, so that a large value
beside a small one hides nothing.

Bounds.  As in block_ref: the stored type's unit roundoff, and 2^-18 relative for the fp32
computation of one place.  A state that stays below the inputs for L positions is a sum of L
terms, each of which a product of up to L factors has scaled: every factor is off by at most
2^-24 (half a unit below one, and as much for the step's own rounding), so 2 L 2^-24 of the
state is added to it."""

import numpy as np
import pytest
import torch

import block_ref as R
from causal_conv1d import gated_recurrence_fn, gated_recurrence_update
from helpers import with_layout
from test_gpu_recurrence import DTYPES, LAYOUTS, _gen, _inputs, _run_and_check

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


# ------------------------------------------------------------------ slow channels
@pytest.mark.parametrize("layout", ["channel_last", "contiguous", "cl_slice"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("L", [257, 1500])
def test_slow_channels_from_zero(L, dtype, layout):
    """Channels that gain e^-8 to e^-20 of x with each token: every one of them, its gradients
    and the same tokens taken by the update, to its own size."""
    B, D = 1, 64
    g = _gen(L)

    def rnd(scale, shift):
        return with_layout((torch.randn(B, D, L, generator=g, device="cuda") * scale + shift).to(dtype), layout)

    x, gate, dout = rnd(0.25, 1.0), rnd(0.25, 0.0), rnd(0.25, 1.0)
    bias = torch.linspace(8.0, 20.0, D, device="cuda")
    init, dfinal = torch.zeros(B, D, device="cuda"), torch.ones(B, D, device="cuda")
    leaves = [v.detach().requires_grad_() for v in (x, gate, bias, init)]
    out, final = gated_recurrence_fn(leaves[0], leaves[1], None, leaves[2], initial_states=leaves[3], return_final_states=True)
    dx, dgate, dbias, dinit = torch.autograd.grad([out, final], leaves, [dout, dfinal])
    w = [R.wide(v) for v in (x, gate, bias, init, dout, dfinal)]
    eo, ef, _, _ = R.recurrence(w[0], w[1], None, w[2], None, w[3])
    e = R.recurrence_grads(w[0], w[1], None, w[2], None, w[3], w[4], w[5])
    steps = R.COMPUTED + 2.0 * L * 2.0 ** -24  # relative error of a channel's states

    def close(got, want, axes, what):
        """Each channel to `steps` of its own largest value, and the stored type's rounding."""
        own = np.abs(want).max(axes, keepdims=True)
        over = np.abs(R.wide(got) - want) - R.UNIT[got.dtype] * np.abs(want) - steps * own - R.TINY[got.dtype]
        assert over.max() <= 0.0, f"{what}: {(over / own).max()} of the channel over the bound"

    close(out, eo, (0, 2), "out")
    close(final, ef, 0, "final_states")
    close(dx, e["dx"], (0, 2), "dx")
    close(dgate, e["dgate"], (0, 2), "dgate")
    close(dbias[None], e["dbias"][None], 0, "dbias")
    close(dinit, e["dinit"], 0, "dinitial_states")
    state = init.clone()
    stepped = gated_recurrence_update(x, state, gate, None, bias)
    close(stepped, eo, (0, 2), "update")
    close(state, ef, 0, "updated state")
