"""gated_recurrence_fn and gated_recurrence_update at the ends of their range: gates and biases
of any size, slow channels, output gates of any size; compared place by place or within a channel, so that a large value
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


def _within(got, want, size, what):
    """got within its type's rounding of want, and 2^-18 of `size`, place by place."""
    g = R.wide(got)
    err = np.abs(g - want) - R.UNIT[got.dtype] * np.abs(want) - R.COMPUTED * size - 2.0 * R.TINY[got.dtype]
    err = np.where(np.isfinite(g) | ~np.isfinite(want), err, np.inf)
    assert (err <= 0.0).all(), f"{what}: {(~(err <= 0.0)).sum()} places, worst {np.nanmax(err)} over the bound"


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


# --------------------------------------------------------------- gates that let go
@pytest.mark.parametrize("layout", ["channel_last", "contiguous", "cl_slice"])
@pytest.mark.parametrize("dtype", DTYPES)
def test_a_reset_leaves_nothing_behind(dtype, layout):
    """One gate far below zero takes the state down by e^gate, to zero in the end, and with it
    the gradient that goes back through it; the states are up to 1e6."""
    B, L = 1, 40
    lowest = torch.finfo(dtype).min
    values = torch.tensor([-15.0, -20.0, -21.0, -25.0, -30.0, -50.0, -80.0, -200.0, -1e4, lowest, float("-inf")])
    D = 66
    at = torch.arange(D) % L  # the place of the reset: another one for each channel
    gate = torch.full((B, D, L), 30.0)
    gate[0, torch.arange(D), at] = values[torch.arange(D) % len(values)]
    gate = with_layout(gate.cuda().to(dtype), layout)
    x = with_layout(torch.zeros(B, D, L, device="cuda").to(dtype), layout)
    init = torch.full((B, D), 1e6, device="cuda")
    dfinal = torch.full((B, D), 1e6, device="cuda")
    dout = with_layout(torch.zeros(B, D, L, device="cuda").to(dtype), layout)
    leaf = init.detach().requires_grad_()
    out, final = gated_recurrence_fn(x, gate, initial_states=leaf, return_final_states=True)
    (dinit,) = torch.autograd.grad([out, final], [leaf], [dout, dfinal])
    w = [R.wide(v) for v in (x, gate, init, dfinal)]
    with np.errstate(over="ignore"):
        _, ef, _, _ = R.recurrence(w[0], w[1], None, None, None, w[2])
        e = R.recurrence_grads(w[0], w[1], None, None, None, w[2], np.zeros_like(w[0]), w[3])
    _within(final, ef, np.abs(ef), "final_states")
    _within(dinit, e["dinit"], np.abs(e["dinit"]), "dinitial_states")
    state = init.clone()
    gated_recurrence_update(x, state, gate)
    _within(state, ef, np.abs(ef), "updated state")


# ------------------------------------------------------------- output gates of any size
ORDINARY = [-1.5, 0.5, 2.0, 5.0]
CLOSED = [-10.0, -19.0, -22.0, -30.0, -60.0, -100.0, -1e3, -6e4]
OPEN = [10.0, 20.0, 40.0, 1e3, 1e4, 6e4]


def _gates(dtype):
    return torch.tensor([*ORDINARY, *CLOSED, torch.finfo(dtype).min, *OPEN])


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("L", [40, 300])
def test_output_gates_of_any_size(L, dtype, layout):
    """silu(z) and its derivative from the type's lowest value up, ordinary values beside."""
    B, D = 1, 70
    t = _inputs(L, B, D, L, dtype, layout, nstates=B)
    values = _gates(dtype).cuda()
    pick = torch.randint(0, len(values), (B, D, L), generator=_gen(2), device="cuda")
    t["z"].copy_(values[pick].to(dtype))
    t["x"].mul_(0.125)
    t["init"].mul_(0.125)
    t["dout"].mul_(2.0 ** -10)
    leaves = [t[k].detach().requires_grad_() for k in ("x", "gate", "z")]
    out = gated_recurrence_fn(*leaves, t["bias"], initial_states=t["init"])
    dz = torch.autograd.grad(out, leaves, t["dout"])[2]
    w = {k: R.wide(v) for k, v in t.items()}
    with np.errstate(over="ignore"):
        eo, _, h, _ = R.recurrence(w["x"], w["gate"], w["z"], w["bias"], None, w["init"])
        e = R.recurrence_grads(w["x"], w["gate"], w["z"], w["bias"], None, w["init"], w["dout"], None)
        s, c = R.sigmoid(w["z"]), R.sigmoid(-w["z"])
    top = np.abs(h).max()
    _within(out, eo, top * np.abs(w["z"]) * s, "out")
    _within(dz, e["dz"], top * np.abs(w["dout"]) * (s + np.abs(w["z"]) * s * c), "dz")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T", [1, 3])
def test_update_with_output_gates_of_any_size(T, dtype):
    B, D = 3, 90
    g = _gen(T)
    x, gate = (torch.randn(B, D, T, generator=g, device="cuda").mul_(0.125).to(dtype) for _ in range(2))
    values = _gates(dtype).cuda()
    z = values[torch.arange(B * D * T, device="cuda").view(B, D, T) % len(values)].to(dtype)
    state = torch.randn(B, D, generator=g, device="cuda") * 0.125
    before = R.wide(state)
    out = gated_recurrence_update(x, state, gate, z)
    w = [R.wide(v) for v in (x, gate, z)]
    with np.errstate(over="ignore"):
        eo, ef, h, _ = R.recurrence(*w, None, None, before)
        size = np.abs(h).max() * np.abs(w[2]) * R.sigmoid(w[2])
    _within(out, eo, size, "out")
    R.check(state, ef, "state")
