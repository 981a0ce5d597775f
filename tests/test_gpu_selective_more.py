"""selective_recurrence_fn and selective_recurrence_update where a call has many states, several tokens or nothing."""

import pytest
import torch

import selective_ref as S
from causal_conv1d import selective_recurrence_fn, selective_recurrence_update
from test_gpu_selective import DTYPES, _gen, _inputs, _packing, _run_and_check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("N", [68, 100, 128, 200, 256])
@pytest.mark.parametrize("layout", ["channel_last", "contiguous"])
@pytest.mark.parametrize("dtype", DTYPES)
def test_many_states(N, layout, dtype):
    """Several passes over a tile: groups, batches, tiles that are not full."""
    for groups, D, L in ((0, 19, 45), (2, 34, 64), (3, 9, 33)):
        _run_and_check(_inputs(N + D, 2, D, L, N, dtype, layout, groups, nstates=2))


@pytest.mark.parametrize("N", [72, 128, 256])
@pytest.mark.parametrize("layout", ["channel_last", "contiguous"])
@pytest.mark.parametrize("dtype", DTYPES)
def test_many_states_packed(N, layout, dtype):
    for L, nseq, groups in ((100, 4, 0), (150, 30, 2)):
        _run_and_check(_inputs(N + L, 2, 18, L, N, dtype, layout, groups, nstates=2 * nseq), _packing(L, 2, L, nseq))


@pytest.mark.parametrize("layout", ["channel_last", "contiguous"])
def test_many_states_long(layout):
    """A sequence that is cut into parts, whole and packed."""
    t = _inputs(3, 1, 12, 1500, 80, torch.float32, layout, nstates=5)
    whole = dict(t)
    whole["init"], whole["dfinal"] = t["init"][:1], t["dfinal"][:1]
    _run_and_check(whole)
    _run_and_check(t, _packing(9, 1, 1500, 5))


@pytest.mark.parametrize("N", [4, 8, 12, 16, 32, 64, 128, 256])
@pytest.mark.parametrize("dtype", DTYPES)
def test_update_of_several_tokens(dtype, N):
    """States, B and C on 16 bytes, which move four at a time, with several tokens of each row."""
    for batch, groups, z, pool, L in ((3, 0, True, False, 2), (4, 2, False, True, 4), (7, 1, True, True, 3)):
        t = _inputs(N + batch, batch, 38, L, N, dtype, "contiguous", groups, z, nstates=batch)
        for k in ("B", "C"):  # states side by side
            t[k] = t[k].movedim(-1, 1).contiguous().movedim(1, -1)
        state = torch.randn(batch + 5, 38, N, generator=_gen(3), device="cuda") if pool else t["init"].clone()
        index = torch.randperm(batch + 5, generator=_gen(4), device="cuda")[:batch] if pool else None
        if pool:
            index[batch // 2] = -1
            t["init"] = state[index.clamp(min=0)]
        before = state.clone()
        out = selective_recurrence_update(*(state if k == "state" else t[k] for k in ("x", "state", "delta", "A", "B", "C", "D", "z", "bias")),
                                          state_indices=index)
        t["dout"] = None
        e = S.statement(S.fp64(t))
        rows = list(range(batch)) if index is None else [k for k in range(batch) if k != batch // 2]
        S.check(out[rows], tuple(v[rows] for v in e["out"]), "out")
        at = rows if index is None else index[rows].tolist()
        S.check(state[at], tuple(v[rows] for v in e["final"]), "state")
        if pool:
            assert (out[batch // 2] == 0).all()
            others = [i for i in range(batch + 5) if i not in at]
            assert torch.equal(state[others], before[others])


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
