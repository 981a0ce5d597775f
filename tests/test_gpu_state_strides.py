"""States that are strided slices of wider tensors."""

import pytest
import torch

import selective_ref as S
from causal_conv1d import beam_search_reorder, selective_recurrence_update
from causal_conv1d.beam_search import beam_search_reorder_ref
from test_gpu_selective import _gen, _inputs

pytestmark = pytest.mark.gpu


def _slices(rows, dim, n):
    """(rows, dim, n) states: every other element of an odd row, channels, rows, and one order of dimensions."""
    g = _gen(n)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    return [r(rows, dim, 2 * n - 1)[..., ::2], r(rows, 2 * dim - 1, n)[:, ::2], r(2 * rows - 1, dim, n)[::2],
            r(rows, 3 * dim - 2, 2 * n - 1)[:, ::3, ::2], r(n, 2 * rows - 1, 2 * dim - 1)[:, ::2, ::2].permute(1, 2, 0)]


def _base(t):
    return t if t._base is None else t._base


@pytest.mark.parametrize("n", [3, 4, 16])
def test_update(n):
    t = _inputs(n, 4, 10, 2, n, torch.float32, nstates=4)
    t["dout"] = None
    e = S.statement(S.fp64(t))
    for state in _slices(4, 10, n):
        whole = _base(state)
        inside = torch.zeros_like(whole, dtype=torch.bool)
        inside.as_strided(state.shape, state.stride(), state.storage_offset()).fill_(True)
        before = whole.clone()
        state.copy_(t["init"])
        out = selective_recurrence_update(*(state if k == "state" else t[k] for k in ("x", "state", "delta", "A", "B", "C", "D", "z", "bias")))
        S.check(out, e["out"], "out")
        S.check(state, e["final"], "state")
        assert torch.equal(whole[~inside], before[~inside])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.bool, torch.complex64])
def test_reorder(dtype):
    parents = torch.tensor([[1, 1, 2], [2, 0, 1]], device="cuda")
    for state in _slices(6, 10, 7):
        wide = _base(state)
        whole = (wide > 0) if dtype == torch.bool else wide.to(dtype)
        state = whole.as_strided(state.shape, state.stride(), state.storage_offset())
        inside = torch.zeros_like(whole, dtype=torch.bool)
        inside.as_strided(state.shape, state.stride(), state.storage_offset()).fill_(True)
        before, want = whole.clone(), beam_search_reorder_ref(state, parents)
        beam_search_reorder(state, parents)
        assert torch.equal(state, want) and torch.equal(whole[~inside], before[~inside])


@pytest.mark.parametrize("beams", [2, 16, 17, 32, 33, 64])
@pytest.mark.parametrize("dtype", [torch.uint8, torch.float16, torch.float32, torch.float64, torch.complex128])
def test_reorder_elements_in_three_dimensions(dtype, beams):
    """Single elements of any size, with fewer and with more beams than move whole elements."""
    values = torch.randint(0, 200, (2 * beams, 5, 12, 13), generator=_gen(beams), device="cuda").to(dtype)
    wide = values[:, ::2, ::3, ::2]
    parents = torch.randint(0, beams, (2, beams), generator=_gen(1), device="cuda")
    for state in (wide, values.flatten()[1:1 + 2 * beams * 64].view(2 * beams, 64)[:, :60].unflatten(1, (5, 3, 4))[..., ::2]):
        before, rest = values.clone(), torch.ones_like(values, dtype=torch.bool)
        rest.as_strided(state.shape, state.stride(), state.storage_offset()).fill_(False)
        want = beam_search_reorder_ref(state, parents)
        beam_search_reorder(state, parents)
        assert torch.equal(state, want) and torch.equal(values[rest], before[rest])
