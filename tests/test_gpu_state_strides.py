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
