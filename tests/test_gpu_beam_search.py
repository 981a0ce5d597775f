"""beam_search_select and beam_search_reorder against their statements."""

import itertools

import pytest
import torch

from causal_conv1d import beam_search_reorder, beam_search_select
from causal_conv1d.beam_search import beam_search_reorder_ref, beam_search_select_ref

pytestmark = pytest.mark.gpu

INF = float("inf")
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _select_and_check(logits, scores, finished=None, end=None, n=None):
    got = beam_search_select(logits, scores, finished, end, n)
    want = beam_search_select_ref(logits, scores, finished, end, n)
    assert [v.dtype for v in got] == [torch.float32, torch.int64, torch.int64]
    assert [v.shape for v in got] == [v.shape for v in want]
    assert torch.equal(got[1], want[1]) and torch.equal(got[2], want[2])
    # a total is rounded once (2^-24) and the sum of exponentials is within 2^-20: 2^v by the
    # hardware 2^-22, its argument |v| <= 126 rounded by 2^-24 |v| with weight exp(-|v|), kept sums
    both = torch.isfinite(want[0])
    assert torch.equal(both, torch.isfinite(got[0])) and torch.equal(got[0][~both], want[0][~both])
    assert ((got[0] - want[0]).abs()[both] <= 2.0 ** -23 * want[0].abs()[both] + 2.0 ** -20).all()
    return got


def _case(seed, batch, beams, vocab, dtype, scale=2.5):
    g = _gen(seed)
    return torch.randn(batch, beams, vocab, generator=g, device="cuda").mul_(scale).to(dtype), -20 * torch.rand(batch, beams, generator=g, device="cuda")


@pytest.mark.parametrize("vocab", [1, 2, 7, 8, 31, 256, 257, 1000, 2049, 5000, 32001])
@pytest.mark.parametrize("dtype", DTYPES)
def test_vocabularies(dtype, vocab):
    for beams, n in ((1, 1), (4, 4), (5, 10)):
        logits, scores = _case(vocab + beams, 3, beams, vocab, dtype)
        _select_and_check(logits, scores, n=min(n, beams * vocab))


@pytest.mark.parametrize("beams,n", [(1, 64), (2, 33), (33, 32), (64, 64), (64, 1), (3, 3), (16, 32)])
@pytest.mark.parametrize("batch", [1, 7])
def test_beams(batch, beams, n):
    logits, scores = _case(beams, batch, beams, 777, DTYPES[beams % 3])
    _select_and_check(logits, scores, n=n)


def test_large():
    logits, scores = _case(1, 64, 8, 100_003, torch.bfloat16)
    _select_and_check(logits, scores, n=16)


@pytest.mark.parametrize("kind", ["any", "masked", "rising", "few values"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_long_rows(dtype, kind):
    """Rows of several steps in each part of a strip, whose largest elements stand at the end, at few places or at many."""
    logits, scores = _case(5, 300, 1, 300_001, dtype)
    if kind == "masked":
        kept = torch.rand(logits.shape, generator=_gen(6), device="cuda") < 1e-5
        logits.masked_fill_(~kept, -INF)
    elif kind == "rising":
        logits = torch.sort(logits, dim=-1).values
    elif kind == "few values":
        logits = logits.round()
    finished = torch.zeros(300, 1, dtype=torch.bool, device="cuda")
    finished[::7] = True
    logits[::7, 0, 1000:] = float("nan")  # not looked at
    scores[1::7] = -INF
    logits[1::7] = float("inf")
    _select_and_check(logits, scores, finished, 3, n=33 if kind == "any" else 8)


@pytest.mark.parametrize("dtype", DTYPES)
def test_ties_go_to_the_lowest_place(dtype):
    logits = torch.zeros(2, 3, 500, device="cuda", dtype=dtype)
    scores = torch.zeros(2, 3, device="cuda")
    got = _select_and_check(logits, scores, n=40)
    assert torch.equal(got[2][0], torch.arange(40, device="cuda")) and (got[1] == 0).all()
    logits = torch.randint(0, 3, (4, 4, 3000), generator=_gen(0), device="cuda").to(dtype)
    _select_and_check(logits, torch.zeros(4, 4, device="cuda"), n=64)
    # -0 and 0 are equal
    logits = torch.zeros(1, 1, 300, device="cuda", dtype=dtype)
    logits[..., ::2] = -0.0
    assert torch.equal(beam_search_select(logits, scores[:1, :1], num_candidates=9)[2][0], torch.arange(9, device="cuda"))


def test_order_of_arrival():
    """Rising and falling logits: every element, or only the first ones, enter the lists."""
    x = torch.linspace(-5, 5, 20_000, device="cuda").expand(1, 2, -1)
    scores = torch.tensor([[0.0, -1.5]], device="cuda")
    for logits in (x, x.flip(-1).contiguous()):
        _select_and_check(logits, scores, n=33)


def test_finished_beams():
    logits, scores = _case(3, 5, 4, 900, torch.float16)
    for flags in itertools.islice(itertools.product([False, True], repeat=4), 1, None):
        finished = torch.tensor([flags] * 5, device="cuda")
        for end in (0, 7, 899):
            _select_and_check(logits, scores, finished, end, 8)
    # nothing but end tokens, then places at -inf
    got = _select_and_check(logits[:, :2, :5], scores[:, :2], torch.ones(5, 2, dtype=torch.bool, device="cuda"), 3, 10)
    assert torch.isinf(got[0][:, 2:]).all()


def test_masked_and_unsound_rows():
    logits, scores = _case(4, 6, 4, 700, torch.float32)
    logits[0, :, 5:] = -INF                              # a grammar that leaves few tokens
    logits[1, 2] = -INF                                  # a beam without any
    logits[2] = -INF                                     # a request without any
    logits[3, 1, 13] = float("nan")
    logits[4, 0, 9] = INF
    logits[5, :, ::2] = torch.finfo(torch.float32).min   # a mask of the lowest value
    for n in (4, 30, 64):
        _select_and_check(logits, scores, n=n)
    first = torch.full((6, 4), -INF, device="cuda")
    first[:, 0] = 0.0                                    # before the first token one beam is in use
    _select_and_check(logits, first, n=8)
    scores[0, 1], scores[1, 0], scores[3, 3] = float("nan"), INF, -INF
    _select_and_check(logits, scores, n=40)
    half = logits.to(torch.bfloat16)
    half[5, :, ::2] = torch.finfo(torch.bfloat16).min
    _select_and_check(half, first, n=64)


def test_far_scores():
    """Beams that start from -1e9, as some programs mark unused ones."""
    logits, scores = _case(6, 2, 3, 400, torch.float32)
    scores[:, 1:] = -1e9
    _select_and_check(logits, scores, n=20)


@pytest.mark.parametrize("dtype", DTYPES)
def test_strides(dtype):
    wide = torch.randn(3, 5, 2 * 1003, generator=_gen(8), device="cuda").to(dtype)
    scores = torch.randn(5, 6, generator=_gen(9), device="cuda").t()
    flags = (torch.rand(5, 6, generator=_gen(10), device="cuda") < 0.3).t()
    for view in (wide[:, :4, 1:1002], wide[..., ::2][:, :4], wide.transpose(0, 1)[:3, :, 3:300], wide[:1, :1, 5:].expand(3, 4, -1)):
        _select_and_check(view, scores[:view.shape[0], :view.shape[1]], flags[:view.shape[0], :view.shape[1]], 1, 7)


def test_select_captured_and_repeated():
    logits, scores = _case(2, 3, 4, 9000, torch.bfloat16)
    beam_search_select(logits, scores)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = beam_search_select(logits, scores)
    for seed in (5, 6):
        a, b = _case(seed, 3, 4, 9000, torch.bfloat16)
        logits.copy_(a)
        scores.copy_(b)
        graph.replay()
        assert all(torch.equal(u, v) for u, v in zip(got, beam_search_select(a, b)))


def test_select_has_no_derivative():
    logits, scores = _case(2, 1, 2, 30, torch.float32)
    best, parents, tokens = beam_search_select(logits.requires_grad_(), scores)
    assert best.requires_grad and not parents.requires_grad and not tokens.requires_grad
    with pytest.raises(RuntimeError, match="no derivative"):
        best.sum().backward()


def test_select_empty_batch():
    got = beam_search_select(torch.empty(0, 2, 9, device="cuda"), torch.empty(0, 2, device="cuda"), num_candidates=3)
    assert [v.shape for v in got] == [(0, 3)] * 3


# ------------------------------------------------------------------------ reordering
def _states(seed, rows, dtype=torch.bfloat16):
    """The convolution's states in both layouts, a recurrence's, and others of odd sizes and types."""
    g = _gen(seed)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    return [r(rows, 3, 70).to(dtype).transpose(1, 2), r(rows, 70, 3).to(dtype), r(rows, 70, 16), r(rows, 33).half(),
            r(rows, 5, 7, 3), torch.randint(0, 99, (rows,), generator=g, device="cuda"),
            torch.randint(0, 2, (rows, 13), generator=g, device="cuda").bool(), r(rows, 4, 100, 18)[:, 1:3, 3:50, ::2], r(rows, 1000)]


@pytest.mark.parametrize("parents_dtype", [torch.int32, torch.int64])
@pytest.mark.parametrize("batch,beams", [(1, 1), (1, 4), (3, 5), (2, 8), (2, 16), (1, 17), (2, 33), (1, 64)])
def test_reorder(batch, beams, parents_dtype):
    states = _states(beams, batch * beams)
    parents = torch.randint(0, beams, (batch, beams), generator=_gen(1), device="cuda").to(parents_dtype)
    want = beam_search_reorder_ref(states, parents)
    before = [t._version for t in states]
    beam_search_reorder(states, parents)
    assert all(torch.equal(a, b) for a, b in zip(states, want))
    assert all(t._version > v for t, v in zip(states, before))
    one = states[2].clone()
    beam_search_reorder(one, parents)
    assert torch.equal(one, beam_search_reorder_ref(states[2], parents))


@pytest.mark.parametrize("parents", [[0, 1, 2, 3], [3, 2, 1, 0], [1, 2, 3, 0], [2, 2, 2, 2], [0, -1, 4, 1], [1, 0, 1, 1 << 40]])
def test_reorder_parents(parents):
    states = _states(3, 4)
    parents = torch.tensor([parents], device="cuda")
    want = beam_search_reorder_ref(states, parents)
    beam_search_reorder(states, parents)
    assert all(torch.equal(a, b) for a, b in zip(states, want))


@pytest.mark.parametrize("index_dtype", [torch.int32, torch.int64])
def test_reorder_pool(index_dtype):
    batch, beams, pool = 3, 4, 20
    states = _states(5, pool)
    index = torch.randperm(pool, generator=_gen(2), device="cuda")[:12].to(index_dtype)
    index[3], index[6], index[9] = -1, 20, 25 if index_dtype == torch.int32 else (1 << 33) + 2
    parents = torch.randint(0, beams, (batch, beams), generator=_gen(3), device="cuda")
    parents[0, 0], parents[1, 1] = 3, 2  # from rows that are none
    want = beam_search_reorder_ref(states, parents, index)
    beam_search_reorder(states, parents, index)
    assert all(torch.equal(a, b) for a, b in zip(states, want))


def test_reorder_many_tensors():
    states = [torch.randn(6, 3 + i, generator=_gen(i), device="cuda") for i in range(60)]
    parents = torch.tensor([[2, 0, 0], [1, 1, 2]], device="cuda")
    want = beam_search_reorder_ref(states, parents)
    beam_search_reorder(states, parents)
    assert all(torch.equal(a, b) for a, b in zip(states, want))


def test_reorder_rows_inside_columns():
    """Rows that lie one element apart, and a pool that is part of a wider one."""
    t = torch.randn(50, 6, generator=_gen(1), device="cuda").t()
    wide = torch.randn(6, 90, generator=_gen(2), device="cuda")
    part, rest = wide[:, 11:64], wide[:, 64:].clone()
    parents = torch.tensor([[1, 2, 0], [2, 2, 1]], device="cuda")
    want = beam_search_reorder_ref([t, part], parents)
    beam_search_reorder([t, part], parents)
    assert torch.equal(t, want[0]) and torch.equal(part, want[1]) and torch.equal(wide[:, 64:], rest)


def test_reorder_nothing():
    beam_search_reorder([], torch.zeros(2, 3, dtype=torch.int64, device="cuda"))
    beam_search_reorder([torch.empty(6, 0, device="cuda")], torch.zeros(2, 3, dtype=torch.int64, device="cuda"))
    beam_search_reorder(torch.empty(0, 4, device="cuda"), torch.zeros(0, 3, dtype=torch.int64, device="cuda"))


def test_reorder_captured():
    state = torch.randn(8, 64, 16, generator=_gen(1), device="cuda")
    parents = torch.zeros(2, 4, dtype=torch.int64, device="cuda")
    beam_search_reorder(state.clone(), parents)
    start = state.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        beam_search_reorder(state, parents)
    for seed in (1, 2):
        state.copy_(start)
        parents.copy_(torch.randint(0, 4, (2, 4), generator=_gen(seed), device="cuda"))
        graph.replay()
        assert torch.equal(state, beam_search_reorder_ref(start, parents))
