"""selective_recurrence_fn and selective_recurrence_update against the 64-bit statement."""

import numpy as np
import pytest
import torch

import selective_ref as S
from causal_conv1d import selective_recurrence_fn, selective_recurrence_update
from causal_conv1d.selective_recurrence import selective_recurrence_bwd_function, selective_recurrence_fwd_function
from helpers import with_layout

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16]
LAYOUTS = ["channel_last", "contiguous", "cl_slice", "rows_slice"]
NAMES = ("x", "delta", "A", "B", "C", "D", "z", "bias", "init")


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _inputs(seed, batch, dim, L, N, dtype, layout="channel_last", groups=0, z=True, skip=True, bias=True, nstates=None):
    """groups 0: B and C without that dimension."""
    g = _gen(seed)

    def rnd(*s, scale=1.0):
        return torch.randn(*s, generator=g, device="cuda") * scale

    def coefficients():
        t = rnd(batch, max(groups, 1), N, L).to(dtype)
        if layout in ("channel_last", "cl_slice"):
            wide = torch.full((batch, L, max(groups, 1) * N + 5), float("nan"), device="cuda", dtype=dtype)
            view = wide[..., 3:3 + max(groups, 1) * N].unflatten(-1, (max(groups, 1), N)).permute(0, 2, 3, 1)
            t = view.copy_(t)
        return t if groups else t[:, 0]

    return {"x": with_layout(rnd(batch, dim, L).to(dtype), layout), "delta": with_layout(rnd(batch, dim, L).to(dtype), layout),
            "A": -torch.exp(rnd(dim, N, scale=0.7)), "B": coefficients(), "C": coefficients(), "D": rnd(dim) if skip else None,
            "z": with_layout(rnd(batch, dim, L).to(dtype), layout) if z else None, "bias": rnd(dim) - 1.0 if bias else None,
            "init": rnd(nstates, dim, N) if nstates else None, "dout": with_layout(rnd(batch, dim, L).to(dtype), layout),
            "dfinal": rnd(nstates, dim, N) if nstates else None}


def _packing(seed, batch, L, nseq, pad=True):
    """Row-unique ids in runs of random lengths, some padding between and after them."""
    r = np.random.default_rng(seed)
    ids = np.full((batch, L), -1, np.int32)
    for b in range(batch):
        edges = [0, *np.sort(r.integers(0, L + 1, nseq - 1)).tolist(), L]
        for k in range(nseq):
            lo, hi = edges[k], edges[k + 1]
            if pad and hi - lo > 4 and r.random() < 0.4:
                hi -= int(r.integers(1, hi - lo - 1))
            ids[b, lo:hi] = b * nseq + k
    return ids


def _run_and_check(t, ids=None, softplus=True):
    """Forward and backward through autograd, every output and gradient against fp64."""
    leaves = {k: t[k].detach().requires_grad_() for k in NAMES if t[k] is not None}
    seq = None if ids is None else torch.from_numpy(ids).cuda()
    kept = t["init"] is not None
    args = [leaves.get(k) for k in ("x", "delta", "A", "B", "C", "D", "z", "bias")]
    got = selective_recurrence_fn(*args, delta_softplus=softplus, seq_idx=seq, initial_states=leaves.get("init"),
                                  return_final_states=kept)
    out, final = got if kept else (got, None)
    outs, grads = ([out, final], [t["dout"], t["dfinal"]]) if kept else ([out], [t["dout"]])
    found = dict(zip(leaves, torch.autograd.grad(outs, list(leaves.values()), grads)))
    e = S.statement(S.fp64(t), ids, use_softplus=softplus)
    S.check(out, e["out"], "out")
    assert out.dtype == t["x"].dtype and out.stride() == torch.empty_like(t["x"]).stride()
    if kept:
        assert final.dtype == torch.float32
        S.check(final, e["final"], "final_states")
    for k, g in found.items():
        assert g.dtype == t[k].dtype
        S.check(g, e["d" + k], "d" + k)
    with torch.no_grad():
        plain = selective_recurrence_fn(t["x"], t["delta"], t["A"], t["B"], t["C"], t["D"], t["z"], t["bias"],
                                        delta_softplus=softplus, seq_idx=seq, initial_states=t["init"])
    assert torch.equal(plain, out)
    return out, final, found


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("L", [1, 2, 4, 5, 31, 32, 33, 64, 130])
def test_lengths(L, dtype, layout):
    _run_and_check(_inputs(L, 2, 40, L, 16, dtype, layout, nstates=2))


@pytest.mark.parametrize("layout", ["channel_last", "contiguous"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N", [1, 2, 3, 4, 5, 8, 9, 12, 15, 16, 17, 20, 32, 33, 64])
def test_states(N, dtype, layout):
    _run_and_check(_inputs(N, 2, 37, 45, N, dtype, layout, nstates=2))


@pytest.mark.parametrize("N", [100, 128, 200, 256])
def test_many_states(N):
    _run_and_check(_inputs(N, 1, 35, 70, N, torch.bfloat16, nstates=1))


@pytest.mark.parametrize("N", [3, 7, 16])
@pytest.mark.parametrize("layout", ["channel_last", "contiguous"])
@pytest.mark.parametrize("D", [1, 2, 31, 32, 33, 64, 129])
def test_channels(D, layout, N):
    _run_and_check(_inputs(D, 3, D, 50, N, DTYPES[D % 3], layout, nstates=3))


@pytest.mark.parametrize("groups,D", [(1, 40), (2, 66), (3, 99), (5, 5), (4, 256)])
@pytest.mark.parametrize("layout", ["channel_last", "contiguous"])
def test_groups(groups, D, layout):
    _run_and_check(_inputs(D, 2, D, 70, 16, DTYPES[groups % 3], layout, groups=groups, nstates=2))


@pytest.mark.parametrize("z,skip,bias,states", [(False, False, False, False), (True, False, False, False),
                                                (False, True, False, True), (False, False, True, True), (True, True, True, False)])
@pytest.mark.parametrize("softplus", [True, False])
@pytest.mark.parametrize("dtype", DTYPES)
def test_optional_inputs(dtype, softplus, z, skip, bias, states):
    t = _inputs(5, 2, 48, 100, 16, dtype, "channel_last", 0, z, skip, bias, 2 if states else None)
    if not softplus:  # the step sizes themselves
        t["delta"] = t["delta"].abs()
        t["bias"] = None if t["bias"] is None else t["bias"].abs()
    _run_and_check(t, softplus=softplus)


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,D,L,nseq,states", [(1, 40, 200, 6, True), (2, 33, 131, 40, True), (1, 64, 400, 3, False), (3, 20, 64, 2, True)])
def test_packed(B, D, L, nseq, states, dtype, layout):
    t = _inputs(nseq, B, D, L, 16, dtype, layout, nstates=B * nseq if states else None)
    _run_and_check(t, _packing(L + nseq, B, L, nseq))


@pytest.mark.parametrize("N", [4, 6, 20])
def test_packed_states(N):
    _run_and_check(_inputs(N, 2, 33, 150, N, torch.float32, nstates=10), _packing(N, 2, 150, 5))


@pytest.mark.parametrize("B,D,L", [(1, 64, 3000), (1, 16, 5000), (2, 130, 1027), (1, 7, 2049)])
@pytest.mark.parametrize("layout", ["channel_last", "contiguous"])
def test_long(B, D, L, layout):
    _run_and_check(_inputs(B + L, B, D, L, 16, DTYPES[(B + D) % 3], layout, nstates=B))


@pytest.mark.parametrize("D,L,nseq", [(32, 2500, 7), (20, 3001, 90)])
def test_long_packed(D, L, nseq):
    _run_and_check(_inputs(D, 1, D, L, 16, torch.float32, nstates=nseq), _packing(L, 1, L, nseq))


def _update(t, state, index=None, one=False):
    pick = (lambda v: None if v is None else v[..., 0]) if one else (lambda v: v)
    return selective_recurrence_update(pick(t["x"]), state, pick(t["delta"]), t["A"], pick(t["B"]), pick(t["C"]), t["D"],
                                       pick(t["z"]), t["bias"], state_indices=index)


@pytest.mark.parametrize("N", [1, 3, 4, 8, 15, 16, 24, 32, 64, 100, 128, 130, 256])
@pytest.mark.parametrize("dtype", DTYPES)
def test_update(dtype, N):
    for L, one in ((1, True), (1, False), (3, False)):
        t = _inputs(N, 5, 33, L, N, dtype, nstates=5)
        state = t["init"].clone()
        out = _update(t, state, one=one)
        t["dout"] = None
        e = S.statement(S.fp64(t))
        S.check(state, e["final"], "state")
        S.check(out, tuple(v[..., 0] for v in e["out"]) if one else e["out"], "out")


@pytest.mark.parametrize("groups", [1, 2, 3])
@pytest.mark.parametrize("index_dtype", [torch.int32, torch.int64])
def test_update_pool(index_dtype, groups):
    t = _inputs(9, 4, 66, 2, 16, torch.bfloat16, groups=groups, nstates=4)
    pool = torch.randn(11, 66, 16, generator=_gen(1), device="cuda")
    before = pool.clone()
    index = torch.tensor([7, -1, 3, 11], device="cuda", dtype=index_dtype)
    out = _update(t, pool, index)
    rows = [0, 2]
    t["init"] = before[[7, 3]]
    for k in ("x", "delta", "B", "C", "z"):
        t[k] = t[k][rows]
    t["dout"] = None
    e = S.statement(S.fp64(t))
    S.check(pool[[7, 3]], e["final"], "state")
    S.check(out[rows], e["out"], "out")
    assert (out[[1, 3]] == 0).all()
    others = [i for i in range(11) if i not in (7, 3)]
    assert torch.equal(pool[others], before[others])


@pytest.mark.parametrize("N", [4, 8, 12, 16, 32, 64, 128, 256])
@pytest.mark.parametrize("dtype", DTYPES)
def test_update_packed(dtype, N):
    """States, B and C on 16 bytes, which move four at a time; batches that do not fill the last rows."""
    for batch, groups, z, pool in ((1, 0, True, False), (3, 0, False, True), (4, 2, True, True), (9, 0, True, False), (6, 1, True, True)):
        t = _inputs(N + batch, batch, 38, 1, N, dtype, "contiguous", groups, z, nstates=batch)
        state = torch.randn(batch + 5, 38, N, generator=_gen(3), device="cuda") if pool else t["init"].clone()
        index = torch.randperm(batch + 5, generator=_gen(4), device="cuda")[:batch] if pool else None
        if pool:
            index[batch // 2] = -1
            t["init"] = state[index.clamp(min=0)]
        before = state.clone()
        one = {k: (v[..., 0].contiguous() if k in ("x", "delta", "B", "C", "z") and v is not None else v) for k, v in t.items()}
        out = selective_recurrence_update(*(one[k] if k != "state" else state for k in ("x", "state", "delta", "A", "B", "C", "D", "z", "bias")),
                                          state_indices=index)
        t["dout"] = None
        e = S.statement(S.fp64(t))
        rows = list(range(batch)) if index is None else [k for k in range(batch) if k != batch // 2]
        S.check(out[rows], tuple(v[rows, :, 0] for v in e["out"]), "out")
        at = rows if index is None else index[rows].tolist()
        S.check(state[at], tuple(v[rows] for v in e["final"]), "state")
        if pool:
            assert (out[batch // 2] == 0).all()
            others = [i for i in range(batch + 5) if i not in at]
            assert torch.equal(state[others], before[others])


def test_update_continues_prefill():
    """The steps after a prefill give what one longer pass gives."""
    t = _inputs(3, 2, 70, 60, 16, torch.float32)
    cut = {k: (v[..., :40] if k in ("x", "delta", "B", "C", "z") else v) for k, v in t.items()}
    args = lambda w: [w[k] for k in ("x", "delta", "A", "B", "C", "D", "z", "bias")]  # noqa: E731
    whole, last = selective_recurrence_fn(*args(t), return_final_states=True)
    _, state = selective_recurrence_fn(*args(cut), return_final_states=True)
    for i in range(40, 60):
        step = {k: (v[..., i:i + 1] if k in ("x", "delta", "B", "C", "z") else v) for k, v in t.items()}
        out = _update(step, state, one=True)
        torch.testing.assert_close(out, whole[..., i], rtol=1e-5, atol=1e-5)
    torch.testing.assert_close(state, last, rtol=1e-5, atol=1e-5)


def test_padding_is_not_read():
    """NaN and infinity at padding positions reach nothing, and gradients there are zero."""
    t = _inputs(8, 2, 40, 120, 16, torch.bfloat16, nstates=6)
    ids = _packing(4, 2, 120, 3)
    ids[0, :5] = -1
    want = _run_and_check(t, ids)
    pad = torch.from_numpy(ids < 0).cuda().unsqueeze(1)
    assert pad.any()
    for k in ("x", "delta", "z", "dout", "B", "C"):
        t[k] = torch.where(pad, float("nan") if k != "B" else float("inf"), t[k])
    leaves = {k: t[k].detach().requires_grad_() for k in NAMES}
    out, final = selective_recurrence_fn(*[leaves[k] for k in ("x", "delta", "A", "B", "C", "D", "z", "bias")],
                                         seq_idx=torch.from_numpy(ids).cuda(), initial_states=leaves["init"], return_final_states=True)
    found = torch.autograd.grad([out, final], list(leaves.values()), [t["dout"], t["dfinal"]])
    assert torch.equal(out, want[0]) and torch.equal(final, want[1])
    for (k, g) in zip(leaves, found):
        assert torch.equal(g, want[2][k]), k


def test_a_sequence_keeps_its_nan():
    """A NaN spoils its own sequence from there on, and nothing of the next one."""
    t = _inputs(8, 1, 36, 100, 16, torch.float32, nstates=2)
    ids = np.repeat(np.array([[0, 1]], np.int32), 50, 1)
    clean = _run_and_check(t, ids)
    t["x"] = t["x"].clone()
    t["x"][0, 3, 20] = float("nan")
    seq = torch.from_numpy(ids).cuda()
    args = [t[k] for k in ("x", "delta", "A", "B", "C", "D", "z", "bias")]
    out, final = selective_recurrence_fn(*args, seq_idx=seq, initial_states=t["init"], return_final_states=True)
    bad = torch.isnan(out)
    assert bad[0, 3, 20:50].all() and bad.sum() == 30
    assert torch.equal(out[~bad], clean[0][~bad])
    assert torch.isnan(final[0, 3]).all() and torch.isnan(final).sum() == 16


def test_empty():
    for B, D, L in ((0, 8, 5), (2, 0, 5), (2, 8, 0)):
        x = torch.randn(B, D, L, device="cuda", requires_grad=True)
        A = -torch.ones(D, 4, device="cuda").requires_grad_()
        bc = torch.randn(B, 4, L, device="cuda", requires_grad=True)
        skip = torch.ones(D, device="cuda", requires_grad=True)
        init = torch.randn(B, D, 4, device="cuda", requires_grad=True)
        out, final = selective_recurrence_fn(x, x, A, bc, bc, skip, initial_states=init, return_final_states=True)
        assert out.shape == x.shape and torch.equal(final, init)
        g = torch.autograd.grad([out, final], [x, A, bc, skip, init], [torch.ones_like(out), torch.ones_like(final)])
        assert (g[1] == 0).all() and (g[3] == 0).all() and (g[4] == 1).all()
        if L == 0:
            assert torch.equal(selective_recurrence_update(x.detach(), init.detach(), x.detach(), A.detach(), bc.detach(), bc.detach()), out)


def test_results_repeat_and_other_stream():
    t = _inputs(8, 2, 70, 300, 16, torch.bfloat16, nstates=2)
    args = [t[k] for k in ("x", "delta", "A", "B", "C", "D", "z", "bias")]

    def both():
        out, final, kept = selective_recurrence_fwd_function(*args, True, None, t["init"], True, None, True)
        g = selective_recurrence_bwd_function(*args, True, None, t["init"], kept, t["dout"], t["dfinal"], True, True)
        return [out, final, *g]

    want = both()
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(both(), want))
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = both()
    torch.cuda.current_stream().wait_stream(stream)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_captured():
    """Forward, backward and token update in one graph, replayed on new inputs."""
    t, other = (_inputs(s, 2, 70, 300, 16, torch.bfloat16, nstates=2) for s in (8, 9))
    state = t["init"].clone()

    def step(w, st):
        leaves = [w[k].detach().requires_grad_() for k in ("x", "delta", "A", "B", "C", "D", "z", "bias")]
        out, final = selective_recurrence_fn(*leaves, initial_states=w["init"], return_final_states=True)
        g = torch.autograd.grad([out, final], leaves, [w["dout"], w["dfinal"]])
        one = selective_recurrence_update(*(w["x"][..., 0], st, w["delta"][..., 0], w["A"], w["B"][..., 0], w["C"][..., 0]))
        return [out.detach(), final.detach(), *g, one]

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step(t, state)
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(t, state)
    for k, v in other.items():
        t[k].copy_(v)
    state.copy_(other["init"])
    graph.replay()
    after = other["init"].clone()
    want = step(other, after)
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and torch.equal(state, after)


def test_gradients_of_absent_inputs():
    """Without delta_bias and initial_states the backward pass gives the gradients of zeros, if it is asked for them."""
    t = _inputs(4, 2, 34, 45, 5, torch.bfloat16, nstates=2)
    args = [t[k] for k in ("x", "delta", "A", "B", "C", "D", "z")]
    zeros = [torch.zeros(34, device="cuda"), torch.zeros_like(t["init"])]
    found = []
    for bias, init in ((None, None), zeros):
        kept = selective_recurrence_fwd_function(*args, bias, True, None, init, False, None, True)[2]
        found.append(selective_recurrence_bwd_function(*args, bias, True, None, init, kept, t["dout"], None, True, True))
        fewer = selective_recurrence_bwd_function(*args, bias, True, None, init, kept, t["dout"], None, False, False)
        assert fewer[7] is None and fewer[8] is None
    assert all(torch.equal(a, b) and a.dtype == b.dtype for a, b in zip(*found))


def test_derivatives_are_refused():
    t = _inputs(1, 1, 8, 20, 4, torch.float32, nstates=1)
    args = [t[k] for k in ("x", "delta", "A", "B", "C")]
    x = t["x"].detach().requires_grad_()
    (g,) = torch.autograd.grad(selective_recurrence_fn(x, *args[1:]).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        torch.autograd.grad(g.sum(), x)
    with pytest.raises(NotImplementedError, match="forward-mode"), torch.autograd.forward_ad.dual_level():
        selective_recurrence_fn(torch.autograd.forward_ad.make_dual(t["x"], t["x"]), *args[1:])
    one = [x[..., 0], t["delta"][..., 0], t["A"], t["B"][..., 0], t["C"][..., 0]]
    version = t["init"]._version
    out = selective_recurrence_update(one[0], t["init"], *one[1:])
    assert t["init"]._version > version and not t["init"].requires_grad
    with pytest.raises(RuntimeError, match="no derivative"):
        out.sum().backward()


def test_gradients_of_some_inputs():
    """What is asked for does not depend on what else is, and a missing gradient counts as zero."""
    t = _inputs(2, 2, 40, 70, 16, torch.float32, nstates=2)
    names = ("x", "delta", "A", "B", "C", "D", "z", "bias", "init")

    def grads(wanted, outs):
        leaves = {k: t[k].detach().requires_grad_(k in wanted) for k in names}
        got = selective_recurrence_fn(*[leaves[k] for k in names[:8]], initial_states=leaves["init"], return_final_states=True)
        return torch.autograd.grad([got[i] for i in outs], [leaves[k] for k in wanted], [(t["dout"], t["dfinal"])[i] for i in outs])

    every = dict(zip(names, grads(names, (0, 1))))
    for k in names:
        assert torch.equal(grads([k], (0, 1))[0], every[k]), k
    for i, zero in ((0, "dfinal"), (1, "dout")):
        w = dict(t)
        w[zero] = torch.zeros_like(t[zero])
        e = S.statement(S.fp64(w))
        for k, g in zip(names, grads(names, (i,))):
            S.check(g, e["d" + k], "d" + k)


def test_parameters_of_other_types():
    t = _inputs(4, 2, 40, 70, 16, torch.float16, nstates=2)
    for k, dtype in (("A", torch.bfloat16), ("D", torch.float16), ("bias", torch.bfloat16)):
        t[k] = t[k].to(dtype)
    _run_and_check(t)


@pytest.mark.parametrize("rows", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("start,D", [(1, 64), (2, 64), (3, 96), (1, 63)])
def test_tensors_that_start_anywhere(start, D, dtype, rows):
    """Slices of wider tensors that are NaN around them, off the alignment of pairs of channels."""
    t = _inputs(start + D, 2, D, 70, 16, dtype, "contiguous" if rows else "channel_last", nstates=2)
    for k in ("x", "delta", "z", "dout"):
        v = t[k] if rows else t[k].transpose(1, 2)
        wide = torch.full((v.shape[0], v.shape[1], v.shape[2] + 7), float("nan"), device="cuda", dtype=dtype)
        wide[..., start:start + v.shape[2]] = v
        view = wide[..., start:start + v.shape[2]]
        t[k] = view if rows else view.transpose(1, 2)
    leaves = {k: t[k].detach().requires_grad_() for k in NAMES}
    out, final = selective_recurrence_fn(*[leaves[k] for k in ("x", "delta", "A", "B", "C", "D", "z", "bias")],
                                         initial_states=leaves["init"], return_final_states=True)
    found = dict(zip(leaves, torch.autograd.grad([out, final], list(leaves.values()), [t["dout"], t["dfinal"]])))
    e = S.statement(S.fp64(t))
    S.check(out, e["out"], "out")
    S.check(final, e["final"], "final")
    for k, g in found.items():
        S.check(g, e["d" + k], "d" + k)


def test_mixed_layouts_and_broadcast_inputs():
    t = _inputs(6, 3, 40, 50, 16, torch.float16, "channel_last", nstates=3)
    t["delta"] = t["delta"].contiguous()
    t["B"] = t["B"].contiguous()                                   # along the sequence, C along the states
    t["z"] = t["z"][:1].expand(3, -1, -1)                          # one output gate for all rows
    t["C"] = t["C"][:1].expand(3, -1, -1)
    t["dout"] = t["dout"][:, :, :1].expand(-1, -1, 50)
    leaves = {k: t[k].detach().requires_grad_() for k in NAMES}
    out = selective_recurrence_fn(*[leaves[k] for k in ("x", "delta", "A", "B", "C", "D", "z", "bias")], initial_states=leaves["init"])
    found = dict(zip(leaves, torch.autograd.grad(out, list(leaves.values()), t["dout"])))
    t["dfinal"] = None
    e = S.statement(S.fp64(t))
    S.check(out, e["out"], "out")
    for k, g in found.items():
        assert g.shape == t[k].shape
        S.check(g, e["d" + k], "d" + k)
    # a leaf that is broadcast gets the sum
    z = t["z"][:1].detach().clone().requires_grad_()
    out = selective_recurrence_fn(*[t[k] for k in ("x", "delta", "A", "B", "C", "D")], z.expand(3, -1, -1), t["bias"], initial_states=t["init"])
    (g,) = torch.autograd.grad(out, z, t["dout"])
    want, bound = e["dz"]
    # each of the three is rounded to fp16 before torch adds them there
    S.check(g, (want.sum(0, keepdims=True), bound.sum(0, keepdims=True) + 4 * 2.0 ** -11 * np.abs(want).sum(0, keepdims=True)), "dz")


def test_slow_and_fast_states():
    """Memories of thousands of steps and of less than one, steps from 1e-4 to 30."""
    t = _inputs(7, 1, 64, 4000, 8, torch.float32, nstates=1)
    t["A"] = -torch.logspace(-4, 2, 8, device="cuda").repeat(64, 1)
    t["bias"] = torch.linspace(-9, 3, 64, device="cuda")
    t["delta"] = t["delta"] * 0.3
    _run_and_check(t)


@pytest.mark.parametrize("u", [-100.0, -60.0, -20.0, -1e-3, 0.0, 15.0, 40.0, 100.0])
def test_step_sizes(u):
    """softplus and its slope to full relative precision: small steps count over long sequences."""
    D, L = 32, 8
    delta = torch.linspace(u - 0.5, u + 0.5, D * L, device="cuda").view(1, D, L)
    x, A = torch.ones(1, D, L, device="cuda"), torch.zeros(D, 1, device="cuda")
    bc = torch.ones(1, 1, L, device="cuda")
    leaf = delta.clone().requires_grad_()
    out = selective_recurrence_fn(x, leaf, A, bc, bc)  # the running sum of the steps
    w = delta.double()
    step = torch.clamp(w, min=0) + torch.log1p(torch.exp(-w.abs()))
    # eight positive terms: each to 2^-21 of itself, the sum's roundings 8 2^-24; below 2^-126 all is zero
    want = step.cumsum(2)
    assert ((out.double() - want).abs() <= 2.0 ** -19 * want + 2.0 ** -125 * 8).all()
    (g,) = torch.autograd.grad(out[..., -1].sum(), leaf)
    slope = torch.sigmoid(w)
    assert ((g.double() - slope).abs() <= 2.0 ** -19 * slope + 2.0 ** -125).all()


def test_batches_that_the_backward_splits():
    """The sums of dB and dC of all rows would take over 2 GB: some rows at a time."""
    t = _inputs(5, 9, 512, 8192, 64, torch.bfloat16, nstates=None)
    t["z"], args = None, ("x", "delta", "A", "B", "C", "D", "z", "bias")

    def grads(w):
        leaves = {k: w[k].detach().requires_grad_() for k in args if w[k] is not None}
        out = selective_recurrence_fn(*[leaves.get(k) for k in args])
        return dict(zip(leaves, torch.autograd.grad(out, list(leaves.values()), w["dout"])))

    whole = grads(t)
    total = {k: torch.zeros_like(t[k], dtype=torch.float64) for k in ("A", "D", "bias")}
    for b in (0, 3, 6, 7, 8):  # on both sides of the splits
        part = grads({k: (v[b:b + 1] if v is not None and v.dim() == 3 else v) for k, v in t.items()})
        for k in ("x", "delta", "B", "C"):
            # the same sums over other parts of the sequence: fp32 roundings, then bf16's
            torch.testing.assert_close(whole[k][b:b + 1], part[k], rtol=2.0 ** -7, atol=2.0 ** -16 * part[k].abs().max().item())
    for b in range(9):
        part = grads({k: (v[b:b + 1] if v is not None and v.dim() == 3 else v) for k, v in t.items()})
        for k in total:
            total[k] += part[k].double()
    for k in total:
        torch.testing.assert_close(whole[k].double(), total[k], rtol=1e-4, atol=1e-4 * total[k].abs().max().item())


@pytest.mark.parametrize("layout", ["channel_last", "contiguous"])
@pytest.mark.parametrize("D,L", [(72, 30_000_128), (71, 30_300_007)])
def test_offsets_past_32_bits(D, L, layout):
    """The ends of a long sequence are what the statements of short stretches give."""
    g = _gen(D)
    x = torch.randn(1, L, D, generator=g, device="cuda", dtype=torch.bfloat16)
    x = x.transpose(1, 2) if layout == "channel_last" else x.view(1, D, L)
    bc = torch.randn(1, L, 2, generator=g, device="cuda", dtype=torch.bfloat16).transpose(1, 2)
    A = -torch.exp(torch.randn(D, 2, generator=g, device="cuda"))
    dfinal = torch.randn(1, D, 2, generator=g, device="cuda")
    args = (x, x, A, bc, bc, None, None, None, True, None)
    _, _, kept = selective_recurrence_fwd_function(*args, None, False, None, True)
    dx, ddelta, _, dB, dC, _, _, _, _ = selective_recurrence_bwd_function(*args, None, kept, x, dfinal, False, False)
    n = 501
    cut = (x[:, :, :L - n], x[:, :, :L - n], A, bc[:, :, :L - n], bc[:, :, :L - n], None, None, None, True, None)
    out, mid, _ = selective_recurrence_fwd_function(*cut, None, True, None, False)
    del out

    def stretch(lo, hi, init, last):
        v = {k: S.wide(w[:, :, lo:hi]) for k, w in (("x", x), ("delta", x), ("B", bc), ("C", bc), ("dout", x))}
        return S.statement({**v, "A": S.wide(A), "init": None if init is None else S.wide(init), "dfinal": None if last is None else S.wide(last)})

    e = stretch(L - n, L, mid, dfinal)
    for k, got in (("dx", dx), ("ddelta", ddelta), ("dB", dB), ("dC", dC)):
        S.check(got[:, :, L - n:], e[k], k + ", tail")
    # the first ones, whose gradients forget what lies 400 positions on (steps of 0.7 and more on average)
    e = stretch(0, n + 400, None, None)
    for k, got in (("dx", dx), ("ddelta", ddelta), ("dB", dB), ("dC", dC)):
        S.check(got[:, :, :n], tuple(w[:, :, :n] for w in e[k]), k + ", head")


def test_two_calls_at_once():
    """Calls on two streams, and two graphs that are replayed in turn, have workspaces of their own."""
    ts = [_inputs(s, 1, 64, 2000, 16, torch.bfloat16, nstates=1) for s in (1, 2)]

    def both(t):
        args = [t[k] for k in ("x", "delta", "A", "B", "C", "D", "z", "bias")]
        out, final, kept = selective_recurrence_fwd_function(*args, True, None, t["init"], True, None, True)
        return [out, final, *selective_recurrence_bwd_function(*args, True, None, t["init"], kept, t["dout"], t["dfinal"], True, True)]

    want = [both(t) for t in ts]
    streams = [torch.cuda.Stream() for _ in ts]
    torch.cuda.synchronize()
    got = []
    for _ in range(3):
        for t, stream in zip(ts, streams):
            with torch.cuda.stream(stream):
                got.append(both(t))
    torch.cuda.synchronize()
    for i, g in enumerate(got):
        assert all(torch.equal(a, b) for a, b in zip(g, want[i % 2]))
    graphs = []
    for t in ts:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=graphs[0][0].pool() if graphs else None):
            graphs.append((graph, both(t)))
    for i in (0, 1, 1, 0):
        graphs[i][0].replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(graphs[i][1], want[i]))
