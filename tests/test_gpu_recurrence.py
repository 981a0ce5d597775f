"""gated_recurrence_fn and gated_recurrence_update against the 64-bit statement."""

import numpy as np
import pytest
import torch

import block_ref as R
from causal_conv1d import gated_recurrence_fn, gated_recurrence_update
from causal_conv1d.gated_recurrence import gated_recurrence_bwd_function, gated_recurrence_fwd_function
from helpers import with_layout

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16]
LAYOUTS = ["channel_last", "contiguous", "cl_slice", "rows_slice"]


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _inputs(seed, B, D, L, dtype, layout, z=True, bias=True, nstates=None):
    g = _gen(seed)

    def rnd(*s, scale=1.0):
        return torch.randn(*s, generator=g, device="cuda") * scale

    t = {"x": with_layout(rnd(B, D, L).to(dtype), layout), "gate": with_layout(rnd(B, D, L, scale=1.5).to(dtype), layout),
         "z": with_layout(rnd(B, D, L).to(dtype), layout) if z else None, "bias": rnd(D) + 1.0 if bias else None,
         "init": rnd(nstates, D) if nstates else None, "dout": with_layout(rnd(B, D, L).to(dtype), layout),
         "dfinal": rnd(nstates, D) if nstates else None}
    return t


def _packing(seed, B, L, nseq, pad=True):
    """Row-unique ids in runs of random lengths, some padding between and after them."""
    r = np.random.default_rng(seed)
    ids = np.full((B, L), -1, np.int32)
    for b in range(B):
        cuts = np.sort(r.integers(0, L + 1, nseq - 1))
        edges = [0, *cuts.tolist(), L]
        for k in range(nseq):
            lo, hi = edges[k], edges[k + 1]
            if pad and hi - lo > 4 and r.random() < 0.4:
                hi -= int(r.integers(1, hi - lo - 1))
            ids[b, lo:hi] = b * nseq + k
    return ids


def _run_and_check(t, ids=None, states=True):
    """Forward and backward through autograd, every output and gradient against fp64."""
    leaves = {}
    for k in ("x", "gate", "z", "bias", "init"):
        if t[k] is not None:
            leaves[k] = t[k].detach().requires_grad_()
    seq = None if ids is None else torch.from_numpy(ids).cuda()
    kept = states and t["init"] is not None
    got = gated_recurrence_fn(leaves["x"], leaves["gate"], leaves.get("z"), leaves.get("bias"), seq_idx=seq,
                              initial_states=leaves.get("init"), return_final_states=kept)
    out, final = got if kept else (got, None)
    outs, grads = ([out, final], [t["dout"], t["dfinal"]]) if kept else ([out], [t["dout"]])
    found = dict(zip(leaves, torch.autograd.grad(outs, list(leaves.values()), grads)))
    w = {k: R.wide(v) for k, v in t.items()}
    eo, ef, _, _ = R.recurrence(w["x"], w["gate"], w["z"], w["bias"], ids, w["init"])
    R.check(out, eo, "out")
    assert out.dtype == t["x"].dtype and out.stride() == torch.empty_like(t["x"]).stride()
    if kept:
        assert final.dtype == torch.float32
        R.check(final, ef, "final_states")
    e = R.recurrence_grads(w["x"], w["gate"], w["z"], w["bias"], ids, w["init"], w["dout"], w["dfinal"] if kept else None)
    for k, g in found.items():
        R.check(g, e["d" + k], "d" + k, e["bias_scale"] if k == "bias" else None)
    with torch.no_grad():
        plain = gated_recurrence_fn(t["x"], t["gate"], t["z"], t["bias"], seq_idx=seq, initial_states=t["init"])
    assert torch.equal(plain, out)
    return out, final, found


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("L", [1, 2, 7, 8, 9, 63, 64, 65, 130, 513])
def test_lengths(L, dtype, layout):
    _run_and_check(_inputs(L, 2, 70, L, dtype, layout, nstates=2))


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [1, 2, 3, 8, 31, 32, 33, 64, 65, 128, 200])
def test_channels(D, dtype, layout):
    _run_and_check(_inputs(D, 3, D, 97, dtype, layout, nstates=3))


@pytest.mark.parametrize("z,bias,states", [(False, False, False), (True, False, False), (False, True, True), (True, True, False)])
@pytest.mark.parametrize("layout", ["channel_last", "contiguous"])
@pytest.mark.parametrize("dtype", DTYPES)
def test_optional_inputs(dtype, layout, z, bias, states):
    _run_and_check(_inputs(5, 2, 96, 300, dtype, layout, z, bias, 2 if states else None))


@pytest.mark.parametrize("B,D,L", [(1, 64, 5000), (1, 1030, 1999), (5, 257, 640), (1, 16, 20000), (16, 40, 300), (1, 2048, 1024)])
@pytest.mark.parametrize("layout", ["channel_last", "contiguous"])
def test_larger(B, D, L, layout):
    dtype = DTYPES[(B + D) % 3]
    _run_and_check(_inputs(B + L, B, D, L, dtype, layout, nstates=B))


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,D,L,nseq,states", [(1, 70, 300, 6, True), (2, 33, 131, 40, True), (1, 128, 1500, 3, False), (3, 65, 64, 2, True)])
def test_packed(B, D, L, nseq, states, dtype, layout):
    ids = _packing(L + nseq, B, L, nseq)
    _run_and_check(_inputs(nseq, B, D, L, dtype, layout, nstates=B * nseq if states else None), ids)


@pytest.mark.parametrize("inner,width", [(96, 96), (96, 104), (94, 98), (95, 103), (37, 41), (130, 133)])
@pytest.mark.parametrize("rows", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
def test_strips_that_start_anywhere(dtype, rows, inner, width):
    """Tensors within wider ones that are NaN around them, each with its own offset and pitch."""
    D, L = (70, inner) if rows else (inner, 75)
    for packed in (False, True):
        t = _inputs(width, 2, D, L, dtype, "contiguous", nstates=6 if packed else 2)
        for i, k in enumerate(("x", "gate", "z", "dout")):
            v = t[k] if rows else t[k].transpose(1, 2)
            pitch, off = width + i % 2 * 2, min(i, width - inner)
            wide = torch.full((*v.shape[:2], pitch), float("nan"), device="cuda", dtype=dtype)
            wide[:, :, off:off + inner] = v
            v = wide[:, :, off:off + inner]
            t[k] = v if rows else v.transpose(1, 2)
        _run_and_check(t, _packing(inner, 2, L, 3) if packed else None)


@pytest.mark.parametrize("layout", ["channel_last", "contiguous"])
def test_padding_is_not_read(layout):
    """Whatever padding holds, NaN and infinities included, nothing depends on it; a batch row
    that is padding throughout gives zeros and leaves its sequences' states alone."""
    B, D, L, nseq = 3, 72, 200, 5
    ids = _packing(3, B, L, nseq)
    ids[1] = -1
    ids[0, :9], ids[2, 100:170] = -7, -1
    t = _inputs(4, B, D, L, torch.bfloat16, layout, nstates=B * nseq)
    want = _run_and_check(t, ids)
    hole = torch.from_numpy(ids < 0).cuda()[:, None, :]
    for k, bad in (("x", float("nan")), ("gate", float("inf")), ("z", float("nan")), ("dout", float("-inf"))):
        t[k].masked_fill_(hole, bad)
    leaves = {k: t[k].detach().requires_grad_() for k in ("x", "gate", "z", "bias", "init")}
    out, final = gated_recurrence_fn(leaves["x"], leaves["gate"], leaves["z"], leaves["bias"], seq_idx=torch.from_numpy(ids).cuda(),
                                     initial_states=leaves["init"], return_final_states=True)
    found = torch.autograd.grad([out, final], list(leaves.values()), [t["dout"], t["dfinal"]])
    assert torch.equal(out, want[0]) and torch.equal(final, want[1])
    for k, g in zip(leaves, found):
        assert torch.equal(g, want[2][k]), k
    assert not out[1].any() and torch.equal(final[nseq:2 * nseq], t["init"][nseq:2 * nseq])
    assert torch.equal(found[4][nseq:2 * nseq], t["dfinal"][nseq:2 * nseq])


@pytest.mark.parametrize("layout", ["channel_last", "contiguous"])
def test_a_sequence_with_nan_leaves_the_others_alone(layout):
    D, L = 64, 300
    ids = np.zeros((1, L), np.int32)
    ids[0, 100:201], ids[0, 201:] = 1, 2
    t = _inputs(6, 1, D, L, torch.float32, layout, nstates=3)
    want = _run_and_check(t, ids)
    t["x"][:, :, 150] = float("nan")
    t["init"][1] = float("inf")
    leaves = {k: t[k].detach().requires_grad_() for k in ("x", "gate", "z", "init")}
    out, final = gated_recurrence_fn(leaves["x"], leaves["gate"], leaves["z"], t["bias"], seq_idx=torch.from_numpy(ids).cuda(),
                                     initial_states=leaves["init"], return_final_states=True)
    found = torch.autograd.grad([out, final], list(leaves.values()), [t["dout"], t["dfinal"]])
    sane = torch.from_numpy(ids[0] != 1).cuda()
    assert torch.isnan(out[0, :, 150:201]).all()
    assert torch.equal(out[:, :, sane], want[0][:, :, sane])
    assert torch.equal(final[[0, 2]], want[1][[0, 2]])
    for i, k in enumerate(("x", "gate", "z")):
        assert torch.equal(found[i][:, :, sane], want[2][k][:, :, sane]), k
    assert torch.equal(found[3][[0, 2]], want[2]["init"][[0, 2]])


def test_nan_travels_within_its_sequence():
    t = _inputs(7, 2, 40, 150, torch.float32, "channel_last", nstates=2)
    for name in ("x", "gate", "z"):
        u = {k: v.clone() for k, v in t.items()}
        u[name][1, 3, 50] = float("nan")
        out, final = gated_recurrence_fn(u["x"], u["gate"], u["z"], u["bias"], initial_states=u["init"], return_final_states=True)
        bad = torch.isnan(out)
        if name == "z":
            assert bad.sum() == 1 and bad[1, 3, 50]
        else:
            assert bad[1, 3, 50:].all() and bad.sum() == 100 and torch.isnan(final).sum() == 1


@pytest.mark.parametrize("layout", ["channel_last", "contiguous"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("name", ["x", "gate", "z", "dout"])
def test_nan_does_not_travel_against_time(name, dtype, layout):
    """A NaN reaches what depends on it and nothing else: not the positions beside it, other
    channels, or a packed neighbour."""
    D, L, at, ch = 70, 100, 45, 9
    ids = np.zeros((1, L), np.int32)
    ids[0, 40:60], ids[0, 60:] = 1, 2
    t = _inputs(23, 1, D, L, dtype, layout, nstates=3)

    def run(v):
        leaves = [v[k].detach().requires_grad_() for k in ("x", "gate", "z")]
        out = gated_recurrence_fn(*leaves, v["bias"], seq_idx=torch.from_numpy(ids).cuda(), initial_states=v["init"])
        return [out, *torch.autograd.grad(out, leaves, v["dout"])]

    want = run(t)
    t[name][0, ch, at] = float("nan")
    got = run(t)
    # places of its own sequence, from it on (out) or up to it (what flows back), or all
    own, before, after, here = (np.zeros(L, bool) for _ in range(4))
    own[40:60], before[40:at + 1], after[at:60], here[at] = True, True, True, True
    reach = {"x": (after, own, own, after), "gate": (after, own, own, after), "z": (here, before, before, here),
             "dout": (here & False, before, before, here)}[name]
    for what, g, w, may in zip(("out", "dx", "dgate", "dz"), got, want, reach):
        same = torch.ones(1, D, L, dtype=torch.bool, device="cuda")
        same[0, ch, torch.from_numpy(may).cuda()] = False
        assert torch.equal(g[same], w[same]), what
    if name != "dout":
        assert torch.isnan(got[0][0, ch, at])


@pytest.mark.parametrize("dtype", DTYPES)
def test_extreme_gates(dtype):
    """Gates that hold on for ever and that let go at once, beyond exp's range."""
    B, D, L = 1, 64, 200
    t = _inputs(8, B, D, L, dtype, "channel_last", nstates=1)
    values = torch.tensor([-1e4, -200.0, -90.0, -30.0, 0.0, 30.0, 90.0, 200.0, 1e4], device="cuda")
    pick = torch.randint(0, 9, (B, D, L), generator=_gen(1), device="cuda")
    t["gate"].copy_(values[pick].to(dtype))
    t["bias"] = None
    t["z"].mul_(40.0)
    with np.errstate(over="ignore"):
        _run_and_check(t)


def test_ids_outside_the_states():
    """An id with no row in the states starts from zero and is stored nowhere."""
    D, L = 48, 90
    ids = np.repeat(np.array([[0, 5, 1]], np.int32), 30, axis=1)
    t = _inputs(9, 1, D, L, torch.float32, "channel_last", nstates=2)
    _run_and_check(t, ids)


def test_final_states_without_initial_states():
    ids = _packing(1, 1, 200, 4)
    t = _inputs(10, 1, 50, 200, torch.float16, "channel_last")
    out, final = gated_recurrence_fn(t["x"], t["gate"], t["z"], t["bias"], seq_idx=torch.from_numpy(ids).cuda(),
                                     return_final_states=True, num_sequences=6)
    w = {k: R.wide(v) for k, v in t.items()}
    eo, ef, _, _ = R.recurrence(w["x"], w["gate"], w["z"], w["bias"], ids, None, nstates=6)
    R.check(out, eo, "out")
    R.check(final, ef, "final_states")
    assert not final[4:].any()


def test_empty_problems():
    for shape in ((0, 8, 5), (2, 0, 5), (2, 8, 0)):
        x = torch.empty(shape, device="cuda", requires_grad=True)
        init = torch.randn(shape[0], shape[1], device="cuda", requires_grad=True)
        bias = torch.zeros(shape[1], device="cuda", requires_grad=True)
        out, final = gated_recurrence_fn(x, x, x, bias, initial_states=init, return_final_states=True)
        assert out.shape == x.shape and torch.equal(final, init)
        gx, gi, gb = torch.autograd.grad([out, final], [x, init, bias], [torch.zeros_like(out), torch.ones_like(final)])
        assert gx.shape == x.shape and torch.equal(gi, torch.ones_like(gi)) and not gb.any()


def test_gradients_of_one_output_only():
    t = _inputs(11, 2, 64, 100, torch.float32, "channel_last", nstates=2)
    w = {k: R.wide(v) for k, v in t.items()}
    for part in ("out", "final"):
        x, init = t["x"].detach().requires_grad_(), t["init"].detach().requires_grad_()
        out, final = gated_recurrence_fn(x, t["gate"], t["z"], t["bias"], initial_states=init, return_final_states=True)
        if part == "out":
            gx, gi = torch.autograd.grad(out, [x, init], t["dout"])
        else:
            gx, gi = torch.autograd.grad(final, [x, init], t["dfinal"])
        e = R.recurrence_grads(w["x"], w["gate"], w["z"], w["bias"], None, w["init"],
                               w["dout"] if part == "out" else np.zeros_like(w["dout"]), w["dfinal"] if part == "final" else None)
        R.check(gx, e["dx"], part + " dx")
        R.check(gi, e["dinit"], part + " dinit")


def test_mixed_layouts_strides_and_broadcast_inputs():
    B, D, L = 2, 66, 130
    g = _gen(12)
    x = torch.randn(B, L, D, generator=g, device="cuda").transpose(1, 2).requires_grad_()
    gate = torch.randn(B, D, L, generator=g, device="cuda").requires_grad_()
    shared = torch.randn(1, D, 1, generator=g, device="cuda").requires_grad_()  # one z for all places
    odd = torch.randn(B, D, 2 * L + 1, generator=g, device="cuda")[:, :, 1::2]
    out = gated_recurrence_fn(x, gate + 0.0 * odd, shared.expand(B, D, L))
    dout = torch.randn(B, D, L, generator=g, device="cuda")
    gx, gg, gz = torch.autograd.grad(out, [x, gate, shared], dout)
    w = [R.wide(v) for v in (x, gate, shared.expand(B, D, L), dout)]
    e = R.recurrence_grads(w[0], w[1], w[2], None, None, None, w[3], None)
    R.check(out, R.recurrence(w[0], w[1], w[2])[0], "out")
    R.check(gx, e["dx"], "dx")
    R.check(gg, e["dgate"], "dgate")
    full = e["dz"].sum((0, 2))[None, :, None]
    R.check(gz, full, "dz", np.abs(e["dz"]).sum((0, 2)).max())
    strided = gated_recurrence_fn(odd, odd, odd)
    w = R.wide(odd)
    R.check(strided, R.recurrence(w, w, w)[0], "strided out")
    unaligned = torch.randn(B, L, D + 1, generator=g, device="cuda").to(torch.bfloat16)[:, :, 1:].transpose(1, 2)
    w = R.wide(unaligned)
    R.check(gated_recurrence_fn(unaligned, unaligned, unaligned), R.recurrence(w, w, w)[0], "unaligned out")


def test_against_differences():
    """Directional differences of the fp32 kernel itself: with a step of 2^-6 the truncation is
    of order 2^-12 / 6 times third derivatives of order one and the rounding of order
    2^-24 sqrt(n) / 2^-6; 2e-3 of the sum's natural size covers both."""
    t = _inputs(13, 2, 32, 80, torch.float32, "channel_last", nstates=2)
    names = ("x", "gate", "z", "bias", "init")
    leaves = {k: t[k].detach().requires_grad_() for k in names}

    def loss(v):
        out, final = gated_recurrence_fn(v["x"], v["gate"], v["z"], v["bias"], initial_states=v["init"], return_final_states=True)
        return (out.double() * t["dout"].double()).sum() + (final.double() * t["dfinal"].double()).sum()

    grads = dict(zip(names, torch.autograd.grad(loss(leaves), list(leaves.values()))))
    g = _gen(14)
    for k in names:
        d = torch.randn(t[k].shape, generator=g, device="cuda")
        up, down = dict(t), dict(t)
        up[k], down[k] = t[k] + d * 2.0 ** -6, t[k] - d * 2.0 ** -6
        want = ((loss(up) - loss(down)) * 2.0 ** 5).item()
        got = (grads[k].double() * d.double()).sum().item()
        size = grads[k].double().norm().item()
        assert abs(got - want) <= 2e-3 * size * 4, (k, got, want, size)


@pytest.mark.parametrize("layout", ["channel_last", "contiguous"])
def test_results_repeat_bit_for_bit(layout):
    t = _inputs(15, 3, 300, 700, torch.bfloat16, layout, nstates=3)

    def once():
        leaves = [t[k].detach().requires_grad_() for k in ("x", "gate", "z", "bias", "init")]
        out, final = gated_recurrence_fn(*leaves[:4], initial_states=leaves[4], return_final_states=True)
        return [out, final, *torch.autograd.grad([out, final], leaves, [t["dout"], t["dfinal"]])]

    first = once()
    for _ in range(20):
        for a, b in zip(first, once()):
            assert torch.equal(a, b)


def test_other_stream_and_graph():
    t = _inputs(16, 2, 128, 500, torch.bfloat16, "channel_last", nstates=2)
    want = gated_recurrence_fn(t["x"], t["gate"], t["z"], t["bias"], initial_states=t["init"])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = gated_recurrence_fn(t["x"], t["gate"], t["z"], t["bias"], initial_states=t["init"])
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, _, ck = gated_recurrence_fwd_function(t["x"], t["gate"], t["z"], t["bias"], None, t["init"], False, None, True)
        grads = gated_recurrence_bwd_function(t["x"], t["gate"], t["z"], t["bias"], None, t["init"], ck, t["dout"], None, True, True)
    t["x"].mul_(0.5)
    graph.replay()
    torch.cuda.synchronize()
    w = {k: R.wide(v) for k, v in t.items()}
    e = R.recurrence_grads(w["x"], w["gate"], w["z"], w["bias"], None, w["init"], w["dout"], None)
    R.check(out, R.recurrence(w["x"], w["gate"], w["z"], w["bias"], None, w["init"])[0], "out")
    for k, g in zip(("dx", "dgate", "dz", "dbias", "dinit"), grads):
        R.check(g, e[k], k, e["bias_scale"] if k == "dbias" else None)


@pytest.mark.parametrize("layout", ["channel_last", "contiguous"])
def test_offsets_past_32_bits(layout):
    """More than 2^31 elements in x: the last places of a long sequence are what the state
    before them gives."""
    B, D, L = 1, 72, 30_000_128
    g = _gen(17)
    x = torch.randn(B, L, D, generator=g, device="cuda", dtype=torch.bfloat16)
    x = x.transpose(1, 2) if layout == "channel_last" else x.view(B, D, L)
    cut = L - 777
    whole, final = gated_recurrence_fn(x, x, return_final_states=True)
    _, mid = gated_recurrence_fn(x[:, :, :cut], x[:, :, :cut], return_final_states=True)
    tail = R.wide(x[:, :, cut:])
    eo, ef, _, _ = R.recurrence(tail, tail, None, None, None, R.wide(mid))
    R.check(whole[:, :, cut:], eo, "tail")
    R.check(final, ef, "final")


def test_type_refusals():
    x = torch.randn(2, 8, 16, device="cuda")
    with pytest.raises(TypeError, match="gate"):
        gated_recurrence_fn(x, x.half())
    with pytest.raises(TypeError, match="dtype"):
        gated_recurrence_fn(x.double(), x.double())
    with pytest.raises(TypeError, match="initial_states"):
        gated_recurrence_fn(x, x, initial_states=torch.zeros(2, 8, device="cuda", dtype=torch.bfloat16))
    with pytest.raises(TypeError, match="seq_idx"):
        gated_recurrence_fn(x, x, seq_idx=torch.zeros(2, 16, device="cuda", dtype=torch.int64))
    with pytest.raises(TypeError, match="state"):
        gated_recurrence_update(x[:, :, 0], torch.zeros(2, 8, device="cuda", dtype=torch.float16), x[:, :, 0])
    with pytest.raises(ValueError, match="one device|CUDA"):
        gated_recurrence_fn(x, x.cpu())


# ------------------------------------------------------------------------- update
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,D,T", [(1, 1, 1), (1, 64, 1), (3, 100, 1), (37, 1000, 3), (128, 513, 1), (2, 4096, 7), (300, 8, 2)])
@pytest.mark.parametrize("z,pool", [(True, False), (False, True), (True, True)])
def test_update(B, D, T, z, pool, dtype):
    g = _gen(B + D + T)
    rows = B + 5 if pool else B
    state = torch.randn(rows, D, generator=g, device="cuda")
    x, gate, zz = (torch.randn(B, D, T, generator=g, device="cuda").to(dtype) for _ in range(3))
    if T == 1:
        x, gate, zz = x[..., 0], gate[..., 0], zz[..., 0]
    bias = torch.randn(D, generator=g, device="cuda").to(dtype)
    index = torch.randperm(rows, generator=g, device="cuda")[:B].to(torch.int32) if pool else None
    if pool and B > 2:
        index[1], index[2] = -1, rows  # padding, either side
    before = state.clone()
    out = gated_recurrence_update(x, state, gate, zz if z else None, bias, index)
    assert out.shape == x.shape and out.dtype == dtype
    idx = index.cpu().numpy() if pool else np.arange(B)
    w = [R.wide(v.view(B, D, T)) for v in (x, gate, zz)]
    live = (idx >= 0) & (idx < rows)
    init = R.wide(before)[np.where(live, idx, 0)]
    eo, ef, _, _ = R.recurrence(w[0], w[1], w[2] if z else None, R.wide(bias), None, init)
    R.check(out.reshape(B, D, T), np.where(live[:, None, None], eo, 0.0), "out")
    es = R.wide(before)
    es[idx[live]] = ef[live]
    R.check(state, es, "state")
    untouched = np.setdiff1d(np.arange(rows), idx[live])
    assert torch.equal(state[untouched], before[untouched])


def test_update_layouts_and_wide_index():
    B, D, T = 6, 96, 2
    g = _gen(5)
    wide = torch.randn(B, T, 3 * D + 1, generator=g, device="cuda").to(torch.bfloat16)
    x, gate, z = (wide[:, :, 1 + i * D:1 + (i + 1) * D].transpose(1, 2) for i in range(3))
    pool = torch.randn(D, 9, generator=g, device="cuda").t()  # (9, D), channel stride 9
    before = R.wide(pool)
    index = torch.tensor([4, 0, 8, 2, 3, 1], device="cuda")  # int64 is converted
    out = gated_recurrence_update(x, pool, gate, z, None, index)
    w = [R.wide(v) for v in (x, gate, z)]
    idx = index.cpu().numpy()
    eo, ef, _, _ = R.recurrence(w[0], w[1], w[2], None, None, before[idx])
    R.check(out, eo, "out")
    before[idx] = ef
    R.check(pool, before, "state")


def test_prefill_then_decode_equals_one_pass():
    B, D, L, n = 3, 160, 61, 9
    t = _inputs(20, B, D, L + n, torch.float32, "channel_last", nstates=B)
    whole, last = gated_recurrence_fn(t["x"], t["gate"], t["z"], t["bias"], initial_states=t["init"], return_final_states=True)
    out, state = gated_recurrence_fn(t["x"][:, :, :L], t["gate"][:, :, :L], t["z"][:, :, :L], t["bias"],
                                     initial_states=t["init"], return_final_states=True)
    steps = [gated_recurrence_update(t["x"][:, :, L + i], state, t["gate"][:, :, L + i], t["z"][:, :, L + i], t["bias"])
             for i in range(n)]
    R.check(torch.cat([out, torch.stack(steps, -1)], -1), R.wide(whole), "out")
    R.check(state, R.wide(last), "state")
