"""Host-side checks of the selective recurrence and of beam search: their formulas against
differences, the PyTorch statements against the 64-bit ones, refusals, and the C ABI's layout."""

import ctypes
import itertools
import math
import os
import subprocess

import numpy as np
import pytest
import torch

import selective_ref as S
from causal_conv1d import (_abi, beam_search_reorder, beam_search_select, selective_recurrence_fn,
                           selective_recurrence_update)
from causal_conv1d.beam_search import beam_search_reorder_ref, beam_search_select_ref
from causal_conv1d.selective_recurrence import selective_recurrence_ref

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
IDS = np.array([[0, 0, 0, 2, 2, -1, -1, 3, 3], [-1, 4, 4, 4, -1, 5, 6, 6, -1]])
GRADS = ("x", "delta", "A", "B", "C", "D", "z", "bias", "init")


def _random(seed, *shape):
    return np.random.default_rng(seed).standard_normal(shape)


def _values(packed, groups):
    batch, dim, L, N = 2, 4, 9, 3
    n = 8 if packed else batch
    coeff = (batch, groups, N, L) if groups else (batch, N, L)
    shapes = {"x": (batch, dim, L), "delta": (batch, dim, L), "B": coeff, "C": coeff, "D": (dim,), "z": (batch, dim, L),
              "bias": (dim,), "init": (n, dim, N), "dout": (batch, dim, L), "dfinal": (n, dim, N)}
    v = {k: _random(i, *s) for i, (k, s) in enumerate(shapes.items())}
    v["A"] = -np.exp(_random(50, dim, N))
    return v, (IDS if packed else None)


@pytest.mark.parametrize("softplus", [True, False])
@pytest.mark.parametrize("packed,groups", [(False, 0), (True, 0), (True, 2), (False, 4)])
def test_gradients_against_differences(packed, groups, softplus):
    v, ids = _values(packed, groups)

    def loss(w):
        w = {k: t for k, t in w.items() if k not in ("dout", "dfinal")}
        e = S.statement(w, ids, use_softplus=softplus)
        return (e["out"][0] * v["dout"]).sum() + (e["final"][0] * v["dfinal"]).sum()

    g = S.statement(v, ids, use_softplus=softplus)
    # truncation of order step^2; rounding: each of the sum's terms is off by some 2^-53 of itself (nine
    # steps of a few operations: 2^-47), and without softplus negative steps make the terms grow
    step = 1e-6
    terms = np.abs(g["out"][0] * v["dout"]).sum() + np.abs(g["final"][0] * v["dfinal"]).sum()
    rounding = 2.0 ** -47 * terms / step
    for name in GRADS:
        d = _random(11, *v[name].shape)
        up, down = dict(v), dict(v)
        up[name], down[name] = v[name] + step * d, v[name] - step * d
        want = (loss(up) - loss(down)) / (2 * step)
        assert abs((g["d" + name][0] * d).sum() - want) < 1e-6 * max(1.0, abs(want)) + rounding, name


@pytest.mark.parametrize("softplus", [True, False])
@pytest.mark.parametrize("packed,groups", [(False, 0), (True, 2)])
def test_statement_matches(packed, groups, softplus):
    v, ids = _values(packed, groups)
    t = {k: torch.tensor(v[k], requires_grad=True) for k in GRADS}
    seq = None if ids is None else torch.tensor(ids, dtype=torch.int32)
    out, final = selective_recurrence_ref(*[t[k] for k in ("x", "delta", "A", "B", "C", "D", "z", "bias")], softplus, seq,
                                          t["init"], True)
    e = S.statement(v, ids, use_softplus=softplus)
    np.testing.assert_allclose(S.wide(out), e["out"][0], atol=1e-12)
    np.testing.assert_allclose(S.wide(final), e["final"][0], atol=1e-12)
    ((out * torch.tensor(v["dout"])).sum() + (final * torch.tensor(v["dfinal"])).sum()).backward()
    for k in t:
        np.testing.assert_allclose(t[k].grad.numpy(), e["d" + k][0], atol=1e-12, err_msg=k)


def test_bounds_hold_for_fp32():
    """The statement in fp32 stays within the bounds that the kernels are held to."""
    v, ids = _values(True, 2)
    t = {k: torch.tensor(x, dtype=torch.float32).requires_grad_(k in GRADS) for k, x in v.items()}
    rounded = {k: S.wide(x) for k, x in t.items()}
    out, final = selective_recurrence_ref(*[t[k] for k in ("x", "delta", "A", "B", "C", "D", "z", "bias")], True,
                                          torch.tensor(ids, dtype=torch.int32), t["init"], True)
    e = S.statement(rounded, ids)
    S.check(out, e["out"], "out")
    S.check(final, e["final"], "final")
    for k, g in zip(GRADS, torch.autograd.grad([out, final], [t[k] for k in GRADS], [t["dout"], t["dfinal"]])):
        S.check(g, e["d" + k], "d" + k)


def _brute_force(logits, scores, finished, end, n):
    best = []
    for b in range(logits.shape[0]):
        every = []
        for k in range(logits.shape[1]):
            row = [float(x) for x in logits[b, k]]
            score = float(scores[b, k])
            ended = finished is not None and bool(finished[b, k])
            top = max(row)
            sound = math.isfinite(score) and (ended or (not any(math.isnan(x) for x in row) and math.isfinite(top)))
            lse = top + math.log(sum(math.exp(x - top) for x in row)) if sound and not ended else 0.0
            for w, x in enumerate(row):
                logp = (0.0 if w == end else -math.inf) if ended else x - lse
                every.append((score + logp if sound else -math.inf, k, w))
        every.sort(key=lambda e: (-e[0], e[1], e[2]))
        best.append(every[:n])
    return best


def test_select_statement_matches_definition():
    r = np.random.default_rng(0)
    logits = torch.tensor(r.integers(-3, 4, (6, 3, 8)).astype(np.float32))
    scores = torch.tensor(r.integers(-2, 1, (6, 3)).astype(np.float32))
    logits[1, 1] = -math.inf
    logits[2, 0, 3] = math.nan
    logits[3, 2, 1] = math.inf
    logits[4, :, 2:] = -math.inf
    scores[5, 0], scores[5, 1], scores[0, 2] = -math.inf, math.nan, math.inf
    finished = torch.tensor(r.random((6, 3)) < 0.3)
    for flags, n in itertools.product((None, finished), (1, 5, 24)):
        got = beam_search_select_ref(logits, scores, flags, 2, n)
        want = _brute_force(logits, scores, flags, 2, n)
        for b, row in enumerate(want):
            assert [(k, w) for _, k, w in row] == list(zip(got[1][b].tolist(), got[2][b].tolist())), b
            np.testing.assert_allclose(got[0][b].numpy(), [t for t, _, _ in row], rtol=1e-6)


def test_reorder_statement_matches_definition():
    t = torch.arange(24.0).view(6, 4)
    got = beam_search_reorder_ref(t, torch.tensor([[2, 0, 0], [1, 5, -1]]))
    assert got[:, 0].tolist() == [8.0, 0.0, 0.0, 16.0, 16.0, 20.0]
    pool = beam_search_reorder_ref(t, torch.tensor([[1, 0, 0]]), torch.tensor([4, 2, -1]))
    assert pool[:, 0].tolist() == [0.0, 4.0, 16.0, 12.0, 8.0, 20.0]


# ------------------------------------------------------------------------ refusals
def test_refusals():
    x, A, bc = torch.empty(2, 8, 16), torch.empty(8, 4), torch.empty(2, 4, 16)
    fn = selective_recurrence_fn
    with pytest.raises(ValueError, match="CUDA"):
        fn(x, x, A, bc, bc)
    with pytest.raises(ValueError, match="3 dimensions"):
        fn(x[0], x[0], A, bc, bc)
    with pytest.raises(ValueError, match="delta"):
        fn(x, x[:, :, :15], A, bc, bc)
    with pytest.raises(ValueError, match="A"):
        fn(x, x, torch.empty(7, 4), bc, bc)
    with pytest.raises(ValueError, match="A"):
        fn(x, x, torch.empty(8), bc, bc)
    with pytest.raises(ValueError, match="B"):
        fn(x, x, A, bc[:, :3], bc)
    with pytest.raises(ValueError, match="C"):
        fn(x, x, A, bc, bc[:1])
    with pytest.raises(ValueError, match="groups"):
        fn(x, x, A, torch.empty(2, 3, 4, 16), torch.empty(2, 3, 4, 16))
    with pytest.raises(ValueError, match="groups"):
        fn(x, x, A, torch.empty(2, 0, 4, 16), torch.empty(2, 0, 4, 16))
    with pytest.raises(ValueError, match="C"):
        fn(x, x, A, torch.empty(2, 2, 4, 16), torch.empty(2, 4, 4, 16))
    with pytest.raises(ValueError, match="B must have 3 dimensions"):
        fn(x, x, A, torch.empty(4, 16), bc)
    with pytest.raises(ValueError, match="D"):
        fn(x, x, A, bc, bc, torch.empty(7))
    with pytest.raises(ValueError, match="z"):
        fn(x, x, A, bc, bc, z=x[:1])
    with pytest.raises(ValueError, match="delta_bias"):
        fn(x, x, A, bc, bc, delta_bias=torch.empty(9))
    with pytest.raises(ValueError, match="seq_idx"):
        fn(x, x, A, bc, bc, seq_idx=torch.zeros(2, 15, dtype=torch.int32))
    with pytest.raises(ValueError, match="initial_states"):
        fn(x, x, A, bc, bc, initial_states=torch.empty(3, 8, 4))
    with pytest.raises(ValueError, match="initial_states"):
        fn(x, x, A, bc, bc, seq_idx=torch.zeros(2, 16, dtype=torch.int32), initial_states=torch.empty(3, 8, 5))
    with pytest.raises(ValueError, match="num_sequences"):
        fn(x, x, A, bc, bc, seq_idx=torch.zeros(2, 16, dtype=torch.int32), return_final_states=True)


def test_update_refusals():
    x, A, bc, state = torch.empty(2, 8), torch.empty(8, 4), torch.empty(2, 4), torch.empty(2, 8, 4)
    fn = selective_recurrence_update
    with pytest.raises(ValueError, match="CUDA"):
        fn(x, state, x, A, bc, bc)
    with pytest.raises(ValueError, match="state"):
        fn(x, torch.empty(3, 8, 4), x, A, bc, bc)
    with pytest.raises(ValueError, match="state"):
        fn(x, torch.empty(2, 8, 5), x, A, bc, bc)
    with pytest.raises(ValueError, match="state_indices"):
        fn(x, state, x, A, bc, bc, state_indices=torch.zeros(3, dtype=torch.int32))
    with pytest.raises(TypeError, match="state_indices"):
        fn(x, state, x, A, bc, bc, state_indices=torch.zeros(2))
    with pytest.raises(ValueError, match="delta"):
        fn(x, state, x[:1], A, bc, bc)
    with pytest.raises(ValueError, match="B must have 2 dimensions"):
        fn(x, state, x, A, torch.empty(4), bc)
    with pytest.raises(ValueError, match="B"):
        fn(x[..., None], state, x[..., None], A, bc[..., None].expand(2, 4, 3), bc[..., None])
    with pytest.raises(RuntimeError, match="no derivative"):
        fn(x, state.requires_grad_(), x, A, bc, bc)


def test_beam_refusals():
    logits, scores = torch.empty(2, 3, 5), torch.empty(2, 3)
    with pytest.raises(ValueError, match="CUDA"):
        beam_search_select(logits, scores)
    with pytest.raises(ValueError, match="3 dimensions"):
        beam_search_select(logits[0], scores)
    with pytest.raises(ValueError, match="scores"):
        beam_search_select(logits, scores[:1])
    with pytest.raises(ValueError, match="finished"):
        beam_search_select(logits, scores, torch.zeros(2, 2, dtype=torch.bool), 1)
    with pytest.raises(TypeError, match="bool"):
        beam_search_select(logits, scores, torch.zeros(2, 3), 1)
    with pytest.raises(ValueError, match="end_token"):
        beam_search_select(logits, scores, torch.zeros(2, 3, dtype=torch.bool))
    parents, state = torch.zeros(2, 3, dtype=torch.int64), torch.empty(6, 4)
    with pytest.raises(ValueError, match="CUDA"):
        beam_search_reorder(state, parents)
    with pytest.raises(ValueError, match="2 dimensions"):
        beam_search_reorder(state, parents[0])
    with pytest.raises(ValueError, match="6 rows"):
        beam_search_reorder([state, state[:5]], parents)
    with pytest.raises(ValueError, match="state_indices"):
        beam_search_reorder(state, parents, torch.zeros(5, dtype=torch.int32))
    with pytest.raises(ValueError, match="dimensions"):
        beam_search_reorder(torch.empty(6, 1, 1, 1, 1), parents)
    with pytest.raises(RuntimeError, match="no derivative"):
        beam_search_reorder(state.requires_grad_(), parents)


# ------------------------------------------------------------------------- the C ABI
def _tensor(ptr=16, dtype=0, strides=(0, 0, 0)):
    return (ptr, dtype, *strides)


_ORDER = ("x", "delta", "A", "B", "C", "D", "z", "bias", "seq_idx", "initial_states", "final_states", "out", "dout",
          "dfinal_states", "dx", "ddelta", "dB", "dC", "dz", "dinitial_states")


def _sel(**kw):
    words = [kw.get(k, d) for k, d in (("batch", 2), ("dim", 2), ("seqlen", 2), ("dstate", 3), ("groups", 1), ("nstates", 2), ("softplus", 1))]
    for k in _ORDER:
        words += kw.get(k, _abi._NONE)
    return _abi.SELECTIVE_PARAMS.pack(*words, 0, 0, 0, 0, 0, 0, 0, kw.get("checkpoints", 0), kw.get("workspace", 0), kw.get("bytes", 0))


def _refused(fn, params, status, text):
    lib = _abi.load_library()
    got = fn(params, None) if len(fn.argtypes) == 2 else fn(params)
    assert got == status
    assert text in lib.cc1d_last_error(), lib.cc1d_last_error()


def test_selective_abi_refusals_need_no_gpu():
    lib = _abi.load_library()
    fwd, bwd, upd = lib.cc1d_selective_fwd_launch, lib.cc1d_selective_bwd_launch, lib.cc1d_selective_update_launch
    t, half = _tensor(), _tensor(dtype=1)
    ins = {"x": t, "delta": t, "A": t, "B": t, "C": t}
    _refused(fwd, None, 1, b"NULL")
    _refused(fwd, _sel(batch=-1), 1, b"sizes")
    _refused(fwd, _sel(seqlen=1 << 31), 1, b"sizes")
    _refused(fwd, _sel(dim=1 << 30, nstates=1 << 30, dstate=16), 1, b"sizes")
    for n in (0, 257):
        _refused(fwd, _sel(dstate=n), 1, b"dstate")
    for g in (0, 3):
        _refused(fwd, _sel(groups=g), 1, b"groups")
    _refused(fwd, _sel(x=_tensor(dtype=3)), 2, b"x must be")
    for k in ("delta", "B", "C", "z", "out"):
        _refused(fwd, _sel(**{**ins, "out": t, k: half}), 2, k.encode())
    _refused(fwd, _sel(**{**ins, "A": _tensor(dtype=4)}), 2, b"A must be a float")
    _refused(fwd, _sel(**ins, out=t, D=_tensor(dtype=3)), 2, b"D must be")
    _refused(fwd, _sel(**ins, out=t, bias=_tensor(dtype=3)), 2, b"delta_bias")
    _refused(fwd, _sel(**ins, out=t, seq_idx=_tensor(dtype=4)), 2, b"seq_idx")
    _refused(fwd, _sel(**ins, out=t, initial_states=half), 2, b"initial_states")
    _refused(fwd, _sel(**ins, out=t, initial_states=t, nstates=3), 1, b"one state")
    for k in ins:
        _refused(fwd, _sel(**{**ins, "out": t, k: _abi._NONE}), 1, k.encode() + b" is required")
    _refused(fwd, _sel(**ins), 1, b"out is required")
    _refused(fwd, _sel(**ins, out=t, checkpoints=8), 1, b"aligned")
    grads = {k: t for k in ("dout", "dx", "ddelta", "dB", "dC")}
    _refused(bwd, _sel(**ins, **grads), 1, b"checkpoints")
    _refused(bwd, _sel(**ins, **grads, z=t, checkpoints=16), 1, b"dz is required")
    _refused(bwd, _sel(**ins, **grads, checkpoints=16), 1, b"workspace")
    _refused(bwd, _sel(**ins, **grads, checkpoints=16, workspace=24, bytes=1 << 40), 1, b"aligned")
    _refused(lib.cc1d_selective_bwd_workspace_bytes, _sel(**ins), -1, b"required")
    big = {"batch": 1, "dim": 1 << 20, "seqlen": (1 << 31) - 1, "dstate": 256, "nstates": 1}
    _refused(lib.cc1d_selective_bwd_workspace_bytes, _sel(**ins, **grads, **big, checkpoints=16), -1, b"large")
    assert lib.cc1d_selective_bwd_workspace_bytes(_sel(**ins, **grads, checkpoints=16)) > 0
    assert fwd(_sel(seqlen=0), None) == 0 and fwd(_sel(batch=0, nstates=0), None) == 0

    def update(sizes=(2, 2, 1, 3, 1, 2), **kw):
        words = [*sizes, 1]
        for k in (*_ORDER[:8], "state", "state_indices", "out"):
            words += kw.get(k, _abi._NONE)
        return _abi.SELECTIVE_UPDATE_PARAMS.pack(*words, 0, 0)

    _refused(upd, update(**ins, state=half, out=t), 2, b"state must be float32")
    _refused(upd, update(**ins, state=t, out=t, state_indices=_tensor(dtype=4)), 2, b"state_indices")
    _refused(upd, update(sizes=(2, 2, 1, 3, 1, 3), **ins, state=t, out=t), 1, b"one state")
    _refused(upd, update(**ins, out=t), 1, b"state is required")
    _refused(upd, update(sizes=(2, 2, 1, 300, 1, 2), **ins, state=t, out=t), 1, b"dstate")
    for strides in ((0, 3, 1), (6, 0, 1), (6, 3, 0), (6, 2, 1), (5, 3, 1), (1, 1, 1), (-6, 3, 1)):
        _refused(upd, update(**ins, state=_tensor(strides=strides), out=t), 1, b"overlap")
    assert upd(update(sizes=(0, 2, 1, 3, 1, 0)), None) == 0


def test_beam_abi_refusals_need_no_gpu():
    lib = _abi.load_library()
    fn = lib.cc1d_beam_select_launch
    logits, scores = _tensor(strides=(10, 5, 1)), _tensor()

    def select(sizes=(2, 2, 5, 2), end=0, logits=logits, scores=scores, finished=0, outs=(16, 16, 16), ws=(0, 0)):
        return _abi.BEAM_SELECT_PARAMS.pack(*sizes, end, *logits, *scores, finished, 2, 1, *outs, *ws)

    _refused(fn, None, 1, b"NULL")
    for sizes, what in (((-1, 2, 5, 2), b"sizes"), ((2, 0, 5, 2), b"beams"), ((2, 65, 5, 2), b"beams"), ((2, 2, 0, 1), b"vocab"),
                        ((2, 2, 5, 0), b"candidates"), ((2, 2, 5, 11), b"candidates"), ((2, 2, 500, 65), b"candidates")):
        _refused(fn, select(sizes), 1, what)
    _refused(fn, select(logits=_tensor(dtype=3)), 2, b"logits")
    _refused(fn, select(scores=_tensor(dtype=2)), 2, b"scores")
    for end in (-1, 5):
        _refused(fn, select(finished=16, end=end), 1, b"end_token")
    _refused(fn, select(logits=_tensor(strides=(10, 5, 2))), 1, b"unit stride")
    _refused(fn, select(outs=(16, 0, 16)), 1, b"required")
    _refused(fn, select(), 1, b"workspace")
    assert lib.cc1d_beam_select_workspace_bytes(select()) > 0
    assert fn(select((0, 2, 5, 2)), None) == 0

    fn = lib.cc1d_beam_reorder_launch

    def reorder(rows, sizes=(2, 3), parents=_tensor(dtype=4), index=_abi._NONE):
        packed = b"".join(_abi.BEAM_ROWS.pack(*r) for r in rows)
        keep = ctypes.create_string_buffer(packed)
        reorder.keep = keep
        return _abi.BEAM_REORDER_PARAMS.pack(*sizes, len(rows), *parents, *index, ctypes.addressof(keep) if rows else 0)

    good = (16, 6, 4, 4, 4, 1, 1, 1, 1, 1)
    _refused(fn, None, 1, b"NULL")
    _refused(fn, reorder([good], sizes=(2, 0)), 1, b"beams")
    _refused(fn, reorder([good], sizes=(2, 65)), 1, b"beams")
    _refused(fn, reorder([good], parents=_tensor(dtype=0)), 2, b"parents")
    _refused(fn, reorder([good], index=_tensor(dtype=4)), 2, b"state_indices")
    _refused(fn, reorder([good, (4096, *good[1:]), good]), 1, b"start at one place")
    _refused(fn, reorder([(16, 6, 4, 3, 4, 1, 1, 1, 1, 1)]), 1, b"element_bytes")
    _refused(fn, reorder([(16, 5, 4, 4, 4, 1, 1, 1, 1, 1)]), 1, b"one row")
    for bad in ((16, 6, 3, 4, 4, 1, 1, 1, 1, 1),     # a row reaches into the next one
                (16, 6, 0, 4, 4, 1, 1, 1, 1, 1),     # rows at one place
                (16, 6, 8, 4, 4, 2, 1, 0, 1, 1),     # elements at one place
                (16, 6, -4, 4, 4, 1, 1, 1, 1, 1)):
        _refused(fn, reorder([bad]), 1, b"overlap")
    assert fn(reorder([], sizes=(2, 3)), None) == 0 and fn(reorder([good], sizes=(0, 3)), None) == 0


C_PROBE = r"""
#include <stddef.h>
#include <stdio.h>
#include "causal_conv1d_b200.h"
int main(void) {
  printf("%zu %zu %zu %zu %zu %d %d %d %d %d\n", sizeof(cc1d_selective_params), sizeof(cc1d_selective_update_params),
         sizeof(cc1d_beam_select_params), sizeof(cc1d_beam_rows), sizeof(cc1d_beam_reorder_params), CC1D_SELECTIVE_CHUNK(4),
         CC1D_SELECTIVE_CHUNK(8), CC1D_SELECTIVE_CHUNK(9),
         CC1D_SELECTIVE_MAX_STATES, CC1D_BEAM_MAX);
  printf("%zu %zu %zu %zu\n", offsetof(cc1d_selective_params, x), offsetof(cc1d_selective_params, dA),
         offsetof(cc1d_selective_update_params, out), offsetof(cc1d_beam_select_params, out_scores));
  return 0;
}
"""


def test_params_layout(tmp_path):
    src, exe = tmp_path / "probe.c", tmp_path / "probe"
    src.write_text(C_PROBE)
    try:
        subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    except (OSError, subprocess.CalledProcessError):
        pytest.skip("gcc unavailable")
    got = [int(v) for v in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    assert got == [_abi.SELECTIVE_PARAMS.size, _abi.SELECTIVE_UPDATE_PARAMS.size, _abi.BEAM_SELECT_PARAMS.size,
                   _abi.BEAM_ROWS.size, _abi.BEAM_REORDER_PARAMS.size, *map(_abi.selective_chunk, (4, 8, 9)), 256, 64,
                   56, 56 + 20 * 40 + 32, 56 + 10 * 40, 40 + 80 + 24]


def test_torch_ops_registered_with_fake_shapes():
    from torch._subclasses.fake_tensor import FakeTensorMode

    ops = torch.ops.causal_conv1d
    with FakeTensorMode():
        x = torch.empty(2, 70, 64, dtype=torch.bfloat16).transpose(1, 2)
        A, D, init = torch.empty(64, 5), torch.empty(64), torch.empty(2, 64, 5)
        bc = torch.empty(2, 70, 5, dtype=torch.bfloat16).transpose(1, 2)
        out, final, ck = ops.selective_recurrence_fwd(x, x, A, bc, bc, D, x, D, True, None, init, True, 0, True)
        assert out.stride() == x.stride() and final.shape == (2, 64, 5) and ck.shape == (2, 5, 64, 8)
        g = ops.selective_recurrence_bwd(x, x, A, bc, bc, None, None, D, True, None, init, ck, x, final, True, True)
        assert g[0].stride() == x.stride() and g[3].shape == bc.shape and g[3].stride() == bc.stride()
        assert g[2].shape == A.shape and g[5].numel() == 0 and g[6].numel() == 0 and g[8].shape == init.shape
        g = ops.selective_recurrence_bwd(x, x, A, bc, bc, None, None, None, True, None, None, ck, x, None, True, True)
        assert g[7].shape == (64,) and g[7].dtype == torch.float32 and g[8].shape == init.shape
        assert ops.selective_recurrence_update(x[..., 0], init, x[..., 0], A, bc[..., 0], bc[..., 0], None, None, None, True, None).shape == (2, 64)
        s, p, t = ops.beam_search_select(torch.empty(3, 4, 9), torch.empty(3, 4), None, None, 6)
        assert s.shape == p.shape == t.shape == (3, 6) and p.dtype == torch.int64
        ops.beam_search_reorder([init], torch.empty(1, 2, dtype=torch.int64), None)
