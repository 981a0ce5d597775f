"""Host-side checks of the recurrent-block operators: their formulas against differences,
the PyTorch statements against the 64-bit ones, refusals, and the C ABI's layout."""

import ctypes
import os
import subprocess

import numpy as np
import pytest
import torch

import block_ref as R
from causal_conv1d import (_abi, dropout_add_rms_norm_fn, gated_recurrence_fn, gated_recurrence_update)
from causal_conv1d.add_norm import dropout_add_rms_norm_mask_ref, dropout_add_rms_norm_ref
from causal_conv1d.gated_recurrence import gated_recurrence_ref

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
IDS = np.array([[0, 0, 0, 2, 2, -1, -1, 3, 3], [-1, 4, 4, 4, -1, 5, 6, 6, -1]])


def _random(seed, *shape):
    return np.random.default_rng(seed).standard_normal(shape)


@pytest.mark.parametrize("packed", [False, True])
def test_recurrence_gradients_against_differences(packed):
    B, D, L = 2, 3, 9
    ids = IDS if packed else None
    n = 8 if packed else B
    v = {"x": _random(1, B, D, L), "gate": _random(2, B, D, L), "z": _random(3, B, D, L), "bias": _random(4, D),
         "init": _random(5, n, D)}
    dout, dfinal = _random(6, B, D, L), _random(7, n, D)

    def loss(w):
        out, final, _, _ = R.recurrence(w["x"], w["gate"], w["z"], w["bias"], ids, w["init"])
        return (out * dout).sum() + (final * dfinal).sum()

    g = R.recurrence_grads(v["x"], v["gate"], v["z"], v["bias"], ids, v["init"], dout, dfinal)
    step = 1e-6  # truncation of order step^2, rounding of order 1e-16 / step
    for name in v:
        d = _random(11, *v[name].shape)
        up, down = dict(v), dict(v)
        up[name], down[name] = v[name] + step * d, v[name] - step * d
        want = (loss(up) - loss(down)) / (2 * step)
        assert abs((g["d" + name] * d).sum() - want) < 1e-7 * max(1.0, abs(want)), name


@pytest.mark.parametrize("packed", [False, True])
def test_recurrence_statement_matches(packed):
    B, D, L = 2, 3, 9
    ids = IDS if packed else None
    n = 8 if packed else B
    t = {k: torch.tensor(_random(i, *s), requires_grad=True) for i, (k, s) in enumerate(
        {"x": (B, D, L), "gate": (B, D, L), "z": (B, D, L), "bias": (D,), "init": (n, D)}.items())}
    seq = None if ids is None else torch.tensor(ids, dtype=torch.int32)
    out, final = gated_recurrence_ref(t["x"], t["gate"], t["z"], t["bias"], seq, t["init"], True)
    w = {k: R.wide(v) for k, v in t.items()}
    eo, ef, _, _ = R.recurrence(w["x"], w["gate"], w["z"], w["bias"], ids, w["init"])
    np.testing.assert_allclose(R.wide(out), eo, atol=1e-12)
    np.testing.assert_allclose(R.wide(final), ef, atol=1e-12)
    dout, dfinal = _random(8, B, D, L), _random(9, n, D)
    ((out * torch.tensor(dout)).sum() + (final * torch.tensor(dfinal)).sum()).backward()
    g = R.recurrence_grads(w["x"], w["gate"], w["z"], w["bias"], ids, w["init"], dout, dfinal)
    for k in t:
        np.testing.assert_allclose(t[k].grad.numpy(), g["d" + k], atol=1e-12, err_msg=k)


def test_add_norm_gradients_against_differences():
    n, d, p, eps = 3, 7, 0.25, 1e-5
    keep = np.random.default_rng(0).random((n, d)) >= p
    v = {"x": _random(1, n, d), "residual": _random(2, n, d), "weight": _random(3, d)}
    dout, dres = _random(4, n, d), _random(5, n, d)

    def loss(w):
        out, r = R.add_norm(w["x"], w["residual"], w["weight"], keep, p, eps, torch.float64)
        return (out * dout).sum() + (r * dres).sum()

    _, stored = R.add_norm(v["x"], v["residual"], v["weight"], keep, p, eps, torch.float64)
    g = R.add_norm_grads(stored, v["weight"], keep, p, eps, dout, dres)
    step = 1e-6
    for name in v:
        e = _random(9, *v[name].shape)
        up, down = dict(v), dict(v)
        up[name], down[name] = v[name] + step * e, v[name] - step * e
        want = (loss(up) - loss(down)) / (2 * step)
        assert abs((g["d" + name] * e).sum() - want) < 1e-7 * max(1.0, abs(want)), name


def test_philox_known_answers():
    """The generator's published test vectors (all zero, all one, digits of pi)."""
    ones = (1 << 64) - 1
    assert R.philox_words(0, 0, [0])[0] == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    assert R.philox_words(ones, ones, [ones])[0] == [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]
    assert R.philox_words(0x299F31D0A4093822, 0x0370734413198A2E, [0x85A308D3243F6A88])[0] == [
        0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1]


def test_mask_statement_matches_definition():
    rng = torch.tensor([-1234567890123456789, 987654321987654321])
    rows, dim, p = 3, 10, 0.3
    words = R.philox_words(int(rng[0]) & ((1 << 64) - 1), int(rng[1]) & ((1 << 64) - 1), range(rows * 3))
    flat = np.array(words, dtype=np.uint64).reshape(rows, 12)[:, :dim]
    assert np.array_equal(dropout_add_rms_norm_mask_ref(rows, dim, p, rng).numpy(), flat >= int(p * 2 ** 32))


def test_add_norm_statement_matches():
    x, res, w = torch.tensor(_random(1, 4, 9)), torch.tensor(_random(2, 4, 9)), torch.tensor(_random(3, 9))
    rng = torch.tensor([5, 6])
    keep = dropout_add_rms_norm_mask_ref(4, 9, 0.4, rng).numpy()
    out, stored = dropout_add_rms_norm_ref(x, w, res, dropout_p=0.4, rng_state=rng)
    eo, er = R.add_norm(x.numpy(), res.numpy(), w.numpy(), keep, 0.4, 1e-5, torch.float64)
    np.testing.assert_allclose(out.numpy(), eo, atol=1e-12)
    np.testing.assert_allclose(stored.numpy(), er, atol=1e-12)


# ------------------------------------------------------------------------ refusals
def test_recurrence_refusals():
    x = torch.empty(2, 8, 16)
    with pytest.raises(ValueError, match="CUDA"):
        gated_recurrence_fn(x, x)
    with pytest.raises(ValueError, match="3 dimensions"):
        gated_recurrence_fn(x[0], x[0])
    with pytest.raises(ValueError, match="gate"):
        gated_recurrence_fn(x, x[:, :, :15])
    with pytest.raises(ValueError, match="z"):
        gated_recurrence_fn(x, x, x[:1])
    with pytest.raises(ValueError, match="gate_bias"):
        gated_recurrence_fn(x, x, None, torch.empty(7))
    with pytest.raises(ValueError, match="seq_idx"):
        gated_recurrence_fn(x, x, seq_idx=torch.zeros(2, 15, dtype=torch.int32))
    with pytest.raises(ValueError, match="initial_states"):
        gated_recurrence_fn(x, x, initial_states=torch.empty(3, 8))
    with pytest.raises(ValueError, match="initial_states"):
        gated_recurrence_fn(x, x, seq_idx=torch.zeros(2, 16, dtype=torch.int32), initial_states=torch.empty(3, 7))
    with pytest.raises(ValueError, match="num_sequences"):
        gated_recurrence_fn(x, x, seq_idx=torch.zeros(2, 16, dtype=torch.int32), return_final_states=True)


def test_recurrence_update_refusals():
    x, state = torch.empty(2, 8), torch.empty(2, 8)
    with pytest.raises(ValueError, match="CUDA"):
        gated_recurrence_update(x, state, x)
    with pytest.raises(ValueError, match="state"):
        gated_recurrence_update(x, torch.empty(3, 8), x)
    with pytest.raises(ValueError, match="state_indices"):
        gated_recurrence_update(x, torch.empty(3, 8), x, state_indices=torch.zeros(3, dtype=torch.int32))
    with pytest.raises(ValueError, match="state"):
        gated_recurrence_update(x, torch.empty(2, 7), x)
    with pytest.raises(ValueError, match="gate"):
        gated_recurrence_update(x, state, x[:1])


def test_add_norm_refusals():
    x, w = torch.empty(4, 8), torch.empty(8)
    with pytest.raises(ValueError, match="CUDA"):
        dropout_add_rms_norm_fn(x, w)
    for p in (1.0, -0.1, float("nan")):
        with pytest.raises(ValueError, match="dropout_p"):
            dropout_add_rms_norm_fn(x, w, dropout_p=p)
    with pytest.raises(ValueError, match="shapes"):
        dropout_add_rms_norm_fn(x, torch.empty(7))
    with pytest.raises(ValueError, match="residual"):
        dropout_add_rms_norm_fn(x, w, x[:3])
    with pytest.raises(ValueError, match="residual"):
        dropout_add_rms_norm_fn(x, w, x.half(), residual_in_fp32=True)
    with pytest.raises(ValueError, match="rng_state"):
        dropout_add_rms_norm_fn(x, w, dropout_p=0.5, rng_state=torch.zeros(3, dtype=torch.int64))


def _tensor(ptr=16, dtype=0, strides=(0, 0, 0)):
    return (ptr, dtype, *strides)


def _rec(**kw):
    order = ("x", "gate", "z", "bias", "seq_idx", "initial_states", "final_states", "out", "dout", "dfinal_states",
             "dx", "dgate", "dz", "dinitial_states")
    words = [kw.get(k, 2) for k in ("batch", "dim", "seqlen", "nstates")]
    for k in order:
        words += kw.get(k, _abi._NONE)
    return _abi.RECURRENCE_PARAMS.pack(*words, kw.get("dbias", 0), kw.get("checkpoints", 0), 0, 0)


def test_abi_refusals_need_no_gpu():
    lib = _abi.load_library()

    def refused(fn, params, status, text):
        assert fn(params, None) == status
        assert text in lib.cc1d_last_error(), lib.cc1d_last_error()

    fwd, bwd, upd = lib.cc1d_recurrence_fwd_launch, lib.cc1d_recurrence_bwd_launch, lib.cc1d_recurrence_update_launch
    t, half = _tensor(), _tensor(dtype=1)
    refused(fwd, None, 1, b"NULL")
    refused(fwd, _rec(batch=-1), 1, b"sizes")
    refused(fwd, _rec(seqlen=1 << 31), 1, b"sizes")
    refused(fwd, _rec(x=_tensor(dtype=3)), 2, b"x must be")
    refused(fwd, _rec(x=t, gate=half), 2, b"gate")
    refused(fwd, _rec(x=t, gate=t, z=half), 2, b"z must")
    refused(fwd, _rec(x=t, gate=t, out=t, seq_idx=_tensor(dtype=4)), 2, b"seq_idx")
    refused(fwd, _rec(x=t, gate=t, out=t, initial_states=half), 2, b"initial_states")
    refused(fwd, _rec(x=t, gate=t, out=t, initial_states=t, nstates=3), 1, b"one state")
    refused(fwd, _rec(x=t, gate=t), 1, b"out is required")
    refused(bwd, _rec(x=t, gate=t, dout=t, dx=t, dgate=t), 1, b"checkpoints")
    refused(bwd, _rec(x=t, gate=t, z=t, dout=t, dx=t, dgate=t, checkpoints=16), 1, b"dz is required")
    refused(bwd, _rec(x=t, gate=t, dout=t, dx=t, dgate=t, checkpoints=16, dbias=16), 1, b"workspace")
    assert lib.cc1d_recurrence_bwd_workspace_bytes(_rec(x=_tensor(dtype=4))) == -1
    assert fwd(_rec(seqlen=0), None) == 0 and fwd(_rec(batch=0, nstates=0), None) == 0

    def update(*tensors, sizes=(2, 2, 1, 2)):
        return _abi.RECURRENCE_UPDATE_PARAMS.pack(*sizes, *[w for v in tensors for w in v])

    none = _abi._NONE
    refused(upd, update(t, t, none, none, half, none, t), 2, b"state must be float32")
    refused(upd, update(t, t, none, none, t, _tensor(dtype=4), t), 2, b"state_indices")
    refused(upd, update(t, t, none, none, t, none, t, sizes=(2, 2, 1, 3)), 1, b"one state")
    assert upd(update(t, t, none, none, t, none, t, sizes=(0, 2, 1, 0)), None) == 0

    def norm(*tensors, rows=2, dim=2, eps=1e-5, p=0.0, dweight=0):
        return _abi.ADD_NORM_PARAMS.pack(rows, dim, *[w for v in tensors for w in v], dweight, 0, 0, eps, p)

    nf, nb = lib.cc1d_add_norm_fwd_launch, lib.cc1d_add_norm_bwd_launch
    m = _tensor(strides=(2, 1, 0))
    rest = (none,) * 4
    refused(nf, norm(m, none, t, none, m, m, *rest, p=1.0), 1, b"dropout_p")
    refused(nf, norm(m, none, t, none, m, m, *rest, p=0.5), 1, b"rng_state")
    refused(nf, norm(m, none, t, none, m, m, *rest, eps=-1.0), 1, b"eps")
    refused(nf, norm(m, none, t, none, m, half, *rest), 2, b"residual_out")
    refused(nf, norm(m, half, t, none, m, m, *rest), 2, b"residual must")
    refused(nf, norm(_tensor(strides=(1, 2, 0)), none, t, none, m, m, *rest), 1, b"stride 1")
    refused(nb, norm(none, none, t, none, none, m, *rest, dweight=16), 1, b"workspace")


C_PROBE = r"""
#include <stddef.h>
#include <stdio.h>
#include "causal_conv1d_b200.h"
int main(void) {
  printf("%zu %zu %zu %d\n", sizeof(cc1d_recurrence_params), sizeof(cc1d_recurrence_update_params),
         sizeof(cc1d_add_norm_params), CC1D_RECURRENCE_CHUNK);
  printf("%zu %zu %zu %zu\n", offsetof(cc1d_recurrence_params, x), offsetof(cc1d_recurrence_params, dbias),
         offsetof(cc1d_recurrence_update_params, out), offsetof(cc1d_add_norm_params, eps));
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
    five = ctypes.sizeof(_abi.CTensor)
    assert five == 40
    assert got == [_abi.RECURRENCE_PARAMS.size, _abi.RECURRENCE_UPDATE_PARAMS.size, _abi.ADD_NORM_PARAMS.size,
                   _abi.RECURRENCE_CHUNK, 32, 32 + 14 * five, 32 + 6 * five, _abi.ADD_NORM_PARAMS.size - 16]


def test_torch_ops_registered_with_fake_shapes():
    from torch._subclasses.fake_tensor import FakeTensorMode

    ops = torch.ops.causal_conv1d
    with FakeTensorMode():
        x = torch.empty(2, 70, 64, dtype=torch.bfloat16).transpose(1, 2)
        bias, init = torch.empty(64), torch.empty(2, 64)
        out, final, ck = ops.gated_recurrence_fwd(x, x, x, bias, None, init, True, 0, True)
        assert out.stride() == x.stride() and final.shape == (2, 64) and ck.shape == (2, 3, 64)
        seq = torch.empty(2, 70, dtype=torch.int32)
        assert ops.gated_recurrence_fwd(x, x, None, None, seq, None, True, 5, False)[1].shape == (5, 64)
        dx, dg, dz, db, di = ops.gated_recurrence_bwd(x, x, None, bias, None, init, ck, x, final, True, True)
        assert dx.stride() == x.stride() and dz.numel() == 0 and db.shape == (64,) and di.shape == (2, 64)
        assert ops.gated_recurrence_update(x[..., 0], init, x[..., 0], None, None, None).shape == (2, 64)
        m, w = torch.empty(3, 64, dtype=torch.float16), torch.empty(64)
        out, res = ops.dropout_add_rms_norm_fwd(m, w, None, 1e-5, 0.0, None, True)
        assert out.dtype == torch.float16 and res.dtype == torch.float32
        dx, dres, dw = ops.dropout_add_rms_norm_bwd(torch.float16, res, w, out, res, 1e-5, 0.0, None)
        assert dx.dtype == torch.float16 and dres.dtype == torch.float32 and dw.shape == (64,)


def test_missing_binding_is_named_on_use():
    missing = _abi._Missing(ImportError("no such file"))
    with pytest.raises(ImportError, match="cc1d_build.*no such file"):
        missing.recurrence(None)
