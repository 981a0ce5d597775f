"""The example model trains, and its decoding continues its prefill; the operators as torch.ops."""

import importlib.util
import os

import pytest
import torch

import causal_conv1d  # noqa: F401  (registers the operators)
from causal_conv1d.add_norm import dropout_add_rms_norm_bwd_function, dropout_add_rms_norm_fwd_function
from causal_conv1d.gated_recurrence import gated_recurrence_bwd_function, gated_recurrence_fwd_function

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
ops = torch.ops.causal_conv1d


def _example():
    spec = importlib.util.spec_from_file_location("recurrent_block", os.path.join(ROOT, "examples", "recurrent_block.py"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def test_example_trains_and_serves():
    ex = _example()
    torch.manual_seed(0)
    gen = torch.Generator(device="cuda").manual_seed(0)
    model = ex.Model(16, 128, 2)
    losses = ex.train(model, 60, 16, gen, log=None)
    assert losses[0] > 2.0 and min(losses[-5:]) < 0.6 * losses[0]
    off, top = ex.serve(model, 16, gen)
    # bf16 activations rounded at the same places in both runs; matrix products of other shapes may
    # sum in another order, so a rounding may fall the other way: a few bf16 units of the logits
    assert off < 8 * 2.0 ** -8 * max(top, 1.0)


def test_example_training_is_one_whole_pass_per_sequence():
    """Packed sequences give what they give alone."""
    ex = _example()
    torch.manual_seed(1)
    gen = torch.Generator(device="cuda").manual_seed(1)
    model = ex.Model(16, 64, 2, dtype=torch.float32)
    tokens, ids, _ = ex.packed_batch(gen, 16, [30, 1, 65])
    with torch.no_grad():
        packed = model(tokens, ids)
        alone = torch.cat([model(tokens[:, a:b]) for a, b in ((0, 30), (30, 31), (31, 96))], 1)
    torch.testing.assert_close(packed, alone, rtol=1e-4, atol=1e-4)


def _inputs(dtype=torch.bfloat16):
    g = torch.Generator(device="cuda").manual_seed(2)
    x, gate, z, dout = (torch.randn(2, 40, 64, generator=g, device="cuda").to(dtype).transpose(1, 2) for _ in range(4))
    return x, gate, z, torch.randn(64, generator=g, device="cuda"), torch.randn(2, 64, generator=g, device="cuda"), dout


def test_ops_match_functions():
    x, gate, z, bias, init, dout = _inputs()
    out, final, ck = ops.gated_recurrence_fwd(x, gate, z, bias, None, init, True, 0, True)
    want = gated_recurrence_fwd_function(x, gate, z, bias, None, init, True, None, True)
    assert all(torch.equal(a, b) for a, b in zip((out, final, ck), want))
    got = ops.gated_recurrence_bwd(x, gate, z, bias, None, init, ck, dout, final, True, True)
    want = gated_recurrence_bwd_function(x, gate, z, bias, None, init, ck, dout, final, True, True)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    state = init.clone()
    first = ops.gated_recurrence_update(x[..., 0], state, gate[..., 0], z[..., 0], bias, None)
    torch.testing.assert_close(first, out[..., 0], rtol=2.0 ** -7, atol=1e-6)
    m, w = x[0].t(), torch.ones(64, device="cuda")
    rng = torch.tensor([1, 2], device="cuda")
    out, res = ops.dropout_add_rms_norm_fwd(m, w, m, 1e-5, 0.2, rng, False)
    want = dropout_add_rms_norm_fwd_function(m, w, m, 1e-5, 0.2, rng, False)
    assert torch.equal(out, want[0]) and torch.equal(res, want[1])
    got = ops.dropout_add_rms_norm_bwd(x.dtype, res, w, out, res, 1e-5, 0.2, rng)
    want = dropout_add_rms_norm_bwd_function(x.dtype, res, w, out, res, 1e-5, 0.2, rng, True, True, True)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_opcheck():
    x, gate, z, bias, init, dout = _inputs()
    _, final, ck = ops.gated_recurrence_fwd(x, gate, z, bias, None, init, True, 0, True)
    torch.library.opcheck(ops.gated_recurrence_fwd, (x, gate, z, bias, None, init, True, 0, True))
    torch.library.opcheck(ops.gated_recurrence_bwd, (x, gate, z, bias, None, init, ck, dout, final, True, True))
    torch.library.opcheck(ops.gated_recurrence_update, (x[..., 0].contiguous(), init, gate[..., 0].contiguous(), None, bias, None))
    m, w, rng = x[0].t().contiguous(), torch.ones(64, device="cuda"), torch.tensor([1, 2], device="cuda")
    torch.library.opcheck(ops.dropout_add_rms_norm_fwd, (m, w, m, 1e-5, 0.2, rng, False))
    torch.library.opcheck(ops.dropout_add_rms_norm_bwd, (m.dtype, m, w, m, m, 1e-5, 0.2, rng))


def test_second_derivatives_are_refused():
    x = torch.randn(1, 8, 20, device="cuda", requires_grad=True)
    out = causal_conv1d.gated_recurrence_fn(x, x)
    (g,) = torch.autograd.grad(out.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        torch.autograd.grad(g.sum(), x)
    m = torch.randn(3, 16, device="cuda", requires_grad=True)
    (g,) = torch.autograd.grad(causal_conv1d.dropout_add_rms_norm_fn(m, torch.ones(16, device="cuda"))[0].sum(), m, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        torch.autograd.grad(g.sum(), m)
