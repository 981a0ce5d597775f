"""Backward passes over more than 2^31 elements: the ends are what the 64-bit statements of a
short stretch, started from what lies before or behind it, give."""

import numpy as np
import pytest
import torch

import block_ref as R
from causal_conv1d.add_norm import dropout_add_rms_norm_bwd_function, dropout_add_rms_norm_fwd_function
from causal_conv1d.gated_recurrence import gated_recurrence_bwd_function, gated_recurrence_fwd_function

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("layout", ["channel_last", "contiguous"])
@pytest.mark.parametrize("D,L", [(72, 30_000_128), (71, 30_300_007)])
def test_recurrence_backward(D, L, layout):
    g = torch.Generator(device="cuda").manual_seed(D)
    x = torch.randn(1, L, D, generator=g, device="cuda", dtype=torch.bfloat16)
    x = x.transpose(1, 2) if layout == "channel_last" else x.view(1, D, L)
    dfinal = torch.randn(1, D, generator=g, device="cuda")
    bias = torch.zeros(D, device="cuda")
    _, _, kept = gated_recurrence_fwd_function(x, x, None, bias, None, None, False, None, True)
    dx, dgate, _, dbias, _ = gated_recurrence_bwd_function(x, x, None, bias, None, None, kept, x, dfinal, True, False)
    n = 777
    # the last positions, from the state before them
    _, mid, _ = gated_recurrence_fwd_function(x[:, :, :L - n], x[:, :, :L - n], None, bias, None, None, True, None, False)
    tail = R.wide(x[:, :, L - n:])
    e = R.recurrence_grads(tail, tail, None, None, None, R.wide(mid), tail, R.wide(dfinal))
    R.check(dx[:, :, L - n:], e["dx"], "dx, tail")
    R.check(dgate[:, :, L - n:], e["dgate"], "dgate, tail")
    # the first ones, whose gradients forget what lies 1000 positions on (a is 1/2 on average)
    head = R.wide(x[:, :, :n + 1000])
    e = R.recurrence_grads(head, head, None, None, None, None, head, None)
    R.check(dx[:, :, :n], e["dx"][:, :, :n], "dx, head")
    R.check(dgate[:, :, :n], e["dgate"][:, :, :n], "dgate, head")
    total, size = torch.zeros(D, device="cuda", dtype=torch.float64), torch.zeros(D, device="cuda", dtype=torch.float64)
    for part in dgate.split(1 << 20, 2):
        total += part.double().sum((0, 2))
        size += part.double().abs().sum((0, 2))
    # dgate is rounded to bf16 here: each addend may be off by 2^-8 of itself
    assert (dbias.double() - total).abs().max() <= 2.0 ** -8 * size.max()


@pytest.mark.parametrize("rows,dim", [(33_000, 65_536), (530_000, 4_100), (540_000, 4_001)])
def test_add_norm_backward(rows, dim):
    g = torch.Generator(device="cuda").manual_seed(dim)
    x = torch.randn(1, dim, generator=g, device="cuda", dtype=torch.bfloat16).expand(rows, dim)
    dout = torch.randn(1, dim, generator=g, device="cuda", dtype=torch.bfloat16).expand(rows, dim)
    w = 1.0 + 0.2 * torch.randn(dim, generator=g, device="cuda")
    rng, p, eps, last = torch.tensor([21, 22], device="cuda"), 0.25, 1e-5, 3
    _, stream = dropout_add_rms_norm_fwd_function(x, w, None, eps, p, rng, False)
    dx, dres, dw = dropout_add_rms_norm_bwd_function(x.dtype, stream, w, dout, None, eps, p, rng, True, True, True)
    per = -(-dim // 4)
    words = R.philox_words(21, 22, range((rows - last) * per, rows * per))
    keep = np.array(words, dtype=np.uint64).reshape(last, 4 * per)[:, :dim] >= int(p * 2 ** 32)
    assert np.array_equal(R.wide(stream[-last:]) != 0, keep & (R.wide(x[-last:]) != 0))
    e = R.add_norm_grads(R.wide(stream[-last:]), R.wide(w), keep, p, eps, R.wide(dout[-last:]), 0.0)
    R.check(dx[-last:], e["dx"], "dx")
    R.check(dres[-last:], e["dresidual"], "dresidual")
    want, size = torch.zeros(dim, device="cuda", dtype=torch.float64), torch.zeros(dim, device="cuda", dtype=torch.float64)
    for part in stream.split(max(1, (1 << 26) // dim)):
        r = part.double()
        t = dout[:1].double() * r * torch.rsqrt((r * r).mean(1, keepdim=True) + eps)
        want += t.sum(0)
        size += t.abs().sum(0)
    R.check(dw, R.wide(want), "dweight", size.max().item())
