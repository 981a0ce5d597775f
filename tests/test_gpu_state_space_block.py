"""The example model with the selective recurrence: training, serving and beam search; the
operators as torch.ops."""

import importlib.util
import os

import pytest
import torch

from causal_conv1d import beam_search_select
from causal_conv1d.selective_recurrence import selective_recurrence_bwd_function, selective_recurrence_fwd_function

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
ops = torch.ops.causal_conv1d


def _example():
    spec = importlib.util.spec_from_file_location("recurrent_block", os.path.join(ROOT, "examples", "recurrent_block.py"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def test_trains_and_serves():
    ex = _example()
    torch.manual_seed(0)
    gen = torch.Generator(device="cuda").manual_seed(0)
    model = ex.Model(16, 128, 2, layer=ex.SelectiveLayer)
    losses = ex.train(model, 3, 16, gen, log=None)
    assert all(l == l for l in losses)
    off, top = ex.serve(model, 16, gen)
    # bf16 activations rounded at the same places in both runs; matrix products of other shapes may
    # sum in another order, so a rounding may fall the other way: a few bf16 units of the logits
    assert off < 8 * 2.0 ** -8 * max(top, 1.0)


def test_gradients_against_differences():
    """The loss along a direction of all parameters."""
    ex = _example()
    torch.manual_seed(3)
    gen = torch.Generator(device="cuda").manual_seed(3)
    model = ex.Model(16, 32, 2, dtype=torch.float32, layer=ex.SelectiveLayer)
    tokens, ids, _ = ex.packed_batch(gen, 16, [30, 1, 65])
    weight = torch.randn(1, 96, 16, generator=gen, device="cuda")
    params = list(model.parameters())

    def loss():
        return (model(tokens, ids) * weight).double().sum()

    grads = torch.autograd.grad(loss(), params)
    found = torch.sqrt(sum((g.double() ** 2).sum() for g in grads))
    step = 1e-2
    values = []
    for sign in (1, -1):
        with torch.no_grad():
            for p, g in zip(params, grads):
                p.add_(g, alpha=sign * step / found.item())
            values.append(loss().item())
            for p, g in zip(params, grads):
                p.sub_(g, alpha=sign * step / found.item())
    # along the gradient the slope is its norm; differences are off by step^2 and 2^-20 |loss| / step
    assert abs((values[0] - values[1]) / (2 * step) - found.item()) < 2e-2 * found.item()


@pytest.mark.parametrize("block", ["Layer", "SelectiveLayer"])
def test_beam_search_follows_its_beams(block):
    """The beams' scores are those of whole passes over prompt and tokens."""
    ex = _example()
    torch.manual_seed(1)
    gen = torch.Generator(device="cuda").manual_seed(1)
    vocab, new, beams = 16, 6, 4
    model = ex.Model(vocab, 64, 2, dtype=torch.float32, layer=getattr(ex, block))
    prompt = torch.randint(0, vocab, (3, 21), generator=gen, device="cuda")
    tokens, scores = ex.beam_search(model, prompt, beams, new, end_token=vocab - 1)
    assert (scores[:, 1:] <= scores[:, :-1]).all()
    with torch.no_grad():
        for b in range(3):
            seen = set()
            for k in range(beams):
                row = tokens[b, k]
                seen.add(tuple(row.tolist()))
                logp = torch.log_softmax(model(torch.cat([prompt[b], row])[None])[0, 20:-1].double(), -1)
                want = 0.0
                for i in range(new):
                    want += logp[i, row[i]].item()
                    if row[i] == vocab - 1:
                        assert (row[i:] == vocab - 1).all()
                        break
                assert abs(scores[b, k].item() - want) < 1e-3
            assert len(seen) == beams


def test_beam_search_of_one_beam_is_greedy():
    ex = _example()
    torch.manual_seed(2)
    model = ex.Model(16, 64, 1, dtype=torch.float32, layer=ex.SelectiveLayer)
    prompt = torch.randint(0, 16, (2, 9), device="cuda")
    tokens, _ = ex.beam_search(model, prompt, 1, 5, end_token=99 % 16)
    with torch.no_grad():
        whole = model(torch.cat([prompt, tokens[:, 0]], 1))[:, 8:-1]
    ended = (tokens[:, 0] == 3).cumsum(-1) - (tokens[:, 0] == 3).long() > 0
    assert ((whole.argmax(-1) == tokens[:, 0]) | ended).all()


def _inputs():
    g = torch.Generator(device="cuda").manual_seed(2)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    x, delta, z, dout = (r(2, 40, 64).bfloat16().transpose(1, 2) for _ in range(4))
    B, C = (r(2, 40, 16).bfloat16().transpose(1, 2) for _ in range(2))
    return [x, delta, -torch.exp(r(64, 16)), B, C, r(64), z, r(64)], r(2, 64, 16), dout


def test_ops_match_functions():
    args, init, dout = _inputs()
    out, final, ck = ops.selective_recurrence_fwd(*args, True, None, init, True, 0, True)
    want = selective_recurrence_fwd_function(*args, True, None, init, True, None, True)
    assert all(torch.equal(a, b) for a, b in zip((out, final, ck), want))
    got = ops.selective_recurrence_bwd(*args, True, None, init, ck, dout, final, True, True)
    want = selective_recurrence_bwd_function(*args, True, None, init, ck, dout, final, True, True)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    state = init.clone()
    one = [t[..., 0] if t.dim() == 3 else t for t in args]
    first = ops.selective_recurrence_update(one[0], state, *one[1:], True, None)
    torch.testing.assert_close(first, out[..., 0], rtol=2.0 ** -7, atol=1e-6)
    logits, scores = torch.randn(2, 3, 50, device="cuda"), torch.randn(2, 3, device="cuda")
    assert all(torch.equal(a, b) for a, b in zip(ops.beam_search_select(logits, scores, None, None, 5),
                                                 beam_search_select(logits, scores, num_candidates=5)))


def test_opcheck():
    args, init, dout = _inputs()
    _, final, ck = ops.selective_recurrence_fwd(*args, True, None, init, True, 0, True)
    torch.library.opcheck(ops.selective_recurrence_fwd, (*args, True, None, init, True, 0, True))
    torch.library.opcheck(ops.selective_recurrence_bwd, (*args, True, None, init, ck, dout, final, True, True))
    one = [t[..., 0].contiguous() if t.dim() == 3 else t for t in args]
    torch.library.opcheck(ops.selective_recurrence_update, (one[0], init, *one[1:], True, None))
    logits, scores = torch.randn(2, 3, 50, device="cuda"), torch.randn(2, 3, device="cuda")
    torch.library.opcheck(ops.beam_search_select, (logits, scores, None, None, 5))
    parents = torch.zeros(1, 2, dtype=torch.int64, device="cuda")
    torch.library.opcheck(ops.beam_search_reorder, ([init, args[0].contiguous()], parents, None))
