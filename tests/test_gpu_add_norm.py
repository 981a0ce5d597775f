"""dropout_add_rms_norm_fn against the 64-bit statement."""

import numpy as np
import pytest
import torch

import block_ref as R
from causal_conv1d import dropout_add_rms_norm_fn
from causal_conv1d.add_norm import dropout_add_rms_norm_mask_ref

pytestmark = pytest.mark.gpu

PAIRS = [(torch.float32, torch.float32), (torch.float16, torch.float16), (torch.float16, torch.float32),
         (torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32)]
EPS = 1e-5


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _matrix(g, rows, dim, dtype, kind="dense"):
    if kind == "odd":  # a slice that starts off its rows' alignment
        return torch.randn(rows, dim + 3, generator=g, device="cuda").to(dtype)[:, 1:1 + dim]
    return torch.randn(rows, dim, generator=g, device="cuda").to(dtype)


def _run_and_check(rows, dim, dtype, stream, p, residual=True, weight=torch.float32, kind="dense", seed=0):
    g = _gen(seed + rows + dim)
    x = _matrix(g, rows, dim, dtype, kind).detach().requires_grad_()
    res = _matrix(g, rows, dim, stream, kind).detach().requires_grad_() if residual else None
    w = (1.0 + 0.2 * torch.randn(dim, generator=g, device="cuda")).to(weight).requires_grad_()
    rng = torch.randint(-(1 << 62), 1 << 62, (2,), generator=g, device="cuda")
    out, kept = dropout_add_rms_norm_fn(x, w, res, EPS, p, rng if p else None, residual_in_fp32=stream == torch.float32)
    assert out.dtype == dtype and kept.dtype == stream and out.shape == x.shape
    keep = dropout_add_rms_norm_mask_ref(rows, dim, p, rng).cpu().numpy() if p else None
    eo, er = R.add_norm(R.wide(x), R.wide(res), R.wide(w), keep, p, EPS, stream)
    R.check(kept, er, "residual_out")
    # the rest is stated from the stream as the kernel stored it: a value that lies between two
    # 16-bit numbers may be rounded to either when computed in 32 or in 64 bits
    eo, _ = R.add_norm(R.wide(kept), None, R.wide(w), None, 0.0, EPS, stream)
    R.check(out, eo, "out")
    dout, dres = _matrix(g, rows, dim, dtype, kind), _matrix(g, rows, dim, stream, kind)
    names = ["x", "weight"] + (["residual"] if residual else [])
    found = dict(zip(names, torch.autograd.grad([out, kept], [x, w] + ([res] if residual else []), [dout, dres])))
    e = R.add_norm_grads(R.wide(kept), R.wide(w), keep, p, EPS, R.wide(dout), R.wide(dres))
    for k, v in found.items():
        R.check(v, e["d" + k], "d" + k, e["weight_scale"] if k == "weight" else None)
    return out, kept, found


@pytest.mark.parametrize("dtype,stream", PAIRS)
@pytest.mark.parametrize("dim", [1, 2, 5, 8, 31, 64, 100, 256, 257, 1000, 1024, 2050])
def test_widths(dim, dtype, stream):
    _run_and_check(9, dim, dtype, stream, 0.3)


@pytest.mark.parametrize("dtype,stream", PAIRS)
@pytest.mark.parametrize("dim", [4096, 4104, 8192, 8200, 16384, 20001, 40000])
def test_wide_rows(dim, dtype, stream):
    _run_and_check(5, dim, dtype, stream, 0.1)


@pytest.mark.parametrize("rows", [1, 2, 3, 7, 64, 65, 1000, 5000])
@pytest.mark.parametrize("dim", [40, 512])
def test_row_counts(rows, dim):
    _run_and_check(rows, dim, torch.bfloat16, torch.float32, 0.2)


@pytest.mark.parametrize("p,residual,kind", [(0.0, True, "dense"), (0.0, False, "dense"), (0.5, False, "dense"), (0.25, True, "odd"), (0.0, True, "odd")])
@pytest.mark.parametrize("dtype,stream", PAIRS)
def test_options(dtype, stream, p, residual, kind):
    _run_and_check(33, 200, dtype, stream, p, residual, weight=dtype, kind=kind)


def test_leading_dimensions():
    x = torch.randn(2, 3, 5, 48, device="cuda")
    w = torch.ones(48, device="cuda")
    rng = torch.tensor([1, 2], device="cuda")
    out, res = dropout_add_rms_norm_fn(x, w, x, dropout_p=0.3, rng_state=rng)
    flat, fres = dropout_add_rms_norm_fn(x.view(30, 48), w, x.view(30, 48), dropout_p=0.3, rng_state=rng)
    assert torch.equal(out.view(30, 48), flat) and torch.equal(res.view(30, 48), fres)
    one, _ = dropout_add_rms_norm_fn(x[0, 0, 0], w)
    assert one.shape == (48,)
    t = torch.randn(3, 48, 5, device="cuda").transpose(1, 2)  # channel stride 5
    assert torch.equal(dropout_add_rms_norm_fn(t, w)[0], dropout_add_rms_norm_fn(t.contiguous(), w)[0])


def test_mask_statistics_and_dependence():
    rows, dim, p = 512, 1024, 0.25
    x = torch.ones(rows, dim, device="cuda")
    w = torch.ones(dim, device="cuda")

    def mask(seed, offset):
        return dropout_add_rms_norm_fn(x, w, dropout_p=p, rng_state=torch.tensor([seed, offset], device="cuda"))[1] != 0

    m = mask(1, 2)
    n = rows * dim
    # the share kept is binomial; six standard deviations
    assert abs(m.double().mean().item() - (1 - p)) < 6 * (p * (1 - p) / n) ** 0.5
    assert torch.equal(m, mask(1, 2))
    for other in (mask(2, 2), mask(1, 3)):
        same = (m == other).double().mean().item()
        want = p * p + (1 - p) ** 2
        assert abs(same - want) < 6 * (want * (1 - want) / n) ** 0.5
    assert torch.equal(m, dropout_add_rms_norm_mask_ref(rows, dim, p, torch.tensor([1, 2], device="cuda")))


def test_dropped_places_are_not_read():
    """A dropped element is left out, whatever it holds."""
    rng = torch.tensor([3, 4], device="cuda")
    keep = dropout_add_rms_norm_mask_ref(20, 300, 0.5, rng)
    x, res = torch.randn(20, 300, device="cuda"), torch.randn(20, 300, device="cuda")
    w = torch.ones(300, device="cuda")
    a = dropout_add_rms_norm_fn(x, w, res, dropout_p=0.5, rng_state=rng)
    b = dropout_add_rms_norm_fn(x.masked_fill(~keep, float("nan")), w, res, dropout_p=0.5, rng_state=rng)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_drawn_state_is_replayed_by_the_backward():
    x = torch.randn(64, 128, device="cuda", requires_grad=True)
    w = torch.ones(128, device="cuda")
    torch.manual_seed(5)
    _, res = dropout_add_rms_norm_fn(x, w, dropout_p=0.4)
    (g,) = torch.autograd.grad(res, x, torch.ones_like(res))
    assert torch.equal(g != 0, res != 0)
    torch.manual_seed(5)
    assert torch.equal(dropout_add_rms_norm_fn(x, w, dropout_p=0.4)[1], res)


def test_zero_rows_of_the_stream():
    """A row of zeros has no direction: its norm is zero and its gradient finite."""
    x = torch.zeros(3, 64, device="cuda", requires_grad=True)
    w = torch.ones(64, device="cuda", requires_grad=True)
    out, res = dropout_add_rms_norm_fn(x, w)
    gx, gw = torch.autograd.grad([out, res], [x, w], [torch.ones_like(out), torch.zeros_like(res)])
    assert not out.any() and not gw.any()
    torch.testing.assert_close(gx, torch.full_like(gx, EPS ** -0.5), rtol=1e-5, atol=0)


@pytest.mark.parametrize("shape", [(0, 16), (3, 0), (0, 0)])
def test_empty(shape):
    x = torch.empty(shape, device="cuda", requires_grad=True)
    w = torch.ones(shape[1], device="cuda", requires_grad=True)
    out, res = dropout_add_rms_norm_fn(x, w, x)
    gx, gw = torch.autograd.grad([out, res], [x, w], [out.detach(), res.detach()])
    assert out.shape == shape and gx.shape == shape and not gw.any()


def test_one_gradient_only():
    g = _gen(9)
    x, res = (torch.randn(40, 96, generator=g, device="cuda").requires_grad_() for _ in range(2))
    w = torch.randn(96, generator=g, device="cuda").requires_grad_()
    d = torch.randn(40, 96, generator=g, device="cuda")
    out, kept = dropout_add_rms_norm_fn(x, w, res)
    zero = np.zeros((40, 96))
    e = R.add_norm_grads(R.wide(kept), R.wide(w), None, 0.0, EPS, R.wide(d), zero)
    for k, v in zip(("dx", "dweight", "dresidual"), torch.autograd.grad(out, [x, w, res], d, retain_graph=True)):
        R.check(v, e[k], k, e["weight_scale"] if k == "dweight" else None)
    gx, gr = torch.autograd.grad(kept, [x, res], d)
    assert torch.equal(gx, d) and torch.equal(gr, d)


def test_against_differences():
    """As for the recurrence: a step of 2^-6 in fp32, 8e-3 of the gradient's norm."""
    g = _gen(21)
    v = {"x": torch.randn(6, 80, generator=g, device="cuda"), "residual": torch.randn(6, 80, generator=g, device="cuda"),
         "weight": torch.randn(80, generator=g, device="cuda")}
    dout, dres = (torch.randn(6, 80, generator=g, device="cuda") for _ in range(2))
    rng = torch.tensor([8, 9], device="cuda")

    def loss(t):
        out, r = dropout_add_rms_norm_fn(t["x"], t["weight"], t["residual"], dropout_p=0.3, rng_state=rng)
        return (out.double() * dout.double()).sum() + (r.double() * dres.double()).sum()

    leaves = {k: t.clone().requires_grad_() for k, t in v.items()}
    grads = dict(zip(v, torch.autograd.grad(loss(leaves), list(leaves.values()))))
    for k in v:
        d = torch.randn(v[k].shape, generator=g, device="cuda")
        up, down = dict(v), dict(v)
        up[k], down[k] = v[k] + d * 2.0 ** -6, v[k] - d * 2.0 ** -6
        want = ((loss(up) - loss(down)) * 2.0 ** 5).item()
        got = (grads[k].double() * d.double()).sum().item()
        assert abs(got - want) <= 8e-3 * grads[k].double().norm().item(), (k, got, want)


def test_results_repeat_and_other_stream():
    g = _gen(30)
    x, res = (torch.randn(3000, 640, generator=g, device="cuda").to(torch.bfloat16).requires_grad_() for _ in range(2))
    w = torch.randn(640, generator=g, device="cuda").requires_grad_()
    rng = torch.tensor([5, 5], device="cuda")
    d = torch.randn(3000, 640, generator=g, device="cuda").to(torch.bfloat16)

    def once():
        out, kept = dropout_add_rms_norm_fn(x, w, res, dropout_p=0.1, rng_state=rng)
        return [out, kept, *torch.autograd.grad([out, kept], [x, res, w], [d, d])]

    first = once()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = once()
    torch.cuda.current_stream().wait_stream(side)
    for _ in range(20):
        for a, b, c in zip(first, once(), other):
            assert torch.equal(a, b) and torch.equal(a, c)


def test_graph_replay_takes_a_new_mask():
    x = torch.randn(100, 256, device="cuda")
    w = torch.ones(256, device="cuda")
    rng = torch.tensor([1, 0], device="cuda")
    dropout_add_rms_norm_fn(x, w, x, dropout_p=0.5, rng_state=rng)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, res = dropout_add_rms_norm_fn(x, w, x, dropout_p=0.5, rng_state=rng)
    for offset in (7, 8):
        rng[1] = offset
        graph.replay()
        torch.cuda.synchronize()
        want = dropout_add_rms_norm_fn(x, w, x, dropout_p=0.5, rng_state=torch.tensor([1, offset], device="cuda"))
        assert torch.equal(out, want[0]) and torch.equal(res, want[1])


def test_offsets_past_32_bits():
    rows, dim = 33000, 65536  # 2.16 G elements
    x = torch.randn(1, dim, device="cuda", dtype=torch.bfloat16).expand(rows, dim)
    w = torch.ones(dim, device="cuda")
    rng = torch.tensor([11, 12], device="cuda")
    out, res = dropout_add_rms_norm_fn(x, w, None, dropout_p=0.5, rng_state=rng)
    keep = dropout_add_rms_norm_mask_ref(rows, dim, 0.5, rng)[-3:].cpu().numpy()
    eo, er = R.add_norm(R.wide(x[-3:]), None, R.wide(w), keep, 0.5, EPS, torch.bfloat16)
    R.check(res[-3:], er, "residual_out")
    R.check(out[-3:], eo, "out")


def test_type_refusals():
    x, w = torch.randn(4, 8, device="cuda"), torch.ones(8, device="cuda")
    with pytest.raises(TypeError, match="residual"):
        dropout_add_rms_norm_fn(x, w, x.half())
    with pytest.raises(TypeError, match="dtype"):
        dropout_add_rms_norm_fn(x.double(), w.double())
    with pytest.raises(TypeError, match="rng_state"):
        dropout_add_rms_norm_fn(x, w, dropout_p=0.5, rng_state=torch.zeros(2, device="cuda"))
