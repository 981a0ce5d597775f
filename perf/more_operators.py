"""Cases, plain forms and 64-bit statements of the selective recurrence and of beam search.

What a state-space language model needs next to the causal convolution:

* ``selective_recurrence_fn``: with step sizes s_t = softplus(delta_t + delta_bias),
  h_t[d, n] = exp(s_t[d] A[d, n]) h_{t-1}[d, n] + s_t[d] x_t[d] B_t[n],
  out_t[d] = (sum_n C_t[n] h_t[d, n] + D[d] x_t[d]) silu(z_t[d]),
  over whole or packed sequences, with its backward pass;
* ``selective_recurrence_update``: the same for a few tokens against states kept in a pool;
* ``beam_search_select``: the best continuations of the beams of each request, over beams and
  vocabulary;
* ``beam_search_reorder``: the states of the beams follow the choice, in place.

``run`` makes one pass of a case, in elementary torch operations or (``own``) by the calls of
the package; ``exact`` states the same in 64 bits.
"""

import math
import os
import sys

import torch

own = False

_DT = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
_SIZE = {"float32": 4, "float16": 2, "bfloat16": 2}


# --------------------------------------------------------------------------- cases
def _recurrence(name, op, dtype, batch, dim, seqlen, dstate=16, groups=1, layout="channel_last", z=True, skip=True,
                states="none", nseq=0, pad=0):
    # states: "none", "out" (final states are returned) or "both" (initial ones are given too)
    return {"name": name, "op": op, "dtype": dtype, "batch": batch, "dim": dim, "seqlen": seqlen, "dstate": dstate,
            "groups": groups, "layout": layout, "z": z, "skip": skip, "states": states, "nseq": nseq, "pad": pad}


def _update(name, dtype, batch, dim, dstate, tokens, slots, groups=1, z=True):
    return {"name": name, "op": "update", "dtype": dtype, "batch": batch, "dim": dim, "dstate": dstate, "tokens": tokens,
            "slots": slots, "groups": groups, "z": z}


def _select(name, dtype, batch, beams, vocab, finished, candidates):
    return {"name": name, "op": "select", "dtype": dtype, "batch": batch, "beams": beams, "vocab": vocab,
            "finished": finished, "candidates": candidates}


def _reorder(name, dtype, batch, beams, dim, dstate, layers, pool):
    return {"name": name, "op": "reorder", "dtype": dtype, "batch": batch, "beams": beams, "dim": dim, "dstate": dstate,
            "layers": layers, "pool": pool}


def listed():
    return [
        # A training step of one layer: 4 sequences of 2048 tokens.
        _recurrence("train_4x4096x2048", "train", "bfloat16", 4, 4096, 2048),
        # A training step on 12 packed documents of different lengths.
        _recurrence("train_packed_5120x8192", "train", "float16", 1, 5120, 8192, nseq=12, pad=96),
        # (batch, dim, seqlen) contiguous, odd sizes, 32-bit, two groups, states carried in and out.
        _recurrence("train_rows_3x770x1027", "train", "float32", 3, 770, 1027, dstate=7, groups=2, layout="rows",
                    states="both"),
        # The largest training step.
        _recurrence("train_4x4096x4096", "train", "bfloat16", 4, 4096, 4096),
        # Serving: the prompts of 8 requests, packed; their states go to the decode steps.
        _recurrence("prefill_packed_8192x8192", "prefill", "bfloat16", 1, 8192, 8192, states="out", nseq=8),
        # Serving: two short prompts.
        _recurrence("prefill_rows_2x1000x77", "prefill", "float16", 2, 1000, 77, layout="rows", states="out"),
        # Decoding one request, one token: latency.
        _update("update_1x4096", "bfloat16", 1, 4096, 16, 1, 0),
        # Decoding 128 requests whose states lie scattered in a pool of 160.
        _update("update_128x8192_pool", "bfloat16", 128, 8192, 16, 1, 160),
        # One request decoded with 4 beams: latency.
        _select("select_1x4x32000", "bfloat16", 1, 4, 32000, False, 4),
        # 64 requests of 8 beams over a large vocabulary, some beams at their end.
        _select("select_64x8x128000", "bfloat16", 64, 8, 128000, True, 16),
        # The states of one request's 4 beams in 4 layers: latency.
        _reorder("reorder_1x4_4_layers", "bfloat16", 1, 4, 2048, 16, 4, False),
        # The states of 32 requests of 8 beams, scattered in a pool, in 4 layers.
        _reorder("reorder_32x8_pool", "bfloat16", 32, 8, 4096, 16, 4, True),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["train", "train", "train", "prefill", "prefill", "update", "update", "select", "select", "reorder"])
    dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
    if op == "select":
        vocab, beams = _spread(rng, 32, 150000), rng.choice([1, 2, 3, 4, 5, 8, 16])
        batch = max(1, min(_spread(rng, 1, 128), (1 << 26) // (vocab * beams)))
        return {"op": op, "dtype": dtype, "batch": batch, "beams": beams, "vocab": vocab, "finished": rng.random() < 0.5,
                "candidates": rng.choice([beams, beams, 2 * beams])}
    if op == "reorder":
        beams = rng.choice([1, 2, 3, 4, 5, 8, 16])
        return {"op": op, "dtype": dtype, "batch": _spread(rng, 1, 32), "beams": beams, "dim": _spread(rng, 64, 4096),
                "dstate": rng.choice([16, 16, 8, 13, 64]), "layers": rng.randint(1, 4), "pool": rng.random() < 0.5}
    dim = _spread(rng, 64, 8192)
    dstate = rng.choice([16, 16, 16, 8, 32, 64, rng.randint(1, 64)])
    groups = rng.choice([1, 1, 1, 2, 4])
    dim = max(1, dim // groups) * groups
    if op == "update":
        batch = max(1, min(_spread(rng, 1, 256), (1 << 25) // (dim * dstate)))
        return {"op": op, "dtype": dtype, "batch": batch, "dim": dim, "dstate": dstate, "tokens": rng.choice([1, 1, 1, 2, 4]),
                "slots": rng.choice([0, batch, batch + rng.randint(1, 64)]), "groups": groups, "z": rng.random() < 0.7}
    packed = rng.random() < 0.35
    most = (1 << 30) // (dim * dstate)
    seqlen = min(_spread(rng, 64 if packed else 1, 16384), most)
    batch = 1 if packed else max(1, min(_spread(rng, 1, 16), most // seqlen))
    return {"op": op, "dtype": dtype, "batch": batch, "dim": dim, "seqlen": seqlen, "dstate": dstate, "groups": groups,
            "layout": rng.choice(["channel_last", "channel_last", "rows"]), "z": rng.random() < 0.7,
            "skip": rng.random() < 0.7, "states": rng.choice(["none", "out", "both"]),
            "nseq": rng.randint(1, 24) if packed else 0, "pad": rng.choice([0, 17]) if packed else 0}


# --------------------------------------------------------------------------- inputs
def _packing(seqlen, nseq, pad, gen):
    """Ids of ``nseq`` packed sequences of random lengths (some may be empty), then -1 padding."""
    end = max(1, seqlen - pad)
    cuts = torch.sort(torch.randint(0, end + 1, (nseq - 1,), generator=gen, device="cuda")).values
    pos = torch.arange(seqlen, device="cuda")
    ids = torch.searchsorted(cuts, pos, right=True)
    return torch.where(pos < end, ids, torch.full_like(ids, -1)).to(torch.int32).unsqueeze(0)


def _prepare_select(case, st, gen, normal):
    batch, beams, vocab = case["batch"], case["beams"], case["vocab"]
    st["logits"] = normal(batch, beams, vocab, scale=2.5).to(_DT[case["dtype"]])
    # cumulative log-probabilities of the beams so far
    st["scores"] = -20.0 * torch.rand(batch, beams, generator=gen, device="cuda")
    st["finished"] = torch.rand(batch, beams, generator=gen, device="cuda") < 0.2 if case["finished"] else None
    return st


def _prepare_reorder(case, st, gen, normal):
    batch, beams, dim = case["batch"], case["beams"], case["dim"]
    rows = batch * beams
    slots = rows + 16 if case["pool"] else rows
    dt = _DT[case["dtype"]]
    st["states"] = []
    for _ in range(case["layers"]):
        # the convolution's states as its decode step likes them, channel-last, and the recurrence's
        st["states"].append(normal(slots, 3, dim).to(dt).transpose(1, 2))
        st["states"].append(normal(slots, dim, case["dstate"]))
    st["parents"] = torch.randint(0, beams, (batch, beams), generator=gen, device="cuda")
    st["indices"] = torch.randperm(slots, generator=gen, device="cuda")[:rows].to(torch.int32) if case["pool"] else None
    return st


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, scale=1.0, dtype=torch.float32):
        return torch.randn(*shape, generator=gen, device="cuda", dtype=dtype).mul_(scale)

    st = {"case": dict(case)}
    if case["op"] == "select":
        return _prepare_select(case, st, gen, normal)
    if case["op"] == "reorder":
        return _prepare_reorder(case, st, gen, normal)
    dt = _DT[case["dtype"]]
    batch, dim, n, groups = case["batch"], case["dim"], case["dstate"], case["groups"]
    tokens = case["tokens"] if case["op"] == "update" else case["seqlen"]
    rows = case.get("layout") == "rows"

    def sequence(scale=1.0):
        if rows:
            return normal(batch, dim, tokens, scale=scale, dtype=dt)
        return normal(batch, tokens, dim, scale=scale, dtype=dt).transpose(1, 2)

    st["x"], st["delta"] = sequence(), sequence(0.5)
    st["z"] = sequence() if case["z"] else None
    # decay rates around 1 to dstate, and steps of 0.001 to 0.1, as such models start
    st["A"] = -torch.arange(1, n + 1, device="cuda", dtype=torch.float32) * torch.exp(normal(dim, n, scale=0.2))
    step = torch.exp(math.log(1e-3) + math.log(100.0) * torch.rand(dim, generator=gen, device="cuda"))
    st["bias"] = step + torch.log(-torch.expm1(-step))
    st["D"] = 1.0 + normal(dim, scale=0.1) if case.get("skip", True) else None
    if rows:
        st["B"], st["C"] = (normal(batch, groups, n, tokens, dtype=dt) for _ in range(2))
    else:
        # B and C lie in one projection, behind the low-rank part that delta is made from
        rank = max(1, dim // 16)
        proj = normal(batch, tokens, rank + 2 * groups * n, dtype=dt)
        st["B"], st["C"] = (proj[..., rank + k * groups * n:rank + (k + 1) * groups * n].unflatten(-1, (groups, n)).permute(0, 2, 3, 1)
                            for k in range(2))
    if groups == 1:
        st["B"], st["C"] = st["B"].squeeze(1), st["C"].squeeze(1)
    if case["op"] == "update":
        pool = case["slots"] or batch
        st["state"] = normal(pool, dim, n, scale=0.5)
        st["indices"] = torch.randperm(pool, generator=gen, device="cuda")[:batch].to(torch.int32) if case["slots"] else None
        if tokens == 1:
            for k in ("x", "delta", "z", "B", "C"):
                st[k] = None if st[k] is None else st[k].squeeze(-1)
        return st
    nstates = case["nseq"] or batch
    st["seq_idx"] = _packing(tokens, case["nseq"], case["pad"], gen) if case["nseq"] else None
    st["init"] = normal(nstates, dim, n, scale=0.5) if case["states"] == "both" else None
    if case["op"] == "train":
        st["dout"] = sequence()
        st["dfinal"] = normal(nstates, dim, n) if case["states"] != "none" else None
        for k in ("x", "delta", "A", "B", "C", "D", "z", "bias", "init"):
            if st[k] is not None:
                st[k] = st[k].detach().requires_grad_()
    return st


# ------------------------------------------------------- the package's operators
def _package():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "cute-causal-conv1d_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import causal_conv1d

    return causal_conv1d


def _run_own(st):
    cc = _package()
    case = st["case"]
    if case["op"] == "select":
        scores, parents, tokens = cc.beam_search_select(st["logits"], st["scores"], finished=st["finished"], end_token=2,
                                                        num_candidates=case["candidates"])
        return {"scores": scores, "parents": parents, "tokens": tokens}
    if case["op"] == "reorder":
        cc.beam_search_reorder(st["states"], st["parents"], state_indices=st["indices"])
        return {"states": st["states"]}
    if case["op"] == "update":
        out = cc.selective_recurrence_update(st["x"], st["state"], st["delta"], st["A"], st["B"], st["C"], st["D"], st["z"],
                                             st["bias"], state_indices=st["indices"])
        return {"out": out, "state": st["state"]}
    kept = case["states"] != "none"

    def forward():
        got = cc.selective_recurrence_fn(st["x"], st["delta"], st["A"], st["B"], st["C"], st["D"], st["z"], st["bias"],
                                         seq_idx=st["seq_idx"], initial_states=st["init"], return_final_states=kept,
                                         num_sequences=case["nseq"] or None)
        return got if kept else (got,)

    if case["op"] == "prefill":
        with torch.no_grad():
            return dict(zip(("out", "final"), forward()))
    outs = forward()
    names = [k for k in ("x", "delta", "A", "B", "C", "D", "z", "bias", "init") if st[k] is not None]
    found = torch.autograd.grad(outs, [st[k] for k in names], (st["dout"], st["dfinal"])[:len(outs)])
    res = dict(zip(("out", "final"), outs))
    res.update({"d" + k: g for k, g in zip(names, found)})
    return res


# ------------------------------------------------------------------- plain forms
def _scan(a, b):
    """h_t = a_t h_{t-1} + b_t along the first axis, from h_{-1} = 0: neighbours are joined,
    the half-length recurrence solved, and the even places filled in from it."""
    n = a.shape[0]
    if n == 1:
        return b
    m = n // 2
    even_a, odd_a, even_b, odd_b = a[0:2 * m:2], a[1::2], b[0:2 * m:2], b[1::2]
    odd = _scan(even_a * odd_a, torch.addcmul(odd_b, odd_a, even_b))
    h = torch.empty_like(b)
    h[1::2] = odd
    h[0] = b[0]
    rest = b[2::2].shape[0]
    h[2::2] = torch.addcmul(b[2::2], a[2::2], odd[:rest])
    return h


def _edges(st, tokens):
    """(valid, first, last) of each place, as (tokens, batch) truth values, and the row of the
    states that its sequence has."""
    x, ids = st["x"], st["seq_idx"]
    if ids is None:
        ids = torch.arange(x.shape[0], device=x.device).unsqueeze(1).expand(x.shape[0], tokens)
    ids = ids.long().t()
    none = torch.full_like(ids[:1], -1)
    valid = ids >= 0
    first = valid & (ids != torch.cat([none, ids[:-1]]))
    last = valid & (ids != torch.cat([ids[1:], none]))
    return valid, first, last, ids.clamp(min=0)


def _time_first(t):
    """(batch, dim, tokens) -> (tokens, batch, dim) in 32 bits."""
    return t.detach().permute(2, 0, 1).float()


def _per_channel(t, groups, dim):
    """B or C as (tokens, batch, groups, 1, dstate) in 32 bits."""
    t = t.detach().float()
    t = t if t.dim() == 4 else t.unsqueeze(1)
    return t.permute(3, 0, 1, 2).unsqueeze(3)


def _by_group(t, groups):
    """(..., dim, dstate) -> (..., groups, dim / groups, dstate), a view."""
    return t.unflatten(-2, (groups, -1))


def _as_input(t, like):
    """(tokens, batch, dim) results in the type and layout of an input."""
    if like.stride(1) == 1:
        return t.permute(1, 0, 2).to(like.dtype, memory_format=torch.contiguous_format).transpose(1, 2)
    return t.permute(1, 2, 0).to(like.dtype, memory_format=torch.contiguous_format)


def _of_group(t, like):
    """(tokens, batch, groups, dstate) gradients in the type and shape of B or C."""
    t = t.permute(1, 2, 3, 0).to(like.dtype)
    return t if like.dim() == 4 else t.squeeze(1)


def _step_size(u):
    return u.clamp(min=0.0) + torch.log1p(torch.exp(-u.abs()))


def _plain_recurrence(st):
    case = st["case"]
    tokens, dim, groups = case["seqlen"], case["dim"], case["groups"]
    x = _time_first(st["x"])
    u = _time_first(st["delta"]) + st["bias"].detach()
    s = _step_size(u)
    A = st["A"].detach()
    B, C = (_per_channel(st[k], groups, dim) for k in ("B", "C"))
    valid, first, last, rows = _edges(st, tokens)
    wide = lambda m: m[..., None, None]  # noqa: E731
    nstates = case["nseq"] or case["batch"]
    zero = torch.zeros((), device=x.device)
    init = st["init"].detach() if st["init"] is not None else torch.zeros(nstates, dim, case["dstate"], device=x.device)
    a = torch.exp(s.unsqueeze(-1) * A)  # (tokens, batch, dim, dstate)
    b = (_by_group((s * x).unsqueeze(-1), groups) * B).flatten(2, 3)
    b.masked_fill_(wide(~valid), 0.0)
    b[first] += a[first] * init[rows[first]]
    h = _scan(a.masked_fill(wide(first | ~valid), 0.0), b)
    del b
    y = (_by_group(h, groups) * C).sum(-1).flatten(2, 3)
    if st["D"] is not None:
        y = y + st["D"].detach() * x
    out = y
    if st["z"] is not None:
        z = _time_first(st["z"])
        sz = torch.sigmoid(z)
        out = y * (z * sz)
    out = torch.where(valid.unsqueeze(-1), out, zero)
    res = {"out": _as_input(out, st["x"])}
    if case["states"] != "none":
        final = init.clone()
        final[rows[last]] = h[last]
        res["final"] = final
    if case["op"] == "prefill":
        return res
    dy = torch.where(valid.unsqueeze(-1), _time_first(st["dout"]), zero)
    if st["z"] is not None:
        res["dz"] = _as_input(dy * y * (sz * (1 + z * (1 - sz))), st["z"])
        dy = dy * (z * sz)
    res["dC"] = _of_group((_by_group(h, groups) * _by_group(dy.unsqueeze(-1), groups)).sum(3), st["C"])
    # the gradient of h, carried from a sequence's last place back
    dh = (_by_group(dy.unsqueeze(-1), groups) * C).flatten(2, 3)
    if st["dfinal"] is not None:
        dh[last] += st["dfinal"][rows[last]]
    nxt = torch.cat([a[1:], torch.zeros_like(a[:1])]).masked_fill_(wide(last | ~valid), 0.0)
    g = _scan(nxt.flip(0), dh.flip(0)).flip(0)
    del nxt, dh
    if st["init"] is not None:
        dinit = st["dfinal"].clone()  # a sequence without tokens hands its state through
        dinit[rows[first]] = a[first] * g[first]
        res["dinit"] = dinit
    gb = (_by_group(g, groups) * B).sum(-1).flatten(2, 3)
    res["dB"] = _of_group((_by_group(g, groups) * _by_group((s * x).unsqueeze(-1), groups)).sum(3), st["B"])
    h = torch.cat([torch.zeros_like(h[:1]), h[:-1]])  # h_{t-1}
    h[first] = init[rows[first]]
    h.mul_(a).mul_(g)
    h.masked_fill_(wide(~valid), 0.0)
    del a, g
    res["dA"] = (h * s.unsqueeze(-1)).sum((0, 1))
    ds = (h * A).sum(-1) + x * gb
    du = torch.where(valid.unsqueeze(-1), ds * torch.sigmoid(u), zero)
    dx = s * gb
    if st["D"] is not None:
        dx = dx + st["D"].detach() * dy
        res["dD"] = (dy * x).sum((0, 1))
    res["dx"] = _as_input(torch.where(valid.unsqueeze(-1), dx, zero), st["x"])
    res["ddelta"] = _as_input(du, st["delta"])
    res["dbias"] = du.sum((0, 1))
    return res


def _plain_update(st):
    groups = st["case"]["groups"]
    x, delta, z, B, C = (st[k] for k in ("x", "delta", "z", "B", "C"))
    flat = x.dim() == 2
    if flat:
        x, delta, z, B, C = (None if t is None else t.unsqueeze(-1) for t in (x, delta, z, B, C))
    x = _time_first(x)
    s = _step_size(_time_first(delta) + st["bias"])
    B, C = _per_channel(B, groups, x.shape[2]), _per_channel(C, groups, x.shape[2])
    a = torch.exp(s.unsqueeze(-1) * st["A"])
    b = (_by_group((s * x).unsqueeze(-1), groups) * B).flatten(2, 3)
    rows = st["indices"].long() if st["indices"] is not None else slice(None)
    b[0] = torch.addcmul(b[0], a[0], st["state"][rows])
    h = _scan(a, b)
    st["state"][rows] = h[-1]
    out = (_by_group(h, groups) * C).sum(-1).flatten(2, 3) + st["D"] * x
    if z is not None:
        z = _time_first(z)
        out = out * (z * torch.sigmoid(z))
    out = out.permute(1, 2, 0)
    return {"out": (out.squeeze(-1) if flat else out).to(st["x"].dtype), "state": st["state"]}


def _plain_select(st):
    """In 64 bits: two continuations' scores may lie closer than 32 bits tell apart."""
    x = st["logits"].double()
    top = x.amax(-1, keepdim=True)
    logp = x - (top + torch.log(torch.exp(x - top).sum(-1, keepdim=True)))
    if st["finished"] is not None:
        # a beam at its end has one continuation, the end token again, at no cost
        vocab = torch.arange(x.shape[-1], device=x.device)
        ended = torch.zeros((), dtype=x.dtype, device=x.device).masked_fill(vocab != 2, -math.inf)
        logp = torch.where(st["finished"].unsqueeze(-1), ended, logp)
    total = (st["scores"].double().unsqueeze(-1) + logp).flatten(1)
    total = torch.where(torch.isnan(total), torch.full_like(total, -math.inf), total)
    best, place = torch.sort(total, dim=1, descending=True, stable=True)
    n = st["case"]["candidates"]
    best, place = best[:, :n], place[:, :n]
    return {"scores": best.float(), "parents": place // x.shape[-1], "tokens": place % x.shape[-1]}


def _plain_reorder(st):
    batch, beams = st["parents"].shape
    source = (torch.arange(batch, device="cuda").unsqueeze(1) * beams + st["parents"]).flatten()
    target = slice(None)
    if st["indices"] is not None:
        target = st["indices"].long()
        source = target[source]
    for t in st["states"]:
        t[target] = t[source]
    return {"states": st["states"]}


def run(st):
    if own:
        return _run_own(st)
    op = st["case"]["op"]
    if op == "update":
        return _plain_update(st)
    if op == "select":
        return _plain_select(st)
    if op == "reorder":
        return _plain_reorder(st)
    return _plain_recurrence(st)


# -------------------------------------------------------------------------- work
def work(case):
    s = _SIZE[case["dtype"]]
    if case["op"] == "select":
        rows = case["batch"] * case["beams"]
        out = case["batch"] * case["candidates"]
        # logits, scores and flags in; scores, parents and tokens out
        return {"bytes": rows * case["vocab"] * s + rows * (4 + int(case["finished"])) + out * 20,
                "flops": 4 * rows * case["vocab"]}
    if case["op"] == "reorder":
        beams, rows = case["beams"], case["batch"] * case["beams"]
        row = case["layers"] * case["dim"] * (3 * s + 4 * case["dstate"])
        # of uniform parents, this share of the beams is another one's child or has children elsewhere
        moved, read = 1 - 1 / beams, 1 - (1 - 1 / beams) ** max(1, beams - 1)
        index = rows * (8 + 4 * int(case["pool"]))
        return {"bytes": rows * row * (moved + read) + index, "flops": 0}
    dim, n, groups, z = case["dim"], case["dstate"], case["groups"], int(case["z"])
    params = 4 * dim * (n + 1 + int(case.get("skip", True)))
    if case["op"] == "update":
        k = case["batch"] * case["tokens"]
        index = 4 * case["batch"] if case["slots"] else 0
        return {"bytes": k * (dim * (3 + z) + 2 * groups * n) * s + 8 * case["batch"] * dim * n + params + index,
                "flops": k * dim * (7 * n + 20)}
    k = case["batch"] * case["seqlen"]
    state = 4 * dim * n * (case["nseq"] or case["batch"]) * {"none": 0, "out": 1, "both": 2}[case["states"]]
    ids = 4 * case["seqlen"] if case["nseq"] else 0
    if case["op"] == "prefill":
        return {"bytes": k * (dim * (3 + z) + 2 * groups * n) * s + params + state + ids, "flops": k * dim * (7 * n + 20)}
    return {"bytes": k * (dim * (6 + 2 * z) + 4 * groups * n) * s + 2 * params + 2 * state + ids,
            "flops": k * dim * (26 * n + 50)}


# ---------------------------------------------------------------- the same in 64 bits
def _softplus64(u):
    return torch.where(u > 0, u + torch.log1p(torch.exp(-u)), torch.log1p(torch.exp(u)))


def _exact_recurrence(st):
    """Step by step through time in 64 bits, forward and then backward."""
    case = st["case"]
    batch, dim, tokens, n, groups = case["batch"], case["dim"], case["seqlen"], case["dstate"], case["groups"]
    nstates = case["nseq"] or batch
    dev, w = st["x"].device, torch.float64

    def seq(t):
        return t.detach().to(w).permute(2, 0, 1).contiguous()

    def coefficients(t):  # (tokens, batch, dim, dstate) on demand, one step at a time
        t = t.detach().to(w)
        return (t.unsqueeze(1) if t.dim() == 3 else t).permute(3, 0, 1, 2).contiguous()

    def spread(t):
        return t.repeat_interleave(dim // groups, 1)

    def gather(t):  # sums over a group's channels
        return t.view(batch, groups, dim // groups, n).sum(2)

    x, u = seq(st["x"]), seq(st["delta"]) + st["bias"].detach().to(w)
    s, A = _softplus64(u), st["A"].detach().to(w)
    B, C = coefficients(st["B"]), coefficients(st["C"])
    skip = st["D"].detach().to(w) if st["D"] is not None else torch.zeros(dim, device=dev, dtype=w)
    init = st["init"].detach().to(w) if st["init"] is not None else torch.zeros(nstates, dim, n, device=dev, dtype=w)
    final = init.clone()
    ids = st["seq_idx"][0].tolist() if st["seq_idx"] is not None else [0] * tokens
    packed = st["seq_idx"] is not None

    def starts(t):
        return t == 0 or ids[t - 1] != ids[t]

    def ends(t):
        return t == tokens - 1 or ids[t + 1] != ids[t]

    def of(states, t):  # the states' rows of the sequences at place t
        return states[ids[t]:ids[t] + 1] if packed else states

    train = case["op"] == "train"
    h = torch.zeros(tokens if train else 1, batch, dim, n, device=dev, dtype=w)
    y = torch.zeros(tokens, batch, dim, device=dev, dtype=w)
    now = None
    for t in range(tokens):
        if ids[t] < 0:
            continue
        if starts(t):
            now = of(init, t)
        now = torch.exp(s[t].unsqueeze(-1) * A) * now + spread(B[t]) * (s[t] * x[t]).unsqueeze(-1)
        y[t] = (now * spread(C[t])).sum(-1) + skip * x[t]
        if train:
            h[t] = now
        if ends(t):
            of(final, t).copy_(now)
    gate = 1.0
    if st["z"] is not None:
        z = seq(st["z"])
        p = 1.0 / (1.0 + torch.exp(-z))
        gate = z * p

    def back(t):
        return t.permute(1, 2, 0)

    res = {"out": back(y * gate)}
    if case["states"] != "none":
        res["final"] = final
    if not train:
        return res
    good = torch.tensor(ids, device=dev).view(-1, 1, 1) >= 0
    dy = seq(st["dout"]) * good
    if st["z"] is not None:
        res["dz"] = back(dy * y * (p + z * p * (1.0 - p)))
        dy = dy * gate
    dfinal = st["dfinal"].to(w) if st["dfinal"] is not None else torch.zeros_like(init)
    dinit = dfinal.clone()
    dx, ds = torch.zeros_like(x), torch.zeros_like(x)
    dA, dB, dC = torch.zeros_like(A), torch.zeros_like(B), torch.zeros_like(C)
    carry = None
    for t in range(tokens - 1, -1, -1):
        if ids[t] < 0:
            continue
        if ends(t):
            carry = of(dfinal, t)
        g = carry + dy[t].unsqueeze(-1) * spread(C[t])
        dC[t] = gather(h[t] * dy[t].unsqueeze(-1))
        dB[t] = gather(g * (s[t] * x[t]).unsqueeze(-1))
        gb = (g * spread(B[t])).sum(-1)
        carry = g * torch.exp(s[t].unsqueeze(-1) * A)
        before = carry * (of(init, t) if starts(t) else h[t - 1])
        dA += (before * s[t].unsqueeze(-1)).sum(0)
        ds[t] = (before * A).sum(-1) + gb * x[t]
        dx[t] = gb * s[t] + skip * dy[t]
        if starts(t):
            of(dinit, t).copy_(carry)
    du = ds / (1.0 + torch.exp(-u))

    def of_group(t, like):
        t = t.permute(1, 2, 3, 0)
        return t if like.dim() == 4 else t.squeeze(1)

    res.update(dx=back(dx), ddelta=back(du), dA=dA, dB=of_group(dB, st["B"]), dC=of_group(dC, st["C"]), dbias=du.sum((0, 1)))
    if st["D"] is not None:
        res["dD"] = (dy * x).sum((0, 1))
    if st["init"] is not None:
        res["dinit"] = dinit
    return res


def _exact_update(st):
    groups = st["case"]["groups"]
    x, delta, z, B, C = (None if st[k] is None else st[k].double() for k in ("x", "delta", "z", "B", "C"))
    one = x.dim() == 2
    if one:
        x, delta, z, B, C = (None if t is None else t[..., None] for t in (x, delta, z, B, C))
    if groups == 1:
        B, C = B.unsqueeze(1), C.unsqueeze(1)
    state = st["state"].double()
    where = st["indices"].long() if st["indices"] is not None else torch.arange(x.shape[0], device=x.device)
    h = state[where]
    per = x.shape[1] // groups
    outs = []
    for t in range(x.shape[2]):
        s = _softplus64(delta[:, :, t] + st["bias"].double())
        h = h * torch.exp(s[:, :, None] * st["A"].double())
        h = h + (s * x[:, :, t])[:, :, None] * B[..., t].repeat_interleave(per, 1)
        y = (h * C[..., t].repeat_interleave(per, 1)).sum(-1) + st["D"].double() * x[:, :, t]
        outs.append(y if z is None else y * z[:, :, t] / (1.0 + torch.exp(-z[:, :, t])))
    state[where] = h
    return {"out": outs[0] if one else torch.stack(outs, -1), "state": state}


def _exact_select(st):
    best = []
    for k in range(st["logits"].shape[0]):  # one request at a time
        logp = torch.log_softmax(st["logits"][k].double(), -1)
        if st["finished"] is not None:
            logp[st["finished"][k]] = -math.inf
            logp[st["finished"][k], 2] = 0.0
        every = (logp + st["scores"][k].double()[:, None]).flatten()
        best.append(torch.topk(every, st["case"]["candidates"]).values)
    return {"scores": torch.stack(best), "parents": None, "tokens": None}


def _exact_reorder(st):
    batch, beams = st["parents"].shape
    place = st["indices"].tolist() if st["indices"] is not None else list(range(batch * beams))
    parents = st["parents"].tolist()
    found = []
    for t in st["states"]:
        new = t.double()
        for b in range(batch):
            for k in range(beams):
                new[place[b * beams + k]] = t[place[b * beams + parents[b][k]]].double()
        found.append(new)
    return {"states": found}


def exact(case, seed):
    st = prepare(case, seed)
    with torch.no_grad():
        if case["op"] == "update":
            return _exact_update(st)
        if case["op"] == "select":
            return _exact_select(st)
        if case["op"] == "reorder":
            return _exact_reorder(st)
        return _exact_recurrence(st)
