"""Cases, plain forms and 64-bit statements of the recurrent-block operators.

Three operators follow the causal convolution in a recurrent language-model block:

* ``gated_recurrence_fn``: a_t = sigmoid(gate_t + gate_bias), h_t = a_t h_{t-1} + (1 - a_t) x_t,
  out_t = h_t silu(z_t), over whole or packed sequences, with its backward pass;
* ``gated_recurrence_update``: the same for a few tokens against states kept in a pool;
* ``dropout_add_rms_norm_fn``: residual_out = residual + dropout(x), stored in the residual's
  type, and out = RMSNorm(residual_out) * weight, with its backward pass; the mask comes from
  Philox4x32-10 and is never stored.

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
def _recurrence(name, op, dtype, batch, dim, seqlen, layout="channel_last", z=True, bias=True, states=True, nseq=0,
                pad=0):
    return {"name": name, "op": op, "dtype": dtype, "batch": batch, "dim": dim, "seqlen": seqlen, "layout": layout,
            "z": z, "bias": bias, "states": states, "nseq": nseq, "pad": pad}


def _update(name, dtype, batch, dim, tokens, slots, z=True, bias=True):
    return {"name": name, "op": "update", "dtype": dtype, "batch": batch, "dim": dim, "tokens": tokens, "slots": slots,
            "z": z, "bias": bias}


def _norm(name, op, dtype, rows, dim, p, residual, weight="float32"):
    return {"name": name, "op": op, "dtype": dtype, "rows": rows, "dim": dim, "p": p, "residual": residual,
            "weight": weight}


def listed():
    return [
        # A training step of one layer: 4 sequences of 2048 tokens, states carried in and out.
        _recurrence("train_4x4096x2048", "train", "bfloat16", 4, 4096, 2048),
        # A training step on 32 packed documents of different lengths.
        _recurrence("train_packed_5120x65536", "train", "float16", 1, 5120, 65536, states=False, nseq=32, pad=96),
        # (batch, dim, seqlen) contiguous, odd sizes, 32-bit, without an output gate.
        _recurrence("train_rows_3x770x1027", "train", "float32", 3, 770, 1027, layout="rows", z=False),
        # The largest training step: 8 sequences of 8192 tokens.
        _recurrence("train_8x4096x8192", "train", "bfloat16", 8, 4096, 8192, states=False),
        # Serving: the prompts of 8 requests, packed; their states go to the decode steps.
        _recurrence("prefill_packed_8192x32768", "prefill", "bfloat16", 1, 8192, 32768, nseq=8),
        # Serving: two short prompts.
        _recurrence("prefill_rows_2x1000x77", "prefill", "float16", 2, 1000, 77, layout="rows"),
        # Decoding one request, one token: latency.
        _update("update_1x4096", "bfloat16", 1, 4096, 1, 0),
        # Decoding 128 requests whose states lie scattered in a pool of 160.
        _update("update_128x8192_pool", "bfloat16", 128, 8192, 1, 160),
        # The block's residual connection in training, residual stream in 32 bits.
        _norm("norm_train_8192x4096", "norm_train", "bfloat16", 8192, 4096, 0.1, "float32"),
        # Odd sizes, residual stream in 16 bits.
        _norm("norm_train_999x1001", "norm_train", "float16", 999, 1001, 0.2, "float16", "float16"),
        # Decoding one token: no dropout.
        _norm("norm_1x4096", "norm", "bfloat16", 1, 4096, 0.0, "float32"),
        # The largest: 65536 tokens, all in 16 bits.
        _norm("norm_train_65536x4096", "norm_train", "bfloat16", 65536, 4096, 0.1, "bfloat16", "bfloat16"),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["train", "train", "train", "prefill", "update", "norm_train", "norm"])
    dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
    if op == "update":
        batch = _spread(rng, 1, 256)
        return {"op": op, "dtype": dtype, "batch": batch, "dim": _spread(rng, 256, 8192), "tokens": rng.choice([1, 1, 1, 2, 4]),
                "slots": rng.choice([0, batch, batch + rng.randint(1, 64)]), "z": rng.random() < 0.7, "bias": rng.random() < 0.7}
    if op in ("norm", "norm_train"):
        dim = _spread(rng, 64, 8192)
        rows = min(_spread(rng, 1, 65536), (1 << 27) // dim)
        return {"op": op, "dtype": dtype, "rows": rows, "dim": dim, "p": rng.choice([0.0, 0.1, 0.25]) if op == "norm_train" else 0.0,
                "residual": rng.choice([dtype, "float32"]), "weight": rng.choice([dtype, "float32"])}
    dim = _spread(rng, 64, 8192)
    packed = rng.random() < 0.35
    seqlen = _spread(rng, 64 if packed else 1, 32768)
    batch = 1 if packed else max(1, min(_spread(rng, 1, 16), (1 << 27) // (dim * seqlen)))
    seqlen = min(seqlen, (1 << 27) // (dim * batch))
    return {"op": op, "dtype": dtype, "batch": batch, "dim": dim, "seqlen": seqlen,
            "layout": rng.choice(["channel_last", "channel_last", "rows"]), "z": rng.random() < 0.7, "bias": rng.random() < 0.7,
            "states": rng.random() < 0.6, "nseq": rng.randint(1, 24) if packed else 0, "pad": rng.choice([0, 17]) if packed else 0}


# --------------------------------------------------------------------------- inputs
def _packing(seqlen, nseq, pad, gen):
    """Ids of ``nseq`` packed sequences of random lengths (some may be empty), then -1 padding."""
    end = max(1, seqlen - pad)
    cuts = torch.sort(torch.randint(0, end + 1, (nseq - 1,), generator=gen, device="cuda")).values
    pos = torch.arange(seqlen, device="cuda")
    ids = torch.searchsorted(cuts, pos, right=True)
    return torch.where(pos < end, ids, torch.full_like(ids, -1)).to(torch.int32).unsqueeze(0)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, scale=1.0, dtype=torch.float32):
        return torch.randn(*shape, generator=gen, device="cuda", dtype=dtype).mul_(scale)

    dt = _DT[case["dtype"]]
    st = {"case": dict(case)}
    if case["op"] in ("norm", "norm_train"):
        rows, dim = case["rows"], case["dim"]
        st["x"] = normal(rows, dim, dtype=dt)
        st["residual"] = normal(rows, dim, scale=2.0, dtype=_DT[case["residual"]])
        st["weight"] = (1.0 + normal(dim, scale=0.1)).to(_DT[case["weight"]])
        # the generator's state of this layer's call: a seed and an offset
        st["rng"] = torch.randint(0, 1 << 62, (2,), generator=gen, device="cuda", dtype=torch.int64) if case["p"] else None
        if case["op"] == "norm_train":
            st["dout"] = normal(rows, dim, dtype=dt)
            st["dresidual_out"] = normal(rows, dim, dtype=_DT[case["residual"]])
            for n in ("x", "residual", "weight"):
                st[n].requires_grad_()
        return st
    batch, dim = case["batch"], case["dim"]
    tokens = case["tokens"] if case["op"] == "update" else case["seqlen"]
    rows = case.get("layout") == "rows"

    def sequence(scale=1.0):
        if rows:
            return normal(batch, dim, tokens, scale=scale, dtype=dt)
        return normal(batch, tokens, dim, scale=scale, dtype=dt).transpose(1, 2)

    st["x"] = sequence()
    st["gate"] = sequence(1.5)
    st["z"] = sequence() if case["z"] else None
    # decay rates from one half to about 0.98, as such gates are initialised
    st["bias"] = torch.rand(dim, generator=gen, device="cuda") * 4.0 if case["bias"] else None
    if case["op"] == "update":
        pool = case["slots"] or batch
        st["state"] = normal(pool, dim, scale=0.5)
        st["indices"] = torch.randperm(pool, generator=gen, device="cuda")[:batch].to(torch.int32) if case["slots"] else None
        if tokens == 1:
            for n in ("x", "gate", "z"):
                st[n] = None if st[n] is None else st[n].squeeze(-1)
        return st
    nstates = case["nseq"] or batch
    st["seq_idx"] = _packing(tokens, case["nseq"], case["pad"], gen) if case["nseq"] else None
    st["init"] = normal(nstates, dim, scale=0.5) if case["states"] else None
    if case["op"] == "train":
        st["dout"] = sequence()
        st["dfinal"] = normal(nstates, dim) if case["states"] else None
        for n in ("x", "gate", "z", "bias", "init"):
            if st[n] is not None:
                st[n].requires_grad_()
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
    if case["op"] == "update":
        out = cc.gated_recurrence_update(st["x"], st["state"], st["gate"], st["z"], st["bias"], state_indices=st["indices"])
        return {"out": out, "state": st["state"]}
    if case["op"] == "norm":
        with torch.no_grad():
            out, res = cc.dropout_add_rms_norm_fn(st["x"], st["weight"], st["residual"])
        return {"out": out, "residual_out": res}
    if case["op"] == "norm_train":
        out, res = cc.dropout_add_rms_norm_fn(st["x"], st["weight"], st["residual"], dropout_p=case["p"], rng_state=st["rng"])
        dx, dres, dw = torch.autograd.grad((out, res), (st["x"], st["residual"], st["weight"]), (st["dout"], st["dresidual_out"]))
        return {"out": out, "residual_out": res, "dx": dx, "dresidual": dres, "dweight": dw}
    kept = bool(case["states"])
    if case["op"] == "prefill":
        with torch.no_grad():
            got = cc.gated_recurrence_fn(st["x"], st["gate"], st["z"], st["bias"], seq_idx=st["seq_idx"],
                                         initial_states=st["init"], return_final_states=kept)
        return {"out": got[0], "final": got[1]} if kept else {"out": got}
    got = cc.gated_recurrence_fn(st["x"], st["gate"], st["z"], st["bias"], seq_idx=st["seq_idx"], initial_states=st["init"],
                                 return_final_states=kept)
    names = [n for n in ("x", "gate", "z", "bias", "init") if st[n] is not None]
    outs, grads = (got, (st["dout"], st["dfinal"])) if kept else ((got,), (st["dout"],))
    found = torch.autograd.grad(outs, [st[n] for n in names], grads)
    res = {"out": outs[0], **({"final": outs[1]} if kept else {})}
    res.update({"d" + n: g for n, g in zip(names, found)})
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
    """(valid, first, last) of each place, as (tokens, batch, 1) truth values, and the row of
    the states that its sequence has."""
    x = st["x"]
    batch = x.shape[0]
    ids = st["seq_idx"]
    if ids is None:
        ids = torch.arange(batch, device=x.device).unsqueeze(1).expand(batch, tokens)
    ids = ids.long().t()
    none = torch.full_like(ids[:1], -1)
    valid = ids >= 0
    first = valid & (ids != torch.cat([none, ids[:-1]]))
    last = valid & (ids != torch.cat([ids[1:], none]))
    return valid.unsqueeze(-1), first.unsqueeze(-1), last.unsqueeze(-1), ids.clamp(min=0)


def _time_first(t):
    return t.detach().permute(2, 0, 1).float()


def _as_input(t, like):
    """(tokens, batch, dim) results in the type and layout of an input."""
    if like.stride(1) == 1:
        return t.permute(1, 0, 2).to(like.dtype, memory_format=torch.contiguous_format).transpose(1, 2)
    return t.permute(1, 2, 0).to(like.dtype, memory_format=torch.contiguous_format)


def _plain_recurrence(st):
    case = st["case"]
    tokens, dim = case["seqlen"], case["dim"]
    x, gate = _time_first(st["x"]), _time_first(st["gate"])
    valid, first, last, rows = _edges(st, tokens)
    nstates = case["nseq"] or case["batch"]
    init = st["init"].detach() if case["states"] else torch.zeros(nstates, dim, device=x.device)
    if st["bias"] is not None:
        gate = gate + st["bias"].detach()
    a, c = torch.sigmoid(gate), torch.sigmoid(-gate)
    zero = torch.zeros((), device=x.device)
    # h_{t-1} at a sequence's first place is its initial state
    b = torch.where(valid, c * x, zero)
    if case["states"]:
        b = torch.where(first, torch.addcmul(b, a, init[rows]), b)
    h = _scan(torch.where(first | ~valid, zero, a), b)
    out = h
    if st["z"] is not None:
        z = _time_first(st["z"])
        sz = torch.sigmoid(z)
        out = h * (z * sz)
    out = torch.where(valid, out, zero)
    res = {"out": _as_input(out, st["x"])}
    at = last.squeeze(-1)
    if case["states"]:
        final = init.clone()
        final[rows[at]] = h[at]
        res["final"] = final
    if case["op"] == "prefill":
        return res
    dy = _time_first(st["dout"])
    dh = dy
    if st["z"] is not None:
        dh = dy * (z * sz)
        dz = torch.where(valid, dy * h * (sz * (1 + z * (1 - sz))), zero)
        del z, sz
    dh = torch.where(valid, dh, zero)
    if case["states"]:
        dh = torch.where(last, dh + st["dfinal"][rows], dh)
    # g_t = dh_t + a_{t+1} g_{t+1} within a sequence, from its last place back
    nxt = torch.cat([a[1:], torch.zeros_like(a[:1])])
    g = _scan(torch.where(last | ~valid, zero, nxt).flip(0), dh.flip(0)).flip(0)
    del nxt, dh
    prev = torch.cat([torch.zeros_like(h[:1]), h[:-1]])
    prev = torch.where(first, init[rows] if case["states"] else zero, prev)
    dgate = torch.where(valid, g * (prev - x) * (a * c), zero)
    res["dx"] = _as_input(torch.where(valid, g * c, zero), st["x"])
    res["dgate"] = _as_input(dgate, st["gate"])
    if st["z"] is not None:
        res["dz"] = _as_input(dz, st["z"])
    if st["bias"] is not None:
        res["dbias"] = dgate.sum((0, 1))
    if case["states"]:
        dinit = st["dfinal"].clone()  # a sequence without tokens hands its state through
        at = first.squeeze(-1)
        dinit[rows[at]] = (a * g)[at]
        res["dinit"] = dinit
    return res


def _plain_update(st):
    x, gate, z = st["x"], st["gate"], st["z"]
    flat = x.dim() == 2
    if flat:
        x, gate, z = x.unsqueeze(-1), gate.unsqueeze(-1), None if z is None else z.unsqueeze(-1)
    x, gate = x.permute(2, 0, 1).float(), gate.permute(2, 0, 1).float()
    if st["bias"] is not None:
        gate = gate + st["bias"]
    a = torch.sigmoid(gate)
    b = torch.sigmoid(-gate) * x
    rows = st["indices"].long() if st["indices"] is not None else slice(None)
    b[0] = torch.addcmul(b[0], a[0], st["state"][rows])
    h = _scan(a, b)
    st["state"][rows] = h[-1]
    out = h
    if z is not None:
        zf = z.permute(2, 0, 1).float()
        out = h * (zf * torch.sigmoid(zf))
    out = out.permute(1, 2, 0)
    return {"out": (out.squeeze(-1) if flat else out).to(st["x"].dtype), "state": st["state"]}


_LOW = 0xFFFFFFFF


def _philox(key, counter):
    """Philox4x32-10 of a (seed, offset) key and a tensor of block numbers: four 32-bit words
    for each block, held in 64-bit integers (products wrap, their halves stay right)."""
    c0, c1 = counter & _LOW, (counter >> 32) & _LOW
    c2, c3 = key[1] & _LOW, (key[1] >> 32) & _LOW
    k0, k1 = key[0] & _LOW, (key[0] >> 32) & _LOW
    for _ in range(10):
        p0, p1 = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = (p1 >> 32 & _LOW) ^ c1 ^ k0, p1 & _LOW, (p0 >> 32 & _LOW) ^ c3 ^ k1, p0 & _LOW
        k0, k1 = (k0 + 0x9E3779B9) & _LOW, (k1 + 0xBB67AE85) & _LOW
    return c0, c1, c2, c3


def _keep(rng, rows, dim, p):
    """The dropout mask: element (row, col) takes word col % 4 of block
    row * ceil(dim / 4) + col // 4 and is kept if that word is at least p * 2^32."""
    per = (dim + 3) // 4
    words = torch.stack(_philox(rng, torch.arange(rows * per, device=rng.device)), -1)
    return words.view(rows, per * 4)[:, :dim] >= int(p * 4294967296.0)


def _plain_norm(st, eps=1e-5):
    case = st["case"]
    x, res = st["x"].detach().float(), st["residual"].detach().float()
    w = st["weight"].detach().float()
    p = case["p"]
    if p:
        scale = _keep(st["rng"], case["rows"], case["dim"], p).float() * (1.0 / (1.0 - p))
        x = x * scale
    stored = (res + x).to(st["residual"].dtype)
    r = stored.float()
    rstd = torch.rsqrt((r * r).mean(-1, keepdim=True) + eps)
    n = r * rstd
    got = {"out": (n * w).to(st["x"].dtype), "residual_out": stored}
    if case["op"] == "norm":
        return got
    dy = st["dout"].float()
    dn = dy * w
    dr = st["dresidual_out"].float() + rstd * (dn - n * (dn * n).mean(-1, keepdim=True))
    got["dx"] = (dr * scale if p else dr).to(st["x"].dtype)
    got["dresidual"] = dr.to(st["residual"].dtype)
    got["dweight"] = (dy * n).sum(0).to(st["weight"].dtype)
    return got


def run(st):
    if own:
        return _run_own(st)
    op = st["case"]["op"]
    if op == "update":
        return _plain_update(st)
    if op in ("norm", "norm_train"):
        return _plain_norm(st)
    return _plain_recurrence(st)


# -------------------------------------------------------------------------- work
def work(case):
    s = _SIZE[case["dtype"]]
    if case["op"] in ("norm", "norm_train"):
        n, rs, ws = case["rows"] * case["dim"], _SIZE[case["residual"]], _SIZE[case["weight"]]
        if case["op"] == "norm":
            return {"bytes": n * (2 * s + 2 * rs) + case["dim"] * ws, "flops": 6 * n}
        return {"bytes": n * (4 * s + 4 * rs) + 2 * case["dim"] * ws, "flops": 18 * n}
    z = int(case["z"])
    bias = 4 * case["dim"] * int(case["bias"])
    if case["op"] == "update":
        n = case["batch"] * case["dim"]
        index = 4 * case["batch"] if case["slots"] else 0
        return {"bytes": n * case["tokens"] * (3 + z) * s + 8 * n + bias + index, "flops": n * case["tokens"] * (8 + 5 * z)}
    n = case["batch"] * case["dim"] * case["seqlen"]
    state = 4 * case["dim"] * (case["nseq"] or case["batch"]) * int(case["states"])
    ids = 4 * case["seqlen"] if case["nseq"] else 0
    if case["op"] == "prefill":
        return {"bytes": n * (3 + z) * s + bias + ids + 2 * state, "flops": n * (8 + 5 * z)}
    return {"bytes": n * (6 + 2 * z) * s + 2 * bias + ids + 4 * state, "flops": n * (24 + 17 * z)}


# ---------------------------------------------------------------- the same in 64 bits
def _exact_recurrence(st):
    """Step by step through time in 64 bits, forward and then backward."""
    case = st["case"]
    batch, dim, tokens = case["batch"], case["dim"], case["seqlen"]
    dev = st["x"].device
    nstates = case["nseq"] or batch
    wide = torch.float64

    def seq(t):
        return t.detach().permute(2, 0, 1).to(wide).contiguous()

    ids = st["seq_idx"].cpu().tolist() if st["seq_idx"] is not None else [[b] * tokens for b in range(batch)]
    per_batch = st["seq_idx"] is not None
    x, u = seq(st["x"]), seq(st["gate"])
    if st["bias"] is not None:
        u += st["bias"].detach().to(wide)
    a = 1.0 / (1.0 + torch.exp(-u))
    keep_less = 1.0 / (1.0 + torch.exp(u))  # 1 - a
    del u
    init = st["init"].detach().to(wide) if case["states"] else torch.zeros(nstates, dim, device=dev, dtype=wide)
    final = init.clone()
    h = torch.zeros(tokens, batch, dim, device=dev, dtype=wide)
    if per_batch:  # one row of packed sequences
        row = ids[0]
        for t in range(tokens):
            if row[t] < 0:
                continue
            before = init[row[t]] if t == 0 or row[t - 1] != row[t] else h[t - 1, 0]
            h[t, 0] = a[t, 0] * before + keep_less[t, 0] * x[t, 0]
            if t == tokens - 1 or row[t + 1] != row[t]:
                final[row[t]] = h[t, 0]
    else:
        now = init
        for t in range(tokens):
            now = a[t] * now + keep_less[t] * x[t]
            h[t] = now
        final = now
    silu = 1.0
    if st["z"] is not None:
        z = seq(st["z"])
        s = 1.0 / (1.0 + torch.exp(-z))
        silu = z * s
    good = torch.tensor(ids, device=dev).t().unsqueeze(-1) >= 0

    def back(t):
        return t.permute(1, 2, 0)

    res = {"out": back(h * silu * good)}
    if case["states"]:
        res["final"] = final
    if case["op"] == "prefill":
        return res
    dy = seq(st["dout"]) * good
    if st["z"] is not None:
        res["dz"] = back(dy * h * (s + z * s * (1.0 - s)))
        dy = dy * silu
        del z, s
    del silu
    dfinal = st["dfinal"].to(wide) if case["states"] else torch.zeros_like(init)
    dinit = dfinal.clone()
    dx = torch.zeros_like(h)
    du = torch.zeros_like(h)
    carry = dfinal if not per_batch else None
    for t in range(tokens - 1, -1, -1):
        if per_batch:
            k = ids[0][t]
            if k < 0:
                continue
            if t == tokens - 1 or ids[0][t + 1] != k:
                carry = dfinal[k]
            start = t == 0 or ids[0][t - 1] != k
            before = init[k] if start else h[t - 1, 0]
        else:
            start = t == 0
            before = init if start else h[t - 1]
        g = dy[t] + carry
        dx[t] = g * keep_less[t]
        du[t] = g * (before - x[t]) * a[t] * keep_less[t]
        carry = a[t] * g
        if start:
            if per_batch:
                dinit[k] = carry[0]
                carry = None
            else:
                dinit = carry
    res["dx"], res["dgate"] = back(dx), back(du)
    if st["bias"] is not None:
        res["dbias"] = du.sum((0, 1))
    if case["states"]:
        res["dinit"] = dinit
    return {k: res[k] for k in ("out", "final", "dx", "dgate", "dz", "dbias", "dinit") if k in res}


def _exact_update(st):
    x, gate, z = (None if st[k] is None else st[k].double() for k in ("x", "gate", "z"))
    if x.dim() == 2:
        x, gate, z = x[..., None], gate[..., None], None if z is None else z[..., None]
    state = st["state"].double()
    where = st["indices"].long() if st["indices"] is not None else torch.arange(x.shape[0], device=x.device)
    h = state[where]
    outs = []
    for t in range(x.shape[2]):
        u = gate[:, :, t] + (st["bias"].double() if st["bias"] is not None else 0.0)
        h = h / (1.0 + torch.exp(-u)) + x[:, :, t] / (1.0 + torch.exp(u))
        outs.append(h if z is None else h * z[:, :, t] / (1.0 + torch.exp(-z[:, :, t])))
    state[where] = h
    out = torch.stack(outs, -1)
    return {"out": out.squeeze(-1) if st["x"].dim() == 2 else out, "state": state}


def _exact_mask(rng, rows, dim, p):
    """The mask's words from 16-bit partial products, one row block at a time."""
    seed, offset = (int(v) for v in rng.tolist())
    per = -(-dim // 4)
    block = torch.arange(rows * per, device=rng.device, dtype=torch.int64)

    def halves(v, m):  # high and low 32 bits of v * m
        lo, hi = v & 0xFFFF, v >> 16
        part0, part1 = lo * m, hi * m
        mid = (part0 >> 16) + (part1 & 0xFFFF)
        return ((part1 >> 16) + (mid >> 16)) & _LOW, ((mid & 0xFFFF) << 16) | (part0 & 0xFFFF)

    c = [block & _LOW, block >> 32, torch.full_like(block, offset & _LOW), torch.full_like(block, (offset >> 32) & _LOW)]
    for r in range(10):
        key0 = ((seed & _LOW) + r * 0x9E3779B9) & _LOW
        key1 = (((seed >> 32) & _LOW) + r * 0xBB67AE85) & _LOW
        h0, l0 = halves(c[0], 0xD2511F53)
        h1, l1 = halves(c[2], 0xCD9E8D57)
        c = [h1 ^ c[1] ^ key0, l1, h0 ^ c[3] ^ key1, l0]
    return (torch.stack(c, 1).reshape(rows, 4 * per)[:, :dim] >= int(p * 2.0 ** 32)).double()


def _exact_norm(st, eps=1e-5):
    case = st["case"]
    n, d, p = case["rows"], case["dim"], case["p"]
    m = _exact_mask(st["rng"], n, d, p) / (1.0 - p) if p else None
    x = st["x"].detach().double()
    total = st["residual"].detach().double() + (x * m if p else x)
    # what is normalised is the residual stream as it is stored
    stored = total.to(st["residual"].dtype).double()
    w = st["weight"].detach().double()
    inv = 1.0 / torch.sqrt((stored ** 2).sum(1, keepdim=True) / d + eps)
    res = {"out": stored * inv * w, "residual_out": total}
    if case["op"] == "norm":
        return res
    dy = st["dout"].double()
    inner = (dy * w * stored).sum(1, keepdim=True) * inv ** 3 / d
    dr = st["dresidual_out"].double() + dy * w * inv - stored * inner
    res["dx"] = dr * m if p else dr
    res["dresidual"] = dr
    res["dweight"] = (dy * stored * inv).sum(0)
    return res


def exact(case, seed):
    st = prepare(case, seed)
    with torch.no_grad():
        if case["op"] == "update":
            return _exact_update(st)
        if case["op"] in ("norm", "norm_train"):
            return _exact_norm(st)
        return _exact_recurrence(st)
