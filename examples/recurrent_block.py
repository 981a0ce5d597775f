"""A small recurrent language model on the package's operators: trained, then served.

Each layer is

    out, residual = dropout_add_rms_norm_fn(hidden, norm, residual, dropout_p=p)
    x, gate, z    = out @ in_proj                    (channel-last, strided slices of one projection)
    x             = causal_conv1d_fn(x, conv)        (SiLU)
    y             = gated_recurrence_fn(x, gate, z)  (h_t = a_t h_{t-1} + (1 - a_t) x_t, y = h silu(z))
    hidden        = y @ out_proj

or, with ``--block selective``, its state-space form

    x, z          = out @ in_proj
    x             = causal_conv1d_fn(x, conv)
    delta, B, C   = x @ x_proj                       (delta of low rank, then @ delta_proj)
    y             = selective_recurrence_fn(x, delta, A, B, C, D, z)

Training packs several sequences into one row (``seq_idx``).  Serving runs the packed prompts
once, takes the states of the convolution and of the recurrence from that pass, and decodes
token by token against them; with ``--beams`` it also continues a prompt by beam search, whose
chosen beams the states follow.

    python examples/recurrent_block.py [--steps 100] [--dim 256] [--layers 2] [--block selective] [--beams 4]

The task is to repeat the token seen ``LAG`` places before; the script prints the loss and the
share of right answers, and checks the decoded logits against a whole pass.
"""

from __future__ import annotations

import argparse
import math
import os
import sys

import torch
import torch.nn.functional as F

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, "cute-causal-conv1d_b200"))

from causal_conv1d import (  # noqa: E402
    beam_search_reorder,
    beam_search_select,
    causal_conv1d_fn,
    causal_conv1d_update,
    dropout_add_rms_norm_fn,
    gated_recurrence_fn,
    gated_recurrence_update,
    selective_recurrence_fn,
    selective_recurrence_update,
)
from causal_conv1d.causal_conv1d_varlen import causal_conv1d_fn_varlen_states  # noqa: E402

WIDTH, LAG = 4, 3


class Layer(torch.nn.Module):
    def __init__(self, dim, inner, dtype, device):
        super().__init__()
        kw = {"device": device, "dtype": dtype}
        self.norm = torch.nn.Parameter(torch.ones(dim, device=device))
        self.in_proj = torch.nn.Linear(dim, 3 * inner, bias=False, **kw)
        self.conv = torch.nn.Parameter(torch.randn(inner, WIDTH, device=device) * 0.5)
        self.conv_bias = torch.nn.Parameter(torch.zeros(inner, device=device))
        self.gate_bias = torch.nn.Parameter(torch.linspace(-1.0, 4.0, inner, device=device))  # fast and slow channels
        self.out_proj = torch.nn.Linear(inner, dim, bias=False, **kw)
        self.inner = inner

    def split(self, out):
        """(batch, tokens, dim) -> x, gate, z as (batch, inner, tokens) views of one projection."""
        return self.in_proj(out).transpose(1, 2).split(self.inner, 1)

    def forward(self, hidden, residual, seq_idx, p):
        out, residual = dropout_add_rms_norm_fn(hidden, self.norm, residual, dropout_p=p, residual_in_fp32=True)
        x, gate, z = self.split(out)
        x = causal_conv1d_fn(x, self.conv, self.conv_bias, seq_idx=seq_idx, activation="silu")
        y = gated_recurrence_fn(x, gate, z, self.gate_bias, seq_idx=seq_idx)
        return self.out_proj(y.transpose(1, 2)), residual

    def prefill(self, hidden, residual, seq_idx, cu_seqlens):
        """Packed prompts in one row; also returns the states that decoding starts from."""
        out, residual = dropout_add_rms_norm_fn(hidden, self.norm, residual, residual_in_fp32=True)
        x, gate, z = self.split(out)
        x, conv_state = causal_conv1d_fn_varlen_states(x, self.conv, cu_seqlens, WIDTH - 1, self.conv_bias, seq_idx, "silu")
        y, state = gated_recurrence_fn(x, gate, z, self.gate_bias, seq_idx=seq_idx, return_final_states=True,
                                       num_sequences=cu_seqlens.numel() - 1)
        return self.out_proj(y.transpose(1, 2)), residual, (conv_state, state)

    def step(self, hidden, residual, states):
        """One token of each sequence: hidden (batch, dim); the states are updated in place."""
        conv_state, state = states
        out, residual = dropout_add_rms_norm_fn(hidden, self.norm, residual, residual_in_fp32=True)
        x, gate, z = self.in_proj(out).split(self.inner, 1)
        x = causal_conv1d_update(x.contiguous(), conv_state, self.conv, self.conv_bias, "silu")
        y = gated_recurrence_update(x, state, gate, z, self.gate_bias)
        return self.out_proj(y), residual


class SelectiveLayer(torch.nn.Module):
    """The same block around the selective recurrence."""

    def __init__(self, dim, inner, dtype, device, dstate=16):
        super().__init__()
        kw = {"device": device, "dtype": dtype}
        self.norm = torch.nn.Parameter(torch.ones(dim, device=device))
        self.in_proj = torch.nn.Linear(dim, 2 * inner, bias=False, **kw)
        self.conv = torch.nn.Parameter(torch.randn(inner, WIDTH, device=device) * 0.5)
        self.conv_bias = torch.nn.Parameter(torch.zeros(inner, device=device))
        self.inner, self.rank, self.dstate = inner, max(1, dim // 16), dstate
        self.x_proj = torch.nn.Linear(inner, self.rank + 2 * dstate, bias=False, **kw)
        self.delta_proj = torch.nn.Linear(self.rank, inner, bias=False, **kw)
        # steps of 0.001 to 0.1 through softplus, decay rates of 1 to dstate
        step = torch.exp(torch.linspace(math.log(1e-3), math.log(0.1), inner, device=device))
        self.delta_bias = torch.nn.Parameter(step + torch.log(-torch.expm1(-step)))
        rates = torch.arange(1, dstate + 1, device=device, dtype=torch.float32)
        self.log_rates = torch.nn.Parameter(torch.log(rates).repeat(inner, 1))
        self.skip = torch.nn.Parameter(torch.ones(inner, device=device))
        self.out_proj = torch.nn.Linear(inner, dim, bias=False, **kw)

    def split(self, out):
        return self.in_proj(out).transpose(1, 2).split(self.inner, 1)

    def coefficients(self, x):
        """(..., inner) -> delta (..., inner), B and C (..., dstate)."""
        low, B, C = self.x_proj(x).split([self.rank, self.dstate, self.dstate], -1)
        return self.delta_proj(low), B, C

    def scan(self, x, z, **kw):
        delta, B, C = (t.transpose(1, 2) for t in self.coefficients(x.transpose(1, 2)))
        return selective_recurrence_fn(x, delta, -torch.exp(self.log_rates), B, C, self.skip, z, self.delta_bias, **kw)

    def forward(self, hidden, residual, seq_idx, p):
        out, residual = dropout_add_rms_norm_fn(hidden, self.norm, residual, dropout_p=p, residual_in_fp32=True)
        x, z = self.split(out)
        x = causal_conv1d_fn(x, self.conv, self.conv_bias, seq_idx=seq_idx, activation="silu")
        y = self.scan(x, z, seq_idx=seq_idx)
        return self.out_proj(y.transpose(1, 2)), residual

    def prefill(self, hidden, residual, seq_idx, cu_seqlens):
        out, residual = dropout_add_rms_norm_fn(hidden, self.norm, residual, residual_in_fp32=True)
        x, z = self.split(out)
        x, conv_state = causal_conv1d_fn_varlen_states(x, self.conv, cu_seqlens, WIDTH - 1, self.conv_bias, seq_idx, "silu")
        y, state = self.scan(x, z, seq_idx=seq_idx, return_final_states=True, num_sequences=cu_seqlens.numel() - 1)
        return self.out_proj(y.transpose(1, 2)), residual, (conv_state, state)

    def step(self, hidden, residual, states):
        conv_state, state = states
        out, residual = dropout_add_rms_norm_fn(hidden, self.norm, residual, residual_in_fp32=True)
        x, z = self.in_proj(out).split(self.inner, 1)
        x = causal_conv1d_update(x.contiguous(), conv_state, self.conv, self.conv_bias, "silu")
        delta, B, C = self.coefficients(x)
        y = selective_recurrence_update(x, state, delta, -torch.exp(self.log_rates), B, C, self.skip, z, self.delta_bias)
        return self.out_proj(y), residual


class Model(torch.nn.Module):
    def __init__(self, vocab, dim, layers, dtype=torch.bfloat16, device="cuda", layer=Layer):
        super().__init__()
        self.embed = torch.nn.Embedding(vocab, dim, device=device, dtype=dtype)
        self.layers = torch.nn.ModuleList(layer(dim, 2 * dim, dtype, device) for _ in range(layers))
        self.norm = torch.nn.Parameter(torch.ones(dim, device=device))
        self.head = torch.nn.Linear(dim, vocab, bias=False, device=device, dtype=dtype)

    def logits(self, hidden, residual):
        return self.head(dropout_add_rms_norm_fn(hidden, self.norm, residual)[0]).float()

    def forward(self, tokens, seq_idx=None, p=0.0):
        hidden, residual = self.embed(tokens), None
        for layer in self.layers:
            hidden, residual = layer(hidden, residual, seq_idx, p)
        return self.logits(hidden, residual)

    @torch.no_grad()
    def prefill(self, tokens, seq_idx, cu_seqlens):
        hidden, residual, states = self.embed(tokens), None, []
        for layer in self.layers:
            hidden, residual, s = layer.prefill(hidden, residual, seq_idx, cu_seqlens)
            states.append(s)
        return self.logits(hidden, residual), states

    @torch.no_grad()
    def step(self, tokens, states):
        hidden, residual = self.embed(tokens), None
        for layer, s in zip(self.layers, states):
            hidden, residual = layer.step(hidden, residual, s)
        return self.logits(hidden, residual)


def packed_batch(gen, vocab, lengths):
    """One row of packed sequences: tokens, seq_idx, targets (-100 where there is nothing to repeat)."""
    total = sum(lengths)
    tokens = torch.randint(0, vocab, (1, total), generator=gen, device="cuda")
    targets = torch.full((1, total), -100, device="cuda")
    ids = torch.empty(1, total, dtype=torch.int32, device="cuda")
    at = 0
    for k, n in enumerate(lengths):
        ids[0, at:at + n] = k
        targets[0, at + LAG:at + n] = tokens[0, at:at + n - LAG]
        at += n
    return tokens, ids, targets


def train(model, steps, vocab, gen, p=0.1, log=print):
    opt = torch.optim.AdamW(model.parameters(), lr=2e-3)
    losses = []
    for step in range(steps):
        tokens, ids, targets = packed_batch(gen, vocab, [300, 40, 500, 7, 177])
        logits = model(tokens, ids, p)
        loss = F.cross_entropy(logits.view(-1, vocab), targets.view(-1), ignore_index=-100)
        opt.zero_grad(set_to_none=True)
        loss.backward()
        opt.step()
        losses.append(loss.item())
        if log and (step % 20 == 0 or step == steps - 1):
            right = (logits.argmax(-1) == targets)[targets >= 0].float().mean().item()
            log(f"step {step}: loss {losses[-1]:.3f}, right {right:.2f}")
    return losses


@torch.no_grad()
def serve(model, vocab, gen, prompts=(37, 5, 64), new=8):
    """Prefill, then `new` forced tokens each; returns the largest difference between the decoded
    logits and those of a whole pass over prompt and new tokens, and their largest value."""
    tokens, ids, _ = packed_batch(gen, vocab, list(prompts))
    cu = torch.tensor([0, *torch.tensor(prompts).cumsum(0).tolist()], device="cuda", dtype=torch.int32)
    extra = torch.randint(0, vocab, (len(prompts), new), generator=gen, device="cuda")
    _, states = model.prefill(tokens, ids, cu)
    got = torch.stack([model.step(extra[:, i], states) for i in range(new)], 1)
    rows = [torch.cat([tokens[0, cu[k]:cu[k + 1]], extra[k]]) for k in range(len(prompts))]
    want = torch.stack([model(r[None])[0, -new:] for r in rows])
    return (got - want).abs().max().item(), want.abs().max().item()


@torch.no_grad()
def beam_search(model, tokens, beams, new, end_token):
    """Continues each prompt of tokens (batch, length) by up to `new` tokens.  Returns the beams'
    tokens (batch, beams, new) and their log-probabilities, the best first."""
    batch, length = tokens.shape
    ids = torch.arange(batch, device="cuda", dtype=torch.int32).repeat_interleave(length).unsqueeze(0)
    cu = torch.arange(0, batch * length + 1, length, device="cuda", dtype=torch.int32)
    logits, states = model.prefill(tokens.reshape(1, -1), ids, cu)
    states = [tuple(t.repeat_interleave(beams, 0) for t in s) for s in states]
    # a prompt's beams are alike at first: one of them is in use
    logits = logits.view(batch, length, -1)[:, -1:].expand(-1, beams, -1)
    scores = torch.full((batch, beams), -math.inf, device="cuda")
    scores[:, 0] = 0.0
    finished = torch.zeros(batch, beams, dtype=torch.bool, device="cuda")
    chosen = torch.empty(batch, beams, 0, dtype=torch.int64, device="cuda")
    for i in range(new):
        scores, parents, picked = beam_search_select(logits, scores, finished, end_token)
        chosen = torch.cat([chosen.gather(1, parents.unsqueeze(-1).expand(-1, -1, i)), picked.unsqueeze(-1)], -1)
        finished = finished.gather(1, parents) | (picked == end_token)
        if i + 1 == new:
            break
        beam_search_reorder([t for s in states for t in s], parents)
        logits = model.step(picked.flatten(), states).view(batch, beams, -1)
    return chosen, scores


def main():
    ap = argparse.ArgumentParser()
    ap.add_argument("--steps", type=int, default=100)
    ap.add_argument("--dim", type=int, default=256)
    ap.add_argument("--layers", type=int, default=2)
    ap.add_argument("--block", choices=("gated", "selective"), default="gated")
    ap.add_argument("--beams", type=int, default=0)
    args = ap.parse_args()
    torch.manual_seed(0)
    gen = torch.Generator(device="cuda").manual_seed(0)
    vocab = 64
    model = Model(vocab, args.dim, args.layers, layer=Layer if args.block == "gated" else SelectiveLayer)
    train(model, args.steps, vocab, gen)
    off, top = serve(model, vocab, gen)
    print(f"decoding differs from a whole pass by at most {off:.4f} (logits up to {top:.2f})")
    if args.beams:
        prompt = torch.randint(0, vocab, (1, 40), generator=gen, device="cuda")
        tokens, scores = beam_search(model, prompt, args.beams, 12, vocab - 1)
        for row, score in zip(tokens[0].tolist(), scores[0].tolist()):
            print(f"{score:9.3f}  {row}")


if __name__ == "__main__":
    main()
