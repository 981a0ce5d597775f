"""Beam search: the best continuations of each request's beams, and the states that follow them.

    total[b, k, v] = scores[b, k] + log_softmax(logits[b, k])[v]

``beam_search_select`` chooses over beams and vocabulary; ``beam_search_reorder`` moves the
states of the convolution and of a recurrence from the chosen parents to their children, in
place.
"""

from __future__ import annotations

import torch
from causal_conv1d._abi import block as _block


def beam_search_select(logits, scores, finished=None, end_token=None, num_candidates=None):
    """The num_candidates (default: beams) best continuations of each request.

    logits: (batch, beams, vocab) fp32, fp16 or bf16; scores: (batch, beams) fp32, the beams'
    log-probabilities so far (-inf: not in use, as all but the first beam before the first
    token).  finished: (batch, beams) bool, beams at their end: such a beam has one
    continuation, end_token again, and keeps its score.

    Returns (scores, parents, tokens), each (batch, num_candidates), in descending order of the
    total log-probability, equal ones by the lowest parent * vocab + token: scores fp32, parents
    (the beam that is continued) and tokens int64.  At most 64 beams and 64 candidates.

    What is no number counts as -inf: a beam whose score is not finite, or whose logits hold a
    NaN, +inf or nothing above -inf, offers its tokens at -inf.  Candidates at -inf are
    returned where there are no others.  Tokens of one beam are ordered by their logits, even
    where a huge score leaves their totals equal.  There is no derivative: a backward pass that
    reaches the returned scores raises.
    """
    return _block.beam_select(logits, scores, finished, end_token, num_candidates)


def beam_search_reorder(states, parents, state_indices=None):
    """states[b * beams + k] becomes what states[b * beams + parents[b, k]] was, in place.

    states: a tensor (batch * beams, ...) of up to four dimensions, or a list of them (the states
    of all layers move in one launch); any dtype.  parents: (batch, beams) int32 or int64, as
    chosen by :func:`beam_search_select`; a beam whose parent is outside [0, beams) keeps its
    state.  state_indices: (batch * beams,) rows of the states, which are then a pool of any
    number of rows, as in :func:`causal_conv1d_update`; a beam whose row or parent's row is
    outside the pool keeps its state, and no row may be named twice.  The indices are int32;
    other signed integers and uint8 are converted.

    At most 64 beams.  No two elements of a tensor may lie at the same place, and no two of the
    tensors may share memory (two that start at one place are refused).  States that require grad are refused outside torch.no_grad().
    """
    _block.beam_reorder([states] if isinstance(states, torch.Tensor) else list(states), parents, state_indices)


def beam_search_select_ref(logits, scores, finished=None, end_token=None, num_candidates=None):
    """PyTorch statement of :func:`beam_search_select`, in fp64."""
    batch, beams, vocab = logits.shape
    x = logits.double()
    top = x.amax(-1, keepdim=True)  # taken off first: a large one would swallow the sum
    above = torch.log(torch.exp(x - top).sum(-1, keepdim=True))
    logp = x - top - above
    sound = torch.isfinite(above.squeeze(-1))
    if finished is not None:
        only = torch.full((vocab,), float("-inf"), dtype=x.dtype, device=x.device)
        only[end_token] = 0.0
        logp = torch.where(finished.unsqueeze(-1), only, logp)
        sound = sound | finished
    total = scores.double().unsqueeze(-1) + logp
    total = torch.where((sound & torch.isfinite(scores)).unsqueeze(-1), total, float("-inf")).flatten(1)
    best, place = torch.sort(total, dim=1, descending=True, stable=True)
    n = beams if num_candidates is None else num_candidates
    return best[:, :n].float(), place[:, :n] // vocab, place[:, :n] % vocab


def beam_search_reorder_ref(states, parents, state_indices=None):
    """PyTorch statement of :func:`beam_search_reorder`: returns new tensors."""
    batch, beams = parents.shape
    rows = list(range(batch * beams)) if state_indices is None else state_indices.tolist()
    found = []
    for t in [states] if isinstance(states, torch.Tensor) else states:
        new = t.clone()
        for b, chosen in enumerate(parents.tolist()):
            for k, parent in enumerate(chosen):
                if not 0 <= parent < beams:
                    continue
                source, target = rows[b * beams + parent], rows[b * beams + k]
                if 0 <= source < t.shape[0] and 0 <= target < t.shape[0]:
                    new[target] = t[source]
        found.append(new)
    return found[0] if isinstance(states, torch.Tensor) else found
