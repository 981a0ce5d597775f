"""The statement of beam_search_select where logits are masked by large finite values."""

import math

import pytest
import torch

from causal_conv1d.beam_search import beam_search_select_ref


@pytest.mark.parametrize("mask", [torch.finfo(torch.float32).min, -1e30, -1e10])
def test_select_statement_of_masked_rows(mask):
    logits = torch.full((1, 2, 100), mask)
    scores = torch.tensor([[-1.0, -30.0]])
    best, parents, tokens = beam_search_select_ref(logits, scores, num_candidates=4)
    assert parents.tolist() == [[0] * 4] and tokens.tolist() == [[0, 1, 2, 3]]
    assert (best - (-1.0 - math.log(100))).abs().max() < 1e-6  # all tokens are alike
    logits[0, 1, 7], logits[0, 1, 40] = 1.0, 2.0
    best, parents, tokens = beam_search_select_ref(logits, torch.tensor([[-math.inf, -3.0]]), num_candidates=3)
    assert parents.tolist() == [[1] * 3] and tokens.tolist() == [[40, 7, 0]]
    lse = math.log(math.exp(1.0) + math.exp(2.0))
    assert abs(best[0, 0] - (2.0 - lse - 3.0)) < 1e-6 and abs(best[0, 1] - (1.0 - lse - 3.0)) < 1e-6
