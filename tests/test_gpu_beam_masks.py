"""beam_search_select where logits are masked by large finite values, and where they are large themselves."""

import pytest
import torch

from causal_conv1d import beam_search_select
from causal_conv1d.beam_search import beam_search_select_ref

pytestmark = pytest.mark.gpu

INF = float("inf")
MASKS = [(torch.float32, v) for v in (torch.finfo(torch.float32).min, -1e30, -1e20, -3e10, -1e10, -5e9, -1e9, -1e4)]
MASKS += [(torch.bfloat16, v) for v in (torch.finfo(torch.bfloat16).min, -1e30, -1e10)]
MASKS += [(torch.float16, torch.finfo(torch.float16).min)]


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _select_and_check(logits, scores, n):
    """Against the definition in 64 bits and the package's statement.  The order of tokens is that of the
    definition; a total is rounded once (2^-24), and the sum of exponentials is within 2^-20 of itself:
    2^v by the hardware 2^-22, v rounded by 2^-24 |v| and weighed by 2^v, kept sums."""
    got = beam_search_select(logits, scores, num_candidates=n)
    logp = torch.log_softmax(logits.double(), -1)
    total = (scores.double().unsqueeze(-1) + torch.where(torch.isnan(logp), -INF, logp)).flatten(1)
    best, place = torch.sort(total, dim=1, descending=True, stable=True)
    vocab = logits.shape[-1]
    want = best[:, :n], place[:, :n] // vocab, place[:, :n] % vocab
    stated = beam_search_select_ref(logits, scores, num_candidates=n)
    for result in (got, stated):
        assert torch.equal(result[1], want[1]) and torch.equal(result[2], want[2])
        low = want[0].float() == -INF  # also what lies below the lowest fp32
        assert torch.equal(result[0] == -INF, low)
        assert ((result[0] - want[0]).abs()[~low] <= 2.0 ** -23 * want[0].abs()[~low] + 2.0 ** -20).all()


def _rows(seed, batch, beams, vocab, dtype, start=0):
    g = _gen(seed)
    wide = torch.full((batch, beams, vocab + 5), float("nan"), device="cuda", dtype=dtype)
    view = wide[..., start:start + vocab]
    return view.copy_(torch.randn(batch, beams, vocab, generator=g, device="cuda") * 2.5), -20 * torch.rand(batch, beams, generator=g, device="cuda")


# few rows, which several CTAs share, and more rows than CTAs run at a time
@pytest.mark.parametrize("batch,beams,vocab", [(2, 3, 128_000), (1, 4, 32_000), (300, 2, 5003), (5, 2, 300)])
@pytest.mark.parametrize("kept", [0, 1, 3, 100])
@pytest.mark.parametrize("dtype,mask", MASKS)
def test_all_but_some_tokens_masked(dtype, mask, kept, batch, beams, vocab):
    for start in (0, 1, 3):  # rows on 16 bytes and off them
        logits, scores = _rows(vocab + kept + start, batch, beams, vocab, dtype, start)
        keep = torch.zeros(batch, beams, vocab, dtype=torch.bool, device="cuda")
        if kept:
            keep.scatter_(2, torch.rand(batch, beams, vocab, generator=_gen(kept), device="cuda").topk(kept, -1).indices, True)
        logits.masked_fill_(~keep, mask)
        _select_and_check(logits, scores, 8)


@pytest.mark.parametrize("dtype,mask", MASKS)
def test_masked_ranges(dtype, mask):
    """Long runs of masked tokens at the front, in the middle and at the end, and -inf beside them."""
    vocab = 40_000
    for start in (0, 1):
        logits, scores = _rows(7 + start, 6, 3, vocab, dtype, start)
        logits[0, :, :30_000] = mask
        logits[1, :, 1000:39_000] = mask
        logits[2, :, 5:] = mask
        logits[3, :, ::2] = mask
        logits[4, :, :20_000] = -INF
        logits[4, :, 20_000:39_990] = mask
        logits[5, 0] = mask  # a beam beside others of ordinary logits
        logits[5, 1, :20_000], logits[5, 1, 20_000:] = -INF, mask
        for n in (3, 40, 64):
            _select_and_check(logits, scores, n)


@pytest.mark.parametrize("level", [-2.0 ** 20, 2.0 ** 20, 3e6, -3e6, 1e9, -1e12, -3e38, 3e38, -2000.0])
def test_large_logits(level):
    """Logits around one large value: a softmax does not depend on it."""
    g = _gen(1)
    step = max(1.0, abs(level) * 2.0 ** -22)  # a few values apart
    logits = level + step * torch.randn(4, 3, 50_000, generator=g, device="cuda")
    logits[1, :, :30_000] = -INF
    logits[2, :, 1000:] = level - 40 * step
    logits[3, 1] = level
    _select_and_check(logits, -20 * torch.rand(4, 3, generator=g, device="cuda"), 40)
