"""Scratch of the selective recurrence's backward pass: the sums of dB and dC of each CTA's channels, of as many
batch rows as 2 GB hold, but of one row at least."""

import pytest

from causal_conv1d import _abi
from test_selective_cpu import _sel, _tensor


def _bytes(batch, dim, seqlen, dstate, groups=1):
    t = _tensor(strides=(dim * seqlen, 1, dim))
    ins = {k: t for k in ("x", "delta", "A", "B", "C", "dout", "dx", "ddelta", "dB", "dC")}
    return _abi.load_library().cc1d_selective_bwd_workspace_bytes(
        _sel(batch=batch, dim=dim, seqlen=seqlen, dstate=dstate, groups=groups, nstates=batch, checkpoints=16, **ins))


def _row(dim, seqlen, dstate, groups=1):
    padded, lanes = -(-dstate // 4) * 4, 1
    while lanes < 16 and 4 * lanes < dstate:
        lanes *= 2
    tiles = groups * -(-(dim // groups) // (128 // lanes))  # CTAs that a position's channels take
    return 8 * seqlen * tiles * padded, 4 * dim * (2 * padded + 3)  # and of one part of a sequence


# the last three take more than 2 GB for one row: 64 bytes for each position and channel at 64 states, 256 at 256
@pytest.mark.parametrize("batch,dim,seqlen,dstate,groups", [(4, 4096, 2048, 16, 1), (9, 512, 8192, 64, 1), (16, 4096, 4096, 64, 1),
                                                            (3, 770, 1027, 7, 2), (64, 2048, 4096, 32, 1), (1, 8192, 16384, 64, 1),
                                                            (3, 8192, 16384, 64, 1), (1, 8192, 16384, 256, 1)])
def test_scratch_of_the_backward(batch, dim, seqlen, dstate, groups):
    row, part = _row(dim, seqlen, dstate, groups)
    rows = max(1, min(batch, int(2e9 // row)))
    got = _bytes(batch, dim, seqlen, dstate, groups)
    # up to 64 parts of each sequence, four blocks on 16 bytes
    assert rows * row <= got <= rows * row + 64 * batch * part + 5 * 16
    assert got <= 2e9 + 64 * batch * part or rows == 1
