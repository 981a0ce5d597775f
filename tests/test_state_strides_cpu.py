"""Which layouts of states the C entries take: elements of their own, however they are interleaved."""

import pytest

from causal_conv1d import _abi
from test_selective_cpu import _ORDER, _refused, _tensor


def _update(strides, dstate=3):
    """So many channels of so many rows that the launcher refuses them after it has looked at the state."""
    t, none = _tensor(), _abi._NONE
    tensors = {"x": t, "delta": t, "A": t, "B": t, "C": t, "out": t, "state": _tensor(strides=strides), "state_indices": _tensor(dtype=3)}
    words = [1 << 18, 1 << 17, 1, dstate, 1, 2, 1]
    for k in (*_ORDER[:8], "state", "state_indices", "out"):
        words += tensors.get(k, none)
    return _abi.SELECTIVE_UPDATE_PARAMS.pack(*words, 0, 0)


D = 1 << 17


@pytest.mark.parametrize("strides", [(5 * D, 5, 2),         # every other element of five
                                     (5, 10, 2),            # rows inside the channels' gaps
                                     (1, 4, 4 * D),         # along the rows
                                     (3 * D, 3, 1)])
def test_update_takes_states_whose_elements_are_apart(strides):
    _refused(_abi.load_library().cc1d_selective_update_launch, _update(strides), 1, b"too large")


@pytest.mark.parametrize("strides", [(4 * D, 4, 2), (5 * D - 1, 5, 2), (5, 9, 2), (4, 10, 2)])
def test_update_refuses_states_that_overlap(strides):
    _refused(_abi.load_library().cc1d_selective_update_launch, _update(strides), 1, b"overlap")


def _reorder(row):
    import ctypes

    rows = [row, (4096, 6, 4, 3, 4, 1, 1, 1, 1, 1)]  # the second one has no element size: nothing is launched
    keep = ctypes.create_string_buffer(b"".join(_abi.BEAM_ROWS.pack(*r) for r in rows))
    _reorder.keep = keep
    return _abi.BEAM_REORDER_PARAMS.pack(2, 3, 2, *_tensor(dtype=4), *_abi._NONE, ctypes.addressof(keep))


@pytest.mark.parametrize("row", [(16, 6, 5, 4, 3, 1, 1, 2, 1, 1),     # every other element of five
                                 (16, 6, 15, 4, 3, 2, 1, 2, 7, 1),
                                 (16, 6, 1, 4, 3, 1, 1, 6, 1, 1)])    # rows side by side
def test_reorder_takes_states_whose_elements_are_apart(row):
    _refused(_abi.load_library().cc1d_beam_reorder_launch, _reorder(row), 1, b"element_bytes")


@pytest.mark.parametrize("row", [(16, 6, 4, 4, 3, 1, 1, 2, 1, 1), (16, 6, 11, 4, 3, 2, 1, 2, 7, 1), (16, 6, 1, 4, 3, 1, 1, 5, 1, 1)])
def test_reorder_refuses_states_that_overlap(row):
    _refused(_abi.load_library().cc1d_beam_reorder_launch, _reorder(row), 1, b"overlap")
