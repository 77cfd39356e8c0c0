"""CPU: states that a reordering refuses by their sizes."""
import pytest
import torch

from nvjsel import _lib, beam

DUMMY = 0x1000  # never dereferenced: validation fails first


def test_a_state_too_large_is_refused_before_any_is_moved():
    """The 25th of 25 states, which the second launch would take."""
    lib = _lib.load()
    small = [DUMMY, 64, 4, 8, 2, 8]
    large = [DUMMY, 1 << 40, 1 << 36, 8, 2, 8]
    table = _lib.states(small * 24 + large)
    assert lib.nvjsel_reorder_states(table, 25, DUMMY, 4, None, None, 2, 4, None) == -1
    assert b"too large" in lib.nvjsel_last_error()
    many = [DUMMY, 1 << 30, 1, 8, 1 << 25, 8]  # with lengths: a block for each outer index
    table = _lib.states(small * 30 + many)
    assert lib.nvjsel_reorder_states(table, 31, DUMMY, 4, None, DUMMY, 2, 4, None) == -1
    assert b"too large" in lib.nvjsel_last_error()


def test_sizes_beyond_32_bits():
    wide = torch.empty(4, 1 << 31, 1, dtype=torch.uint8, device="meta")
    assert _lib.states([DUMMY, *beam._describe_state(wide, 4, 1)])
    with pytest.raises(ValueError, match="2\\^31"):
        beam._describe_state(wide, 4, 2)
    with pytest.raises(ValueError, match="2\\^31"):
        beam._describe_state(torch.empty(1 << 31, 1, dtype=torch.uint8, device="meta"), None, None)
