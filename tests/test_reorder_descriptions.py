"""CPU: states that a reordering refuses by their sizes."""
from nvjsel import _lib

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
