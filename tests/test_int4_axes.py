"""The axes of an append without positions, at the C symbol: a new token then is at its place in the cache on every axis that a pair may turn with."""
import pytest

from flashck_b200 import _lib

P = 4096  # an address that is never read: the calls have no tokens


def _append(axes, pair):
    rc = _lib.lib().FmhaFwdAppendKVInt4(0, 0, P, P, 0, P, P, 0, 0, 0, P, 0, 0, 0, P, P, pair, P, 0, 2, 0, 0, 4, 2, 64, 32, axes, 64, 10, 2, 4, 16, 8, 0, 4)
    return rc, _lib.last_error()


@pytest.mark.parametrize("axes", [1, 3, 4])
def test_pairs_turn_with_any_axis(axes):
    rc, text = _append(axes, bytes(i % axes for i in range(32)))
    assert rc in (0, 3), text  # (3: no GPU here, which comes after the arguments)


def test_pairs_of_axes_that_are_not_there():
    rc, text = _append(2, bytes([2] * 32))
    assert rc == 1 and "turns with axis 2 of 2" in text
    assert _append(5, bytes(32))[0] == 2 and _append(0, bytes(32))[0] == 2
    assert _append(0, None)[0] in (0, 3)  # (no pair asks for an axis)
