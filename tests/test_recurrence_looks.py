"""The limit on the gated recurrence's waits, as it is set and asked for (CPU only)."""
from reimagined_amd import _lib


def test_limit():
    looks = _lib.lib().nsosx_gated_recurrence_looks
    assert looks(-1) == 1 << 22
    try:
        assert looks(7) == 1 << 22 and looks(-5) == 7 and looks(0) == 7 and looks(2**31 - 1) == 0
        assert looks(-1) == 1 << 22  # the most there are
    finally:
        looks(1 << 22)
    assert looks(-1) == 1 << 22
