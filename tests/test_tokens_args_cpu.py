"""CPU: arguments of the multi-token calls that the Python layer passes on or refuses."""
import pytest

import eakv_b200 as E


def test_fork_passes_a_capacity_of_zero_on(monkeypatch):
    """0 positions is the caller's error, for the library to refuse; None is the source's capacity."""
    asked = []

    class Library:
        @staticmethod
        def eakv_cache_fork(h, n, size, out):
            asked.append(size)
            return E.EAKV_ERR_INVALID

        @staticmethod
        def eakv_cache_max_seq_len(h):
            return 77

        def __getattr__(self, name):   # the error's record
            return getattr(real, name)

    real = E.lib()
    monkeypatch.setattr(E, "lib", lambda: Library())
    c = E.Cache.__new__(E.Cache)
    c.h = None
    for size in (0, None, 5, -1):
        with pytest.raises(E.EakvError):
            c.fork(3, size)
    assert asked == [0, 77, 5, -1]
