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


class Host:
    """A cache as the argument checks see one, on the host."""
    h, shape = 0, (2, 4, 64, -1)


def test_rotary_tables_and_positions_go_together():
    import torch
    x, tab, pos = torch.zeros(3, 4, 64), torch.zeros(8, 32), torch.zeros(3, dtype=torch.int32)
    whole = dict(cos=tab, sin=tab, positions=pos)
    for given in (["cos"], ["sin"], ["positions"], ["cos", "sin"], ["cos", "positions"], ["sin", "positions"]):
        with pytest.raises(ValueError, match="together"):
            E.append_rotary([Host()], 0, [3], x, x, **{k: whole[k] for k in given})


def test_packed_arguments_are_the_structures():
    """The calls pass eakv_rows_t and eakv_rotary_t as packed bytes: the same bytes as the ctypes structures,
    whose layout is the header's."""
    import ctypes
    rows = (2 ** 63 + 16, 2 ** 40 + 3, 2 ** 33, E.EAKV_BF16)
    assert E._pack_rows(*rows) == bytes(E._Rows(*rows))
    rot = (2 ** 63 + 32, 2 ** 62, 7, 128, 1, 2 ** 61 + 4, 2 ** 35, 3, 20, 30, 14, 0)
    packed = E._pack_rotary(*rot)
    assert packed == bytes(E._Rotary(*rot[:8], (ctypes.c_int * 4)(*rot[8:])))
