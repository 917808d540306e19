"""CPU: refusals of the multi-token calls that need no device (no cache can be
made here): NULL arguments, and the checks of the Python layer."""
import ctypes

import pytest

import eakv_b200 as E


def rows():
    return E._Rows(64, 8, 8, E.EAKV_F32)


def refused(rc):
    assert rc == E.EAKV_ERR_INVALID
    assert E.last_error()[0] == E.EAKV_ERR_INVALID and E.last_error()[1]


def test_null_caches_are_refused():
    L, r = E.lib(), rows()
    n = (ctypes.c_int * 1)(1)
    none = (ctypes.c_void_p * 1)(None)
    ref = ctypes.byref(r)
    for caches in (None, none):
        refused(L.eakv_append_rotary(caches, 1, 0, n, ref, ref, None, None, 1, None, None))
        refused(L.eakv_extend_attention(caches, 1, 0, n, ref, ref, 1, 0.0, 0, None, None, None, 0, None))
        refused(L.eakv_cache_read(caches, 1, 0, 1, n, n, ref, ref, 0, None))
        size = ctypes.c_size_t(7)
        refused(L.eakv_extend_workspace(caches, 1, n, 0, 1, 0, 0, ctypes.byref(size)))
        assert size.value == 0
    refused(L.eakv_extend_attention(none, 1, 0, n, None, ref, 1, 0.0, 0, None, None, None, 0, None))
    refused(L.eakv_cache_copy(none, 1, 0, None, 0, 1, None))
    refused(L.eakv_cache_copy(None, 1, 0, None, 0, 1, None))
    refused(L.eakv_cache_gather(None, 0, None, 64, 0, 0, 1, None))
    refused(L.eakv_cache_compact(None, 0, 64, 0, 0, 1, None))
    out = ctypes.c_void_p(5)
    refused(L.eakv_cache_fork(None, 1, 1, ctypes.byref(out)))
    assert out.value is None
    refused(L.eakv_cache_fork(None, 1, 1, None))


@pytest.mark.parametrize("n", [0, -1, 257])
def test_cache_counts_are_refused(n):
    L, r = E.lib(), rows()
    arr = (ctypes.c_void_p * 257)()
    cnt = (ctypes.c_int * 257)()
    ref = ctypes.byref(r)
    refused(L.eakv_append_rotary(arr, n, 0, cnt, ref, ref, None, None, 1, None, None))
    refused(L.eakv_extend_attention(arr, n, 0, cnt, ref, ref, 1, 0.0, 0, None, None, None, 0, None))
    refused(L.eakv_cache_read(arr, n, 0, 1, cnt, cnt, ref, ref, 0, None))
    refused(L.eakv_cache_copy(arr, n, 0, None, 0, 1, None))


def test_struct_layouts_match_the_header():
    assert ctypes.sizeof(E._Rows) == 32
    assert E._Rotary.positions.offset == 32 and E._Rotary.sections.offset == 52
    assert ctypes.sizeof(E._Rotary) == 72


class FakeCache:
    """What the argument checks ask of a cache."""
    h, shape = 0, (2, 4, 64, 0)


def test_python_checks_refuse_before_the_library():
    import torch
    c = FakeCache()
    x = torch.zeros(3, 4, 64)
    with pytest.raises(ValueError, match="is on cpu"):
        E._rows(x, c, 4, 3, "k")
    with pytest.raises(ValueError, match="shape"):
        E._rows(x, c, 4, 2, "k")
    with pytest.raises(ValueError, match="contiguous"):
        E._rows(x.transpose(1, 2).contiguous().transpose(1, 2), c, 4, 3, "k")
    with pytest.raises(TypeError):
        E._dtype(x.to(torch.float64))
    with pytest.raises(ValueError, match="entries"):
        E._ints([1, 2], 3, "counts")
    with pytest.raises(ValueError, match="int32"):
        E._index(torch.zeros(3), c)
    with pytest.raises(ValueError, match="layers"):
        E._index(torch.zeros(3, 4, 5, dtype=torch.int32), c)
    with pytest.raises(ValueError, match="contiguous"):
        E._contiguous(torch.zeros(4, 2).t(), c, "float32", (2, 4), "lse")


@pytest.mark.parametrize("sections", [[16, 17], [-1, 33], [2 ** 40, 0], [16.0, 16], [32]])
def test_bad_sections_are_refused(sections):
    import torch

    class Host(FakeCache):
        shape = (2, 4, 64, -1)   # as if tensors on the host were on its device

    x, tab = torch.zeros(3, 4, 64), torch.zeros(8, 32)
    pos = torch.zeros(2, 3, dtype=torch.int32)
    with pytest.raises((ValueError, E.EakvError)):
        E.append_rotary([Host()], 0, [3], x, x, cos=tab, sin=tab, positions=pos, sections=sections)
