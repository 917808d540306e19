"""GPU: calls at the edges of what copies, gathers, compactions, reads and appends take."""
import ctypes

import numpy as np
import pytest

import eakv_b200 as E
from gpu_util import kv_data

pytestmark = pytest.mark.gpu


def make(L, H, hd, size, n, seed=0):
    c = E.Cache(L, H, hd, size)
    if n:
        assert c.load_raw(kv_data(np.random.default_rng(seed), L, H, n, hd), n) == 0
    return c


@pytest.mark.parametrize("shape", [(0,), (2, 0), (3, 2, 0), (1, 1, 0)])
def test_empty_lists(gpu, shape):
    """No accepted draft token, nothing kept: an empty list moves nothing and sets the length."""
    import torch
    src, dst = make(3, 2, 64, 100, 90), make(3, 2, 64, 100, 20)
    index = torch.empty(shape, dtype=torch.int32, device=gpu)
    assert index.data_ptr() == 0
    before = [c.dequantize(0, 0, 0, 7) for c in (src, dst)]
    E.gather_positions(dst, 7, src, index)
    src.compact(80, index)
    assert (dst.seq_len, src.seq_len) == (7, 80)
    for c, was in zip((src, dst), before):
        assert np.array_equal(c.dequantize(0, 0, 0, 7), was)
    L = E.lib()
    assert L.eakv_cache_compact(src.h, 80, None, 0, 0, 1, None) == E.EAKV_ERR_INVALID
    assert L.eakv_cache_gather(dst.h, 7, src.h, None, 0, 0, 1, None) == E.EAKV_ERR_INVALID
    assert (dst.seq_len, src.seq_len) == (7, 80)
    src.free()
    dst.free()


def test_misaligned_lists_and_positions_are_refused(gpu):
    """An address that is no multiple of 4 is refused on the host."""
    import torch
    L = E.lib()
    src, dst = make(1, 2, 64, 100, 90), make(1, 2, 64, 100, 20)
    room = torch.zeros(64, dtype=torch.int32, device=gpu)
    x = torch.zeros(4, 2, 64, device=gpu)
    tab = torch.ones(8, 32, device=gpu)
    rows = E._Rows(x.data_ptr(), 128, 64, E.EAKV_F32)
    hs, n = (ctypes.c_void_p * 1)(dst.h), (ctypes.c_int * 1)(4)
    for off in (1, 2, 3):
        at = room.data_ptr() + off
        assert L.eakv_cache_gather(dst.h, 0, src.h, at, 0, 0, 4, None) == E.EAKV_ERR_INVALID
        assert L.eakv_cache_compact(src.h, 0, at, 0, 0, 4, None) == E.EAKV_ERR_INVALID
        rot = E._Rotary(tab.data_ptr(), tab.data_ptr(), 8, 64, 0, at, 0, 1, (ctypes.c_int * 4)(32, 0, 0, 0))
        assert L.eakv_append_rotary(hs, 1, 0, n, ctypes.byref(rows), ctypes.byref(rows), None, None, 2,
                                    ctypes.byref(rot), None) == E.EAKV_ERR_INVALID
        assert "misaligned" in E.last_error()[1] or "4-byte" in E.last_error()[1]
    assert (src.seq_len, dst.seq_len) == (90, 20)
    src.free()
    dst.free()
    assert E.device_status(0) == 0
