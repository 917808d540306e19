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


def test_outputs_that_overlap_are_refused(gpu):
    """A broadcast tensor as an output would be written by several rows at once; as an input it is
    one row for all."""
    import torch
    c = make(2, 2, 64, 40, 20)
    n, H, G, hd = 3, 2, 2, 64
    k = torch.randn(n, H, hd, device=gpu)
    q = torch.randn(n, H * G, hd, device=gpu)
    tab = torch.ones(8, 32, device=gpu)
    pos = torch.zeros(n, dtype=torch.int32, device=gpu)
    turn = dict(cos=tab, sin=tab * 0, positions=pos)
    one_token, one_head = torch.zeros(1, H * G, hd, device=gpu), torch.zeros(n, 1, hd, device=gpu)
    near = torch.zeros(n * H * G * 8 + hd, device=gpu).as_strided((n, H * G, hd), (H * G * 8, 8, 1))
    bad = [one_token.expand(n, -1, -1), one_head.expand(-1, H * G, -1), near]
    for out in bad:
        with pytest.raises(E.EakvError, match="overlap"):
            E.append_rotary([c], 0, [n], k, k, q=q, q_out=out, **turn)
        with pytest.raises(E.EakvError, match="overlap"):
            E.extend_attention([c], 0, [n], q, out)
    out = torch.zeros(2, 2, n, H, hd, device=gpu)
    for dim in range(4):
        with pytest.raises((E.EakvError, ValueError), match="overlap"):
            E.read_positions([c], [0], [n], out[(slice(None),) * dim + (slice(0, 1),)].expand(out.shape))
    # as inputs, and where there is one row along the stride
    torch.cuda.synchronize()
    E.append_rotary([c], 0, [n], k[:1].expand(n, -1, -1), k[:, :1].expand(-1, H, -1), q=q, **turn)
    E.extend_attention([c], 0, [n], one_token.expand(n, -1, -1), q)
    E.extend_attention([c], 0, [1], q[:1], one_token.as_strided((1, H * G, hd), (0, hd, 1)))
    E.read_positions([c], [0], [1], torch.zeros(2, H * hd, device=gpu).as_strided((1, 2, 1, H, hd), (0, H * hd, 0, hd, 1)))
    c.synchronize()
    got = torch.zeros(1, 2, n, H, hd, device=gpu)
    torch.cuda.synchronize()
    E.read_positions([c], [20], [n], got)
    c.synchronize()
    assert torch.equal(got[0, 0, 0], got[0, 0, 1]) and torch.equal(got[0, 1, :, 0], got[0, 1, :, 1])
    c.free()
    assert E.device_status(0) == 0


def test_captured_moves(gpu):
    """Copy, gather and compact in one graph, replayed: each replay moves what its sources and
    lists hold then, for the lengths that it was captured with."""
    import torch
    src, keep, a, b = (make(2, 2, 128, 300, 200, seed=i) for i in range(4))
    index = torch.arange(0, 200, 2, dtype=torch.int32, device=gpu)
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        E.copy_positions([a], 5, src, 10, 150, stream=s.cuda_stream)
        E.gather_positions(b, 0, src, index, stream=s.cuda_stream)
        keep.compact(0, index, stream=s.cuda_stream)
    assert (a.seq_len, b.seq_len, keep.seq_len) == (155, 100, 100)
    for step in (1, 2):
        data = kv_data(np.random.default_rng(10 + step), 2, 2, 200, 128)
        for c in (src, keep):
            c.clear()
            assert c.load_raw(data, 200) == 0
        index.copy_(torch.arange(step, 100 + step, dtype=torch.int32, device=gpu))
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert keep.seq_len == 200       # a replay is the device's work alone
        assert keep.restore(100) == 0
        for l in range(2):
            for kv in (0, 1):
                whole = src.dequantize(l, kv, 0, 200)
                assert np.array_equal(a.dequantize(l, kv, 5, 155), whole[:, 10:160])
                assert np.array_equal(b.dequantize(l, kv, 0, 100), whole[:, step:100 + step])
                assert np.array_equal(keep.dequantize(l, kv, 0, 100), whole[:, step:100 + step])
    del g
    for c in (src, keep, a, b):
        c.free()
    assert E.device_status(0) == 0


def test_copies_to_256(gpu):
    src = make(1, 1, 64, 80, 70)
    dsts = [make(1, 1, 64, 75 + i % 7, 3) for i in range(257)]
    with pytest.raises(E.EakvError, match="256"):
        E.copy_positions(dsts, 3, src, 0, 70)
    E.copy_positions(dsts[:256], 3, src, 0, 70)
    src.synchronize()
    want = [src.dequantize(0, kv, 0, 70) for kv in (0, 1)]
    for d in dsts[:256]:
        assert d.seq_len == 73
        assert all(np.array_equal(d.dequantize(0, kv, 3, 73), want[kv]) for kv in (0, 1))
    assert dsts[256].seq_len == 3
    for c in dsts + [src]:
        c.free()
    assert E.device_status(0) == 0
