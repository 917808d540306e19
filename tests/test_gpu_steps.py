"""GPU: whole steps of the multi-token calls, captured and at the widest batch."""
import numpy as np
import pytest

import eakv_b200 as E
from gpu_util import kv_data
from test_gpu_extend import DT

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _reset():
    E.force_splits(0)
    E.force_path(0)
    yield
    E.force_splits(0)
    E.force_path(0)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("new", [[1, 1, 1], [5, 0, 70]])
def test_a_captured_step(gpu, new, dtype):
    """Append, attention and read-back of a step in one graph: replayed on new rows it gives the
    eager calls' bits, for the lengths that it was captured with."""
    import torch
    t = getattr(torch, DT[dtype])
    rng = np.random.default_rng(sum(new))
    H, nq, hd, old, total = 2, 8, 128, [500, 63, 2000], sum(new)
    def batch():
        caches = []
        for i, n in enumerate(old):
            c = E.Cache(1, H, hd, 2100)
            assert c.load_raw(kv_data(np.random.default_rng(i), 1, H, n, hd), n) == 0
            caches.append(c)
        return caches

    mine, eager = batch(), batch()
    tab = torch.rand(64, hd // 2, device=gpu)
    sin = 1 - tab   # made here: on torch's stream it would not be ordered with the calls'
    pos = torch.randint(0, 64, (total,), dtype=torch.int32, device=gpu)

    def buffers():
        return dict(x=torch.zeros(total, nq + 2 * H, hd, dtype=t, device=gpu),
                    q=torch.zeros(total, nq, hd, dtype=t, device=gpu),
                    o=torch.zeros(total, nq, hd, dtype=t, device=gpu),
                    kv=torch.zeros(1, 2, total, H, hd, device=gpu))

    def step(caches, b, stream, ws):
        x = b["x"]
        E.append_rotary(caches, 0, new, x[:, nq:nq + H], x[:, nq + H:], x[:, :nq], b["q"], tab, sin, pos,
                        stream=stream)
        E.extend_attention(caches, 0, new, b["q"], b["o"], workspace=ws, stream=stream)
        E.read_positions(caches, old, new, b["kv"], stream=stream)

    E.force_splits(3)
    need = E.extend_workspace(mine, new, getattr(E, "EAKV_" + dtype.upper()), nq)
    ws = torch.zeros(need, dtype=torch.uint8, device=gpu)
    s = torch.cuda.Stream()
    b, ref = buffers(), buffers()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        step(mine, b, s.cuda_stream, ws)
    for k in range(3):
        rows = torch.from_numpy(rng.standard_normal(b["x"].shape).astype(np.float32)).to(gpu).to(t)
        b["x"].copy_(rows)
        ref["x"].copy_(rows)
        torch.cuda.synchronize()
        g.replay()
        step(eager, ref, None, None)
        torch.cuda.synchronize()
        for name in ("q", "o", "kv"):
            assert torch.equal(b[name], ref[name])
    del g
    for c in mine + eager:
        c.free()
    assert E.device_status(0) == 0


def test_the_widest_batch(gpu):
    """256 caches with 0 to 40 tokens each, in one call of each kind: the bits of calls with one
    cache alone (append, read) and results close to theirs (attention, which cuts its work anew)."""
    import torch
    rng = np.random.default_rng(5)
    n, H, nq, hd, size = 256, 1, 2, 64, 200
    caches, alone = [], []
    counts = rng.integers(0, 41, n).tolist()
    old = rng.integers(0, 150, n).tolist()
    for i in range(n):
        for group in (caches, alone):
            c = E.Cache(1, H, hd, size)
            if old[i]:
                assert c.load_raw(kv_data(np.random.default_rng(i), 1, H, old[i], hd), old[i]) == 0
            group.append(c)
    total = sum(counts)
    x = torch.from_numpy(rng.standard_normal((total, nq + 2 * H, hd)).astype(np.float32)).to(gpu).bfloat16()
    k, v, q = x[:, nq:nq + H], x[:, nq + H:], x[:, :nq]
    out, one = torch.zeros(total, nq, hd, dtype=x.dtype, device=gpu), torch.zeros(total, nq, hd, dtype=x.dtype, device=gpu)
    kv, kv1 = torch.zeros(1, 2, total, H, hd, device=gpu), torch.zeros(1, 2, total, H, hd, device=gpu)
    torch.cuda.synchronize()
    E.append_rotary(caches, 0, counts, k, v)
    E.extend_attention(caches, 0, counts, q, out)
    E.read_positions(caches, old, counts, kv)
    caches[0].synchronize()
    first = 0
    for c, m, o in zip(alone, counts, old):
        at = slice(first, first + m)
        E.append_rotary([c], 0, [m], k[at], v[at])
        E.extend_attention([c], 0, [m], q[at], one[at])
        E.read_positions([c], [o], [m], kv1[:, :, at])
        first += m
    torch.cuda.synchronize()
    for c in alone:
        c.synchronize()
    assert torch.equal(kv, kv1)
    assert (out.float() - one.float()).abs().max() <= 2.0 ** -6 * one.float().abs().max()
    many = caches + [E.Cache(1, H, hd, size)]
    for call in (lambda: E.append_rotary(many, 0, counts + [0], k, v),
                 lambda: E.extend_attention(many, 0, counts + [0], q, out),
                 lambda: E.read_positions(many, old + [0], counts + [0], kv)):
        with pytest.raises(E.EakvError, match="256"):
            call()
    for c in many + alone:
        c.free()
    assert E.device_status(0) == 0


def test_scales_that_leave_f32_are_refused(gpu):
    """A scale whose base-2 form is infinite, or that is no number."""
    import torch
    c = E.Cache(1, 1, 64, 20)
    assert c.advance(18) == 0
    q = torch.ones(2, 2, 64, device=gpu)
    for scale in (3e38, -3e38, 2.4e38, float("inf"), float("nan")):
        with pytest.raises(E.EakvError, match="scale"):
            E.extend_attention([c], 0, [2], q, torch.empty_like(q), scale=scale)
    c.free()


@pytest.mark.parametrize("hd,caches,new,old", [(128, 4, 130, 0), (128, 5, 130, 700), (64, 9, 129, 300),
                                               (64, 12, 129, 3000), (128, 96, 1, 600), (64, 200, 1, 100)])
def test_plans_agree(gpu, hd, caches, new, old):
    """Batches that are cut into runs, into whole items or into one part each give the same results to
    twice the output's half step."""
    import torch
    H, nq = 8, 32
    group = []
    for i in range(caches):
        c = E.Cache(1, H, hd, old + new)
        g = torch.Generator(device=gpu).manual_seed(i)
        raw = torch.randn(1, 2, H, old + new, hd, generator=g, device=gpu)
        torch.cuda.synchronize()
        assert c.load_raw_device(raw, old + new) == 0
        c.synchronize()
        assert c.restore(old) == 0
        group.append(c)
    q = torch.randn(caches * new, nq, hd, device=gpu).bfloat16()
    outs = []
    for splits in (0, 1, 3):
        out = torch.zeros_like(q)
        torch.cuda.synchronize()
        E.force_splits(splits)
        E.extend_attention(group, 0, [new] * caches, q, out)
        group[0].synchronize()
        outs.append(out.float())
    for o in outs[1:]:
        assert ((o - outs[0]).abs() <= 2.0 ** -7 * outs[0].abs() + 2.0 ** -9).all()
    for c in group:
        c.free()
    assert E.device_status(0) == 0


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("splits", [0, 1, 4])
@pytest.mark.parametrize("hd,new", [(64, [3, 1]), (128, [150, 9, 70])])
def test_out_may_be_q(gpu, hd, new, splits, dtype):
    """In place, whole or cut: the bits of a call with an output of its own."""
    import torch
    t = getattr(torch, DT[dtype])
    group = []
    for i in range(len(new)):
        c = E.Cache(1, 2, hd, 2000)
        assert c.load_raw(kv_data(np.random.default_rng(i), 1, 2, 1500, hd), 1500) == 0
        group.append(c)
    q = torch.randn(sum(new), 8, hd, device=gpu).to(t)
    out, own = torch.empty_like(q), q.clone()
    torch.cuda.synchronize()
    E.force_splits(splits)
    for _ in range(3):
        own.copy_(q)
        torch.cuda.synchronize()
        E.extend_attention(group, 0, new, q, out)
        E.extend_attention(group, 0, new, own, own)
        group[0].synchronize()
        assert torch.equal(out, own)
    for c in group:
        c.free()
    assert E.device_status(0) == 0


@pytest.mark.parametrize("splits", [2, 3, 10])
@pytest.mark.parametrize("hd,window,size,new,G", [(64, 18, 2598, 349, 3), (128, 100, 448, 260, 2), (64, 0, 64, 60, 3),
                                                  (128, 1, 577, 513, 1)])
def test_parts_behind_the_last_page(gpu, hd, window, size, new, G, splits):
    """A cache filled to its last page, whose last tile has fewer pairs of pages than the others: its
    empty parts lie behind the pages, and count as empty."""
    import torch
    c = E.Cache(1, 1, hd, size)
    assert c.load_raw(kv_data(np.random.default_rng(size), 1, 1, size, hd), size) == 0
    assert c.restore(size - new) == 0
    q = torch.randn(new, G, hd, device=gpu).bfloat16()
    outs = []
    for s in (1, splits):
        for path in (2, 3):
            out = torch.full_like(q, float("nan"))
            torch.cuda.synchronize()
            E.force_splits(s)
            E.force_path(path)
            E.extend_attention([c], 0, [new], q, out, window=window)
            c.synchronize()
            outs.append(out.float())
    assert E.device_status(0, reset=True) == 0
    for o in outs[1:]:
        assert ((o - outs[0]).abs() <= 2.0 ** -7 * outs[0].abs() + 2.0 ** -7).all()
    c.free()
