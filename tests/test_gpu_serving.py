"""GPU: the multi-token calls as a server runs them together, and what several
calls, graphs, streams and large caches could do to each other."""
import numpy as np
import pytest

import eakv_b200 as E
from gpu_util import kv_data
from test_gpu_extend import DT, HALF_STEP, Batch, _reset, check, limits, plain, rounded, run  # noqa: F401

pytestmark = pytest.mark.gpu


def tables(rows, pairs):
    ang = np.arange(rows)[:, None] / 10000.0 ** (np.arange(pairs) / pairs)
    return np.cos(ang).astype(np.float32), np.sin(ang).astype(np.float32)


def values(c, layer, kv, begin, end):
    """Positions [begin, end) in 64 bits, those not advanced over among them."""
    n = c.seq_len
    assert c.advance(end - n) == 0
    d = c.dequantize(layer, kv, begin, end).astype(np.float64)
    assert c.restore(n) == 0
    return d


class View:
    """What test_gpu_extend.plain needs of a batch: the caches' values in 64 bits
    with the new tokens in, one layer."""

    def __init__(self, caches, layer, new):
        self.old, self.new, self.H = [c.seq_len for c in caches], new, caches[0].n_kv_heads
        n = [a + b for a, b in zip(self.old, new)]
        self.k = [{layer: values(c, layer, 0, 0, s)} for c, s in zip(caches, n)]
        self.v = [{layer: values(c, layer, 1, 0, s)} for c, s in zip(caches, n)]


def close(got, want, lim):
    err = np.abs(got - want)
    assert (err <= lim).all(), f"worst {np.max(err / lim)} of the limit"


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("hd,nq,nkv,old,draft", [(128, 8, 2, [70, 0], 5), (64, 8, 1, [200, 129], 13)])
def test_speculative_steps(gpu, hd, nq, nkv, old, draft, dtype):
    """Two layers, two sequences: a tree of draft tokens goes in with its rotary
    positions and is attended under its mask; the accepted path is kept (compact),
    and the next single token agrees between extend_attention and the decode over
    the positions that are left. A fork goes on from the same prefix."""
    import torch
    rng = np.random.default_rng(draft)
    L, B, pairs = 2, len(old), hd // 2
    t = getattr(torch, DT[dtype])
    caches = []
    for n in old:
        c = E.Cache(L, nkv, hd, max(old) + draft + 1)
        if n:
            assert c.load_raw(kv_data(rng, L, nkv, n, hd), n) == 0
        caches.append(c)
    cos, sin = tables(max(old) + draft + 2, pairs)
    dcos, dsin = torch.from_numpy(cos).to(gpu), torch.from_numpy(sin).to(gpu)
    # token j's parent is j - 1 but for the last, whose parent is the first
    parent = list(range(-1, draft - 2)) + [0]
    depth, mask = [], []
    for j, p in enumerate(parent):
        depth.append(0 if p < 0 else depth[p] + 1)
        mask.append((0 if p < 0 else mask[p]) | 1 << j)
    total = B * draft
    pos = torch.tensor([[n + d for n in old for d in depth]], dtype=torch.int32, device=gpu)
    tree = torch.tensor(mask * B, dtype=torch.int64, device=gpu)

    def rows(n, heads):
        x = rng.standard_normal((n, heads, hd)).astype(np.float32)
        return torch.from_numpy(x).to(gpu).to(t)

    before = [c.dequantize(0, 0, 0, n) for c, n in zip(caches, old)]
    for layer in range(L):
        k, v, q = rows(total, nkv), rows(total, nkv), rows(total, nq)
        turned, out = torch.empty_like(q), torch.empty_like(q)
        torch.cuda.synchronize()
        E.append_rotary(caches, layer, [draft] * B, k, v, q, turned, dcos, dsin, pos)
        E.extend_attention(caches, layer, [draft] * B, turned, out, tree=tree)
        caches[0].synchronize()
        view = View(caches, layer, [draft] * B)
        want, _, size = plain(view, layer, turned.float().cpu().numpy(), hd ** -0.5, 0,
                              np.array(mask * B, np.uint64))
        lim, _ = limits(dtype, want, size, draft * nq // nkv, max(old) + draft)
        close(out.double().cpu().numpy(), want, lim)
    for c in caches:
        assert c.advance(draft) == 0
    # tokens 0 and the last are accepted: the branch of the tree
    fork = caches[0].fork(old[0]) if old[0] else None
    for c, n in zip(caches, old):
        kept = [[c.dequantize(l, kv, n + j, n + j + 1) for j in (0, draft - 1)]
                for l in range(L) for kv in (0, 1)]
        c.compact(n, torch.tensor([n, n + draft - 1], dtype=torch.int32, device=gpu))
        c.synchronize()
        assert c.seq_len == n + 2
        for i, pair in enumerate(kept):
            got = c.dequantize(i // 2, i % 2, n, n + 2)
            assert np.array_equal(got, np.concatenate(pair, axis=1))
    for c, n, was in zip(caches, old, before):
        assert np.array_equal(c.dequantize(0, 0, 0, n), was)
    # one more token in every layer
    q32 = torch.empty(B, L, nq, hd, device=gpu)
    outs = []
    pos1 = torch.tensor([[n + 2 for n in old]], dtype=torch.int32, device=gpu)
    lims = []
    for layer in range(L):
        k, v, q = rows(B, nkv).float(), rows(B, nkv).float(), rows(B, nq).float()
        out = torch.empty_like(q)
        torch.cuda.synchronize()
        E.append_rotary(caches, layer, [1] * B, k, v, q, None, dcos, dsin, pos1)   # in place
        E.extend_attention(caches, layer, [1] * B, q, out)
        caches[0].synchronize()
        want, _, size = plain(View(caches, layer, [1] * B), layer, q.cpu().numpy(), hd ** -0.5)
        lim, _ = limits("f32", want, size, nq // nkv, max(old) + 3)
        close(out.double().cpu().numpy(), want, lim)
        q32[:, layer] = q
        outs.append(out)
        lims.append(lim)
    for c in caches:
        assert c.advance(1) == 0
    dec = torch.empty_like(q32)
    torch.cuda.synchronize()
    E.decode_attention(caches, q32, nq, dec)
    caches[0].synchronize()
    for layer in range(L):   # the decode's own bar is 1e-4
        close(dec[:, layer].double().cpu().numpy(), outs[layer].double().cpu().numpy(), lims[layer] + 1e-4)
    if fork is not None:
        assert fork.seq_len == old[0]
        out = torch.empty(L, 2, 3, nkv, hd, device=gpu)
        E.read_positions([fork], [old[0] - 3], [3], out)
        fork.synchronize()
        assert np.array_equal(out[0, 0].cpu().numpy().transpose(1, 0, 2), before[0][:, old[0] - 3:])
        fork.free()
    assert E.device_status(0) == 0
    for c in caches:
        c.free()


# ragged lengths: more work in some items than a CTA's equal share, so that runs cut
# items and hold several
RAGGED = [
    # hd, nq, nkv, old, new
    (64, 16, 4, [5200, 300, 64, 0, 900, 2400], [9, 20, 3, 40, 1, 8]),
    (128, 8, 2, [3900, 100, 1000, 63], [150, 33, 64, 300]),
    (64, 8, 8, [30, 2000, 60, 90, 6000], [140, 257, 8, 31, 129]),
]


@pytest.mark.parametrize("dtype,path", [("f32", "auto"), ("bf16", "auto"), ("bf16", "mma"), ("f16", "umma")])
@pytest.mark.parametrize("hd,nq,nkv,old,new", RAGGED)
def test_ragged_runs(gpu, hd, nq, nkv, old, new, dtype, path):
    rng = np.random.default_rng(hd + nq)
    b = Batch(rng, 1, nkv, hd, old, new)
    q = rng.standard_normal((sum(new), nq, hd)).astype(np.float32)
    check(gpu, b, 0, q, dtype, nq)
    check(gpu, b, 0, q, dtype, nq, window=777)
    b.free()


@pytest.mark.parametrize("dtype,path", [("f32", "auto"), ("bf16", "mma"), ("bf16", "umma")])
@pytest.mark.parametrize("splits", [0, 1, 3])
def test_runs_that_give_up_leave_the_next_call_whole(gpu, dtype, path, splits):
    """A page (or tile) that never comes, in equal runs and in splits: status bit 1,
    and the same call is right again, so the counters are back at zero."""
    rng = np.random.default_rng(61)
    hd, nq, nkv, old, new = RAGGED[1]
    b = Batch(rng, 1, nkv, hd, old, new)
    q = rng.standard_normal((sum(new), nq, hd)).astype(np.float32)
    E.force_splits(splits)
    want, _ = run(gpu, b, 0, q, dtype, nq)
    E.test_stall(1, 2000)
    run(gpu, b, 0, q, dtype, nq)
    E.test_stall(-1)
    assert E.device_status(0, reset=True) == 1
    for _ in range(2):
        again, _ = run(gpu, b, 0, q, dtype, nq)
        assert np.array_equal(again, want)
    assert E.device_status(0) == 0
    b.free()


@pytest.mark.parametrize("dtype,path", [("f32", "auto"), ("bf16", "umma")])
def test_calls_side_by_side(gpu, dtype, path):
    """Two streams, each with a workspace of its own, in flight together, and both
    captured in graphs that are replayed together: the bits of one call alone."""
    import torch
    rng = np.random.default_rng(67)
    t = getattr(torch, DT[dtype])
    sets = []
    for hd, nq, nkv, old, new in (RAGGED[0], RAGGED[2]):
        b = Batch(rng, 1, nkv, hd, old, new)
        q = rng.standard_normal((sum(new), nq, hd)).astype(np.float32)
        want, _ = run(gpu, b, 0, q, dtype, nq)
        need = E.extend_workspace(b.caches, new, getattr(E, "EAKV_" + dtype.upper()), nq)
        assert need > 0
        dq = torch.from_numpy(q).to(gpu).to(t)
        sets.append((b, new, dq, torch.zeros_like(dq), torch.zeros(need, dtype=torch.uint8, device=gpu), want,
                     torch.cuda.Stream()))

    def call(s):
        b, new, dq, out, ws, _, stream = s
        E.extend_attention(b.caches, 0, new, dq, out, workspace=ws, stream=stream.cuda_stream)

    torch.cuda.synchronize()
    for _ in range(4):
        for s in sets:
            call(s)
    torch.cuda.synchronize()
    for s in sets:
        assert np.array_equal(s[3].double().cpu().numpy(), s[5])
    graphs = []
    for s in sets:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s[6]):
            call(s)
        graphs.append(g)
    for _ in range(3):
        for s in sets:
            s[3].zero_()
        torch.cuda.synchronize()
        for g, s in zip(graphs, sets):
            with torch.cuda.stream(s[6]):
                g.replay()
        torch.cuda.synchronize()
        for s in sets:
            assert np.array_equal(s[3].double().cpu().numpy(), s[5])
    del graphs
    for s in sets:
        s[0].free()
    assert E.device_status(0) == 0


def test_captured_decode_outlives_extend_calls(gpu):
    """A decode with splits, captured on the cache's own scratch; extend calls that grow
    what the same cache keeps for them; the replay still gives the decode's bits."""
    import torch
    rng = np.random.default_rng(79)
    b = Batch(rng, 1, 2, 128, [3000], [600])
    c = b.caches[0]
    s = torch.cuda.Stream()
    q = torch.from_numpy(rng.standard_normal((1, 1, 8, 128)).astype(np.float32)).to(gpu)
    out = torch.zeros_like(q)
    torch.cuda.synchronize()
    E.force_splits(5)
    E.decode_attention([c], q, 8, out, stream=s.cuda_stream)
    torch.cuda.synchronize()
    want = out.clone()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        E.decode_attention([c], q, 8, out, stream=s.cuda_stream)
    rows = torch.from_numpy(rng.standard_normal((600, 8, 128)).astype(np.float32)).to(gpu)
    res = torch.empty_like(rows)
    torch.cuda.synchronize()
    held = lambda: E.lib().eakv_cache_device_bytes(c.h)  # noqa: E731
    before = held()
    for n, splits in ((1, 5), (600, 7), (600, 40)):
        E.force_splits(splits)
        E.extend_attention([c], 0, [n], rows[:n], res[:n])
        c.synchronize()
    assert held() > before
    for _ in range(2):
        out.zero_()
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    del g
    b.free()
    assert E.device_status(0) == 0


def test_the_same_cache_twice_and_padded_rows(gpu):
    """extend_attention only reads the caches: one of them may be there twice, with
    different counts. Rows behind the last token stay as they are, and a call without
    tokens does nothing."""
    import torch
    rng = np.random.default_rng(71)
    b = Batch(rng, 1, 2, 64, [150], [6])
    c = b.caches[0]
    for dtype in ("f32", "bf16"):
        t = getattr(torch, DT[dtype])
        q = torch.from_numpy(rng.standard_normal((12, 6, 64)).astype(np.float32)).to(gpu).to(t)
        out = torch.full((12, 6, 64), 7.0, device=gpu, dtype=t)
        one = torch.empty(6, 6, 64, device=gpu, dtype=t)
        torch.cuda.synchronize()
        E.extend_attention([c, c], 0, [6, 3], q[:9], out[:9])
        E.extend_attention([c], 0, [6], q[:6], one)
        E.extend_attention([c, c], 0, [0, 0], q[:0], out[:0])
        c.synchronize()
        assert torch.equal(out[:6], one) and (out[9:] == 7.0).all()
        E.extend_attention([c], 0, [3], q[6:9], one[:3])
        c.synchronize()
        assert torch.equal(out[6:9], one[:3])
    b.free()


def test_offsets_behind_four_gigabytes(gpu):
    """The last layer of a slab of 4.3 GB: append, attention, read, copy and compact."""
    import torch
    rng = np.random.default_rng(73)
    L, H, hd, nq, S, n = 64, 8, 128, 16, 52480, 5
    c, other = E.Cache(L, H, hd, S), E.Cache(L, H, hd, 64)
    last, at = L - 1, S - 40
    pages = S // 64
    assert L * 2 * H * pages * 5120 > 1 << 32
    assert c.advance(at) == 0
    k, v = (torch.from_numpy(rng.standard_normal((40, H, hd)).astype(np.float32)).to(gpu) for _ in range(2))
    torch.cuda.synchronize()
    E.append_rotary([c], last, [40], k, v)
    c.synchronize()
    assert c.advance(40 - n) == 0
    view = View.__new__(View)
    view.old, view.new, view.H = [40 - n], [n], H
    view.k, view.v = ([{last: values(c, last, kv, at, S)}] for kv in (0, 1))
    q = rng.standard_normal((n, nq, hd)).astype(np.float32)
    window = 40 - n + 1   # the first new token's window begins where the appended ones do
    for dtype in ("f32", "bf16"):
        dq = torch.from_numpy(q).to(gpu).to(getattr(torch, DT[dtype]))
        for path in ((0,) if dtype == "f32" else (2, 3)):
            out = torch.empty_like(dq)
            torch.cuda.synchronize()
            E.force_path(path)
            E.extend_attention([c], last, [n], dq, out, window=window)
            E.force_path(0)
            c.synchronize()
            want, _, size = plain(view, last, rounded(q, dtype), hd ** -0.5, window)
            lim, _ = limits(dtype, want, size, 64 if path == 3 else 1, 40)
            close(out.double().cpu().numpy(), want, lim)
    assert c.advance(n) == 0
    got = torch.empty(1, 2, 40, H, hd, device=gpu)
    E.read_positions([c], [at], [40], got, layer=last)
    E.copy_positions([other], 0, c, at, 40)
    torch.cuda.synchronize()
    c.synchronize()
    got = got.cpu().numpy()
    for kv in (0, 1):
        want = view.k if kv == 0 else view.v
        assert np.array_equal(got[0, kv].transpose(1, 0, 2).astype(np.float64), want[0][last])
        assert np.array_equal(other.dequantize(last, kv, 0, 40).astype(np.float64), want[0][last])
    c.compact(at, torch.arange(at + 3, at + 40, 4, dtype=torch.int32, device=gpu))
    c.synchronize()
    assert np.array_equal(c.dequantize(last, 1, at, c.seq_len).astype(np.float64), view.v[0][last][:, 3::4])
    assert E.device_status(0) == 0
    c.free()
    other.free()
