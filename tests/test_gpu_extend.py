"""GPU: attention of several new tokens per cache (eakv_extend_attention)
against a plain softmax in 64 bits over the cache's own dequantized values."""
import numpy as np
import pytest

import eakv_b200 as E
from gpu_util import bits, kv_data

pytestmark = pytest.mark.gpu

DT = {"f32": "float32", "f16": "float16", "bf16": "bfloat16"}
HALF_STEP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}


# both kernels on every case: the library's choice (few rows: warp-level
# kernel, many: tcgen05), or one of them for 16-bit types
PATH = "auto"
CODE = {"auto": 0, "mma": 2, "umma": 3}


@pytest.fixture(autouse=True)
def _reset(request):
    global PATH
    PATH = request.node.callspec.params.get("path", "auto") if hasattr(request.node, "callspec") else "auto"
    E.force_splits(0)
    E.force_path(CODE[PATH])
    yield
    E.force_splits(0)
    E.force_path(0)
    E.test_stall(-1)
    PATH = "auto"


class Batch:
    """Caches of L layers holding old + new positions, the new ones not yet
    advanced over, and their values in 64 bits."""

    def __init__(self, rng, L, H, hd, old, new, size=None, data=None):
        self.old, self.new, self.H, self.hd = old, new, H, hd
        size = size or max(a + b for a, b in zip(old, new))
        self.caches, self.k, self.v, self.step = [], [], [], []
        for i, (a, b) in enumerate(zip(old, new)):
            c = E.Cache(L, H, hd, max(size, 1))
            n = a + b
            d = kv_data(rng, L, H, max(n, 1), hd) if data is None else data[i]
            if n:
                assert c.load_raw(d[:, :, :, :n], n) == 0
            self.k.append([c.dequantize(l, 0, 0, n).astype(np.float64) for l in range(L)])
            self.v.append([c.dequantize(l, 1, 0, n).astype(np.float64) for l in range(L)])
            self.caches.append(c)
            assert c.restore(a) == 0

    def free(self):
        for c in self.caches:
            c.free()


def allowed(old, n, window=0, tree=None):
    i, j = np.arange(n)[:, None], np.arange(old + n)[None, :]
    ok = j < old if tree is not None else j <= old + i
    ok = np.broadcast_to(ok, (n, old + n)).copy()
    if tree is not None:
        for t in range(n):
            for b in range(n):
                ok[t, old + b] = (int(tree[t]) >> b) & 1
    if window:
        ok &= j > old + i - window
    return ok


def plain(batch, layer, q, scale, window=0, tree=None):
    """(out, lse, size): f64 attention [total, nq, hd], and for the tolerance
    per row: sum_j p_j max|v_j| and the largest sum_i |q_i k_i| scale."""
    total, nq, hd = q.shape
    G = nq // batch.H
    out, lse = np.zeros((total, nq, hd)), np.full((total, nq), -np.inf)
    vmean, reach = np.zeros((total, nq)), np.zeros((total, nq))
    first = 0
    for b, (a, n) in enumerate(zip(batch.old, batch.new)):
        if n == 0:
            continue
        ok = allowed(a, n, window, None if tree is None else tree[first:first + n])
        for h in range(nq):
            k, v = batch.k[b][layer][h // G], batch.v[b][layer][h // G]
            qq = q[first:first + n, h].astype(np.float64)
            with np.errstate(invalid="ignore", over="ignore"):
                s = qq @ k.T * scale
            s = np.where(ok, s, -np.inf)
            m = s.max(1)
            m0 = np.where(np.isfinite(m), m, 0.0)
            p = np.where(ok, np.exp(s - m0[:, None]), 0.0)
            l = p.sum(1)
            some = l > 0
            pn = p / np.where(some, l, 1.0)[:, None]
            out[first:first + n, h] = np.where(pn[:, :, None] != 0, pn[:, :, None] * v, 0.0).sum(1) if n * len(v) * hd < 4e6 \
                else pn @ v
            with np.errstate(divide="ignore"):
                lse[first:first + n, h] = np.where(some, m0 + np.log(l), -np.inf)
            vmean[first:first + n, h] = pn @ np.abs(v).max(1)
            reach[first:first + n, h] = (np.abs(qq) @ np.abs(k).T * np.where(ok, 1, 0)).max(1) * abs(scale)
        first += n
    return out, lse, (vmean, reach)


def limits(dtype, out, size, rows_per_head, longest):
    """What the kernel's roundings allow.
    Scores: f32 sums of exact products of the rounded operands. Operands of
    22 bits (f32) leave 2^-22 of sum |q k| <= reach, and 128 additions in f32
    with truncation 128 2^-23 = 2^-16 of it at worst; K in f16 (the 16-bit types
    with many rows: value and scale rounded) leaves 3 2^-11. A score off by d
    moves every weight by a factor within e^(2d), the output by 2 d vmean.
    Outputs: weights of 22 bits or 2^-11 (f16, half a step), V in f16 another
    3 2^-11 of every term; the centred nibbles and bias of a value sum to at
    most 4 max|v| in absolute terms; truncated f32 sums 2^-23 per step of 16
    positions, at most `longest` / 64 steps per warp and 256 for the merge.
    Then half a step of the output's type."""
    vmean, reach = size
    wide = dtype != "f32" and (PATH == "umma" or (PATH == "auto" and rows_per_head > 32))
    d = reach * (2.0 ** -16 + (3 * 2.0 ** -11 if wide else 0.0))
    w = (2.0 ** -22 if dtype == "f32" else 2.0 ** -11) + (3 * 2.0 ** -11 if wide else 0.0)
    w += (longest / 64 + 256) * 2.0 ** -23
    lim = (2 * d + 4 * w) * vmean
    return lim[:, :, None] + HALF_STEP[dtype] * np.abs(out), d + 2.0 ** -16


def run(gpu, batch, layer, q, dtype, nq, lse=True, **kw):
    """The call on device tensors -> (out, lse) on the host."""
    import torch
    dq = torch.from_numpy(q).to(gpu).to(getattr(torch, DT[dtype]))
    out = torch.full_like(dq, float("nan"))
    dl = torch.full(dq.shape[:2], float("nan"), device=gpu) if lse else None
    torch.cuda.synchronize()
    E.extend_attention(batch.caches, layer, batch.new, dq, out, lse=dl, **kw)
    batch.caches[0].synchronize()
    return out.double().cpu().numpy(), (dl.double().cpu().numpy() if lse else None)


def rounded(q, dtype):
    import torch
    return torch.from_numpy(q).to(getattr(torch, DT[dtype])).float().numpy()


def check(gpu, batch, layer, q, dtype, nq, window=0, tree=None, scale=0.0, **kw):
    import torch
    sc = scale or 1.0 / np.sqrt(batch.hd)
    dt = None if tree is None else torch.from_numpy(tree.astype(np.int64)).to(gpu)
    got, lse = run(gpu, batch, layer, q, dtype, nq, window=window, tree=dt, scale=scale, **kw)
    want, wl, size = plain(batch, layer, rounded(q, dtype), sc, window, tree)
    lim, ll = limits(dtype, want, size, max(batch.new) * nq // batch.H,
                     max(a + b for a, b in zip(batch.old, batch.new)))
    err = np.abs(got - want)
    assert (err <= lim).all(), f"worst {np.nanmax(err / lim)} of the limit, nan {np.isnan(got).sum()}"
    assert np.array_equal(np.isneginf(lse), np.isneginf(wl))
    live = ~np.isneginf(wl)
    assert (np.abs(lse[live] - wl[live]) <= (ll + 2.0 ** -22 * np.abs(wl))[live]).all()
    assert E.device_status(0) == 0
    return float(np.max(err / np.where(lim > 0, lim, 1))) if err.size else 0.0


CASES = [
    # hd, nq, nkv, old, new
    (128, 8, 2, [0], [1]),
    (128, 8, 2, [63], [1]),
    (64, 32, 4, [64], [2]),
    (128, 32, 8, [700, 0, 129], [5, 3, 1]),
    (64, 7, 1, [100, 31], [3, 9]),
    (128, 12, 4, [40], [0]),
    (128, 12, 4, [40, 3], [0, 11]),
    (128, 4, 4, [0, 130], [65, 17]),
    (64, 8, 8, [1000], [33]),
    (128, 16, 1, [500], [19]),
    (128, 8, 2, [1], [200]),
    (64, 6, 2, [60, 0, 5], [130, 64, 257]),
    (128, 8, 8, [300], [129]),
    (128, 40, 2, [77], [31]),
]


KINDS = [("f32", "auto"), ("f16", "auto"), ("bf16", "auto"), ("bf16", "mma"), ("bf16", "umma")]


@pytest.mark.parametrize("dtype,path", KINDS)
@pytest.mark.parametrize("hd,nq,nkv,old,new", CASES)
def test_causal(gpu, hd, nq, nkv, old, new, dtype, path):
    rng = np.random.default_rng(hd + nq + sum(old))
    b = Batch(rng, 2, nkv, hd, old, new, size=max(x + y for x, y in zip(old, new)) + 5)
    q = rng.standard_normal((sum(new), nq, hd)).astype(np.float32)
    if sum(new):
        check(gpu, b, 1, q, dtype, nq)
    b.free()


@pytest.mark.parametrize("dtype,path", KINDS)
@pytest.mark.parametrize("window", [1, 2, 63, 64, 65, 128, 300])
@pytest.mark.parametrize("hd,nq,nkv,old,new", [(128, 8, 2, [500, 10], [3, 1]), (64, 8, 4, [200], [70]),
                                               (128, 4, 1, [131, 0], [100, 90])])
def test_window(gpu, hd, nq, nkv, old, new, window, dtype, path):
    rng = np.random.default_rng(window)
    b = Batch(rng, 1, nkv, hd, old, new)
    q = rng.standard_normal((sum(new), nq, hd)).astype(np.float32)
    check(gpu, b, 0, q, dtype, nq, window=window)
    b.free()


@pytest.mark.parametrize("dtype,path", KINDS)
@pytest.mark.parametrize("window", [0, 40])
@pytest.mark.parametrize("hd,nq,nkv,old,new", [(128, 8, 2, [0], [1]), (64, 8, 1, [100, 0], [13, 64]),
                                               (128, 8, 8, [61], [9]), (128, 32, 8, [63, 128], [64, 40])])
def test_tree(gpu, hd, nq, nkv, old, new, window, dtype, path):
    """Random masks: tokens that attend none, one or all of the new tokens,
    later ones too; with no cached position a token may attend nothing."""
    rng = np.random.default_rng(hd + sum(new) + window)
    b = Batch(rng, 1, nkv, hd, old, new)
    masks = []
    for n in new:
        m = rng.integers(0, 2 ** 63, n, dtype=np.uint64) * np.uint64(2) + rng.integers(0, 2, n, dtype=np.uint64)
        m &= np.uint64((1 << n) - 1)
        m[::4] = 0
        if n > 2:
            m[2] = (1 << n) - 1
        masks.append(m)
    q = rng.standard_normal((sum(new), nq, hd)).astype(np.float32)
    check(gpu, b, 0, q, dtype, nq, window=window, tree=np.concatenate(masks))
    b.free()


@pytest.mark.parametrize("dtype,path", KINDS)
@pytest.mark.parametrize("splits", [2, 3, 7, 50])
def test_forced_splits_and_own_workspace(gpu, splits, dtype, path):
    """Splits of any length, with the cache's scratch and with a workspace of
    the caller's, three calls on it: the same bits each time."""
    import torch
    rng = np.random.default_rng(splits)
    b = Batch(rng, 1, 2, 128, [1300, 40], [7, 2])
    q = rng.standard_normal((9, 8, 128)).astype(np.float32)
    E.force_splits(splits)
    check(gpu, b, 0, q, dtype, 8)
    need = E.extend_workspace(b.caches, b.new, getattr(E, "EAKV_" + dtype.upper()), 8)
    assert need > 0
    ws = torch.zeros(need, dtype=torch.uint8, device=gpu)
    first, _ = run(gpu, b, 0, q, dtype, 8)
    for _ in range(3):
        got, _ = run(gpu, b, 0, q, dtype, 8, workspace=ws)
        assert np.array_equal(got, first)
    with pytest.raises(E.EakvError, match="workspace"):
        run(gpu, b, 0, q, dtype, 8, workspace=ws[:need - 16])
    b.free()


@pytest.mark.parametrize("dtype,path", KINDS)
@pytest.mark.parametrize("new", [[4], [150]])
def test_what_is_not_attended_has_no_influence(gpu, new, dtype, path):
    """NaN and infinities in later tokens, in a tree's siblings, before the
    window and behind the appended tokens leave the bits as they were; where
    they are attended, the outputs are NaN."""
    import torch
    rng = np.random.default_rng(5)
    H, hd, nq, old = 2, 128, 8, 70
    n = new[0]
    data = kv_data(rng, 1, H, 300, hd)
    clean = Batch(rng, 1, H, hd, [old], new, size=300, data=[data])
    q = rng.standard_normal((n, nq, hd)).astype(np.float32)
    want, wl = run(gpu, clean, 0, q, dtype, nq)
    dirty = data.copy()
    t = n - 2                                    # spoil the last two tokens' K and V
    dirty[:, :, :, old + t:] = np.nan
    dirty[:, :, :, old + n - 1:, ::3] = np.inf
    bad = Batch(rng, 1, H, hd, [old], new, size=300, data=[dirty])
    # and what lies behind them in the pages
    c = bad.caches[0]
    c.restore(0)
    assert c.load_raw(dirty, 300) == 0
    c.restore(old)
    got, gl = run(gpu, bad, 0, q, dtype, nq)
    assert np.array_equal(got[:t], want[:t]) and np.array_equal(gl[:t], wl[:t])
    assert np.isnan(got[t:]).all()
    # only one group of one head's V: its dims alone
    spot = data.copy()
    spot[0, 1, 1, old + n - 1, 64:] = np.nan
    b3 = Batch(rng, 1, H, hd, [old], new, size=300, data=[spot])
    got, gl = run(gpu, b3, 0, q, dtype, nq)
    assert np.array_equal(got[:-1], want[:-1]) and np.array_equal(gl, wl)
    assert np.array_equal(got[-1, :4], want[-1, :4])
    assert np.isnan(got[-1, 4:, 64:]).all()
    # the spoiled group's scale is 1 and attended: it may move the power of two
    # that the weights are held by, so each of them rounds anew, to 22 bits (f16
    # otherwise) of max|v| < 8 at most, and the output to its type
    off = np.abs(got[-1, 4:, :64] - want[-1, 4:, :64])
    assert (off <= (2.0 ** -22 if dtype == "f32" else 2.0 ** -11) * 2 * 8
            + 2 * HALF_STEP[dtype] * np.abs(want[-1, 4:, :64])).all()
    # before the window
    spot = data.copy()
    spot[:, :, :, :40] = np.nan
    b4 = Batch(rng, 1, H, hd, [old], new, size=300, data=[spot])
    w4, _ = run(gpu, clean, 0, q, dtype, nq, window=30)
    got, _ = run(gpu, b4, 0, q, dtype, nq, window=30)
    assert np.array_equal(got, w4)
    # an infinity or NaN in one query row
    q2 = q.copy()
    q2[0, 0, 3], q2[1, 5, 100] = np.inf, np.nan
    got, _ = run(gpu, clean, 0, q2, dtype, nq)
    assert np.isnan(got[0, 0]).all() and np.isnan(got[1, 5]).all()
    keep = np.ones((n, nq), bool)
    keep[0, 0] = keep[1, 5] = False
    assert np.array_equal(got[keep], want[keep])
    for x in (clean, bad, b3, b4):
        x.free()
    assert E.device_status(0) == 0


@pytest.mark.parametrize("dtype,path", [k for k in KINDS if k[0] != "f16"])   # f16 holds no 1e20
@pytest.mark.parametrize("n", [3, 160])
@pytest.mark.parametrize("kscale,vscale,qscale", [(1, 1e-30, 1), (1, 1e30, 1), (1e-20, 1, 1e20), (1e20, 1, 1e-20),
                                                  (1, 1e4, 1e-6), (1, 1, 30.0)])
def test_magnitudes(gpu, n, kscale, vscale, qscale, dtype, path):
    """Values over 60 orders of magnitude, and V growing 2^14 along the sequence."""
    rng = np.random.default_rng(17)
    H, hd, nq, old = 2, 128, 8, 300
    data = kv_data(rng, 1, H, old + n, hd)
    data[:, 0] *= np.float32(kscale)
    data[:, 1] *= np.float32(vscale)
    data[:, 1, :, 150:] *= np.float32(2.0 ** 14 if vscale <= 1 else 16.0)
    b = Batch(rng, 1, H, hd, [old], [n], data=[data])
    q = (rng.standard_normal((n, nq, hd)) * qscale).astype(np.float32)
    check(gpu, b, 0, q, dtype, nq)
    b.free()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_strides_scale_and_lengths(gpu, dtype):
    """q and out as slices of wider buffers, at odd addresses too; a scale of
    the caller's, a negative one among them; seq_len 0 with one token."""
    import torch
    rng = np.random.default_rng(23)
    H, hd, nq, new = 2, 64, 6, [3, 50]
    b = Batch(rng, 1, H, hd, [9, 0], new)
    total = sum(new)
    q = rng.standard_normal((total, nq, hd)).astype(np.float32)
    base, _ = run(gpu, b, 0, q, dtype, nq)
    tdt = getattr(torch, DT[dtype])
    for pad, off in ((8, 4), (3, 1)):
        wide = torch.zeros(total, nq, hd + pad, dtype=tdt, device=gpu)
        wide[..., off:off + hd] = torch.from_numpy(q).to(gpu).to(tdt)
        room = torch.full((total, nq + 2, hd + pad), 3.0, dtype=tdt, device=gpu)
        torch.cuda.synchronize()
        E.extend_attention(b.caches, 0, new, wide[..., off:off + hd], room[:, 1:nq + 1, off:off + hd])
        b.caches[0].synchronize()
        assert np.array_equal(room[:, 1:nq + 1, off:off + hd].double().cpu().numpy(), base)
        room[:, 1:nq + 1, off:off + hd] = 3.0
        assert (room == 3.0).all()               # nothing else was written
    for scale in (0.03, -0.2):
        check(gpu, b, 0, q, dtype, nq, scale=scale)
    b.free()


def test_rows_and_neighbours_agree(gpu):
    """A token's result does not depend on how the tokens are grouped: one call
    with all of them against one call each (the same kernel, f32)."""
    rng = np.random.default_rng(31)
    H, hd, nq, old, n = 2, 128, 8, 200, 6
    data = [kv_data(rng, 1, H, old + n, hd)]
    b = Batch(rng, 1, H, hd, [old], [n], data=data)
    q = rng.standard_normal((n, nq, hd)).astype(np.float32)
    whole, _ = run(gpu, b, 0, q, "f32", nq)
    for t in range(n):
        one = Batch(rng, 1, H, hd, [old + t], [1], data=data)
        got, _ = run(gpu, one, 0, q[t:t + 1], "f32", nq)
        np.testing.assert_allclose(got[0], whole[t], rtol=0, atol=2.0 ** -17 * np.abs(whole).max())
        one.free()
    b.free()


def test_graph_capture_and_streams(gpu):
    """Captured with a workspace of its own and replayed on a stream; with the
    scratch, a captured call that needs one is refused."""
    import torch
    rng = np.random.default_rng(41)
    b = Batch(rng, 1, 2, 128, [2000], [4])
    q = rng.standard_normal((4, 8, 128)).astype(np.float32)
    E.force_splits(5)
    want, _ = run(gpu, b, 0, q, "bf16", 8, lse=False)
    dq = torch.from_numpy(q).to(gpu).bfloat16()
    out = torch.zeros_like(dq)
    ws = torch.zeros(E.extend_workspace(b.caches, [4], E.EAKV_BF16, 8), dtype=torch.uint8, device=gpu)
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        E.extend_attention(b.caches, 0, [4], dq, out, workspace=ws, stream=s.cuda_stream)
    for _ in range(3):
        out.zero_()
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert np.array_equal(out.double().cpu().numpy(), want)
    del g
    E.force_splits(0)
    b.free()
    assert E.device_status(0) == 0


def test_a_wait_that_runs_out_is_reported(gpu):
    """A page that is never requested: status bit 1, and the next call is right."""
    rng = np.random.default_rng(43)
    b = Batch(rng, 1, 2, 128, [600], [3])
    q = rng.standard_normal((3, 8, 128)).astype(np.float32)
    want, _ = run(gpu, b, 0, q, "f32", 8)
    for splits in (1, 3):
        E.force_splits(splits)
        first, _ = run(gpu, b, 0, q, "f32", 8)
        E.test_stall(1, 2000)
        run(gpu, b, 0, q, "f32", 8)
        E.test_stall(-1)
        assert E.device_status(0, reset=True) == 1
        again, _ = run(gpu, b, 0, q, "f32", 8)
        assert np.array_equal(again, first)
    b.free()


def test_refusals(gpu):
    import torch
    rng = np.random.default_rng(47)
    b = Batch(rng, 2, 2, 128, [10], [4], size=14)
    c = b.caches
    q = torch.zeros(4, 8, 128, device=gpu)
    out = torch.zeros_like(q)

    def no(*args, **kw):
        with pytest.raises((E.EakvError, ValueError, TypeError)):
            E.extend_attention(*args, **kw)

    five = torch.zeros(5, 8, 128, device=gpu)
    no(c, 0, [5], five, five)                     # beyond max_seq_len
    no(c, 0, [-1], q, out)
    no(c, 2, [4], q, out)
    no(c, -1, [4], q, out)
    no(c, 0, [4], q[:, :3], out[:, :3])           # 3 query heads over 2
    no(c, 0, [4], q, out.half())
    no(c, 0, [4], q.double(), out.double())
    no(c, 0, [4], q, out, window=-1)
    no(c, 0, [4], q, out, scale=float("nan"))
    no(c, 0, [4], q, out, scale=float("inf"))
    no(c, 0, [4], q.cpu(), out)
    no(c, 0, [4], q, out, tree=torch.zeros(3, dtype=torch.int64, device=gpu))
    no(c, 0, [4], q, out, lse=torch.zeros(4, 7, device=gpu))
    no(c, 0, [2, 2], q, out)
    big = E.Cache(1, 2, 128, 80)
    many = torch.zeros(65, 2, 128, device=gpu)
    no([big], 0, [65], many, many, tree=torch.zeros(65, dtype=torch.int64, device=gpu))
    wide = E.Cache(1, 1, 256, 8)
    x = torch.zeros(1, 1, 256, device=gpu)
    no([wide], 0, [1], x, x)
    E.extend_attention(c, 0, [0], q[:0], out[:0])
    big.free()
    wide.free()
    b.free()
    assert E.device_status(0) == 0
