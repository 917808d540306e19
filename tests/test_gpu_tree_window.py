"""GPU: token trees under a sliding window that goes by positions
(eakv_extend_attention_depths)."""
import ctypes

import numpy as np
import pytest

import eakv_b200 as E
from gpu_util import kv_data
from test_gpu_extend import CODE, DT, KINDS, Batch, limits, rounded

import test_gpu_extend

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _path(request):
    path = request.node.callspec.params.get("path", "auto") if hasattr(request.node, "callspec") else "auto"
    test_gpu_extend.PATH = path
    E.force_path(CODE[path])
    E.force_splits(0)
    yield
    test_gpu_extend.PATH = "auto"
    E.force_path(0)
    E.force_splits(0)


def tree(rng, n, deep):
    """(masks, depths, parents) of a random tree; deep: long branches."""
    mask, depth, parent = [], [], []
    for t in range(n):
        p = -1 if t == 0 else int(rng.integers(max(0, t - 2) if deep else 0, t))
        parent.append(p)
        mask.append(1 << t | (mask[p] if p >= 0 else 0))
        depth.append(depth[p] + 1 if p >= 0 else 0)
    return mask, depth, parent


def plain(b, q, scale, window, masks, depths):
    """64-bit outputs, LSE, and for the limits sum_j p_j max|v_j| and the largest sum |q k| scale."""
    nq = q.shape[1]
    out, lse = np.zeros(q.shape), np.full(q.shape[:2], -np.inf)
    vmean, reach = np.zeros(q.shape[:2]), np.zeros(q.shape[:2])
    first = 0
    for i, (old, n) in enumerate(zip(b.old, b.new)):
        for t in range(n):
            m, d = int(masks[first + t]), depths[first + t]
            at = [j for j in range(old) if not window or j > old + d - window]
            at += [old + j for j in range(n) if m >> j & 1 and (not window or depths[first + j] > d - window)]
            if not at:
                continue
            for h in range(nq):
                k, v = (x[i][0][h * b.H // nq][at] for x in (b.k, b.v))
                x = q[first + t, h].astype(np.float64)
                s = k @ x * scale
                p = np.exp(s - s.max())
                out[first + t, h], lse[first + t, h] = p @ v / p.sum(), s.max() + np.log(p.sum())
                vmean[first + t, h] = p @ np.abs(v).max(1) / p.sum()
                reach[first + t, h] = (np.abs(k) @ np.abs(x)).max() * scale
        first += n
    return out, lse, (vmean, reach)


def call(gpu, b, q, dtype, masks, depths, window, **kw):
    import torch
    dq = torch.from_numpy(q).to(gpu).to(getattr(torch, DT[dtype]))
    out, lse = torch.full_like(dq, float("nan")), torch.full(q.shape[:2], float("nan"), device=gpu)
    t = torch.from_numpy(np.array(masks, np.uint64).astype(np.int64)).to(gpu)
    d = torch.tensor(depths, dtype=torch.int32, device=gpu)
    torch.cuda.synchronize()
    E.extend_attention(b.caches, 0, b.new, dq, out, window=window, tree=t, depth=d, lse=lse, **kw)
    b.caches[0].synchronize()
    return out.double().cpu().numpy(), lse.double().cpu().numpy()


@pytest.mark.parametrize("dtype,path", KINDS)
@pytest.mark.parametrize("window", [0, 1, 2, 9, 40, 70, 300])
@pytest.mark.parametrize("hd,nq,nkv,old,new", [(128, 8, 2, [100, 0], [13, 64]), (64, 8, 1, [61, 300], [9, 40])])
def test_depths(gpu, hd, nq, nkv, old, new, window, dtype, path):
    rng = np.random.default_rng(window + hd)
    b = Batch(rng, 1, nkv, hd, old, new)
    masks, depths = [], []
    for n in new:
        m, d, _ = tree(rng, n, deep=n > 20)
        masks += m
        depths += d
    q = rounded(rng.standard_normal((sum(new), nq, hd)).astype(np.float32), dtype)
    got, lse = call(gpu, b, q, dtype, masks, depths, window)
    want, wl, size = plain(b, q, hd ** -0.5, window, masks, depths)
    lim, ll = limits(dtype, want, size, max(new) * nq // nkv, max(old) + max(new))
    assert (np.abs(got - want) <= lim).all()
    assert (np.abs(lse - wl) <= ll + 2.0 ** -22 * np.abs(wl)).all()
    # split and with a workspace of the query's size, the same rows
    import torch
    E.force_splits(3)
    need = E.extend_workspace(b.caches, new, getattr(E, "EAKV_" + dtype.upper()), nq, window, True, True)
    ws = torch.zeros(need, dtype=torch.uint8, device=gpu) if need else None
    got, _ = call(gpu, b, q, dtype, masks, depths, window, workspace=ws)
    assert (np.abs(got - want) <= lim).all()
    b.free()
    assert E.device_status(0) == 0


@pytest.mark.parametrize("dtype,path", KINDS)
@pytest.mark.parametrize("window", [5, 24, 90])
def test_an_accepted_branch_is_what_its_tokens_attend_one_by_one(gpu, window, dtype, path):
    """The rows of a branch in the tree's call, against the branch's tokens appended and attended one
    after the other under the same window."""
    import torch
    rng = np.random.default_rng(window)
    H, hd, nq, old, n = 2, 64, 8, 100, 30
    data = kv_data(rng, 1, H, old + n, hd)
    b = Batch(rng, 1, H, hd, [old], [n], data=[data])
    masks, depths, parent = tree(rng, n, deep=True)
    q = rounded(rng.standard_normal((n, nq, hd)).astype(np.float32), dtype)
    got, _ = call(gpu, b, q, dtype, masks, depths, window)
    branch, t = [], int(np.argmax(depths))
    while t >= 0:
        branch.insert(0, t)
        t = parent[t]
    assert len(branch) > 10
    want, _, size = plain(b, q, hd ** -0.5, window, masks, depths)
    lim, _ = limits(dtype, want, size, n * nq // H, old + n)
    c = E.Cache(1, H, hd, old + n)
    assert c.load_raw(np.ascontiguousarray(data[:, :, :, :old]), old) == 0
    for t in branch:
        for kv in (0, 1):
            assert c.append(np.ascontiguousarray(data[0, kv, :, old + t:old + t + 1]), 0, kv, 1) == 0
        x = torch.from_numpy(q[t:t + 1]).to(gpu).to(getattr(torch, DT[dtype]))
        one = torch.empty_like(x)
        torch.cuda.synchronize()
        E.extend_attention([c], 0, [1], x, one, window=window)
        c.synchronize()
        assert c.advance(1) == 0
        assert (np.abs(got[t] - one[0].double().cpu().numpy()) <= 2 * lim[t]).all()
    c.free()
    b.free()


def test_depths_out_of_range_and_refusals(gpu):
    """A depth outside [0, t] is reported and counts as t; depths want a tree and alignment."""
    import torch
    rng = np.random.default_rng(1)
    b = Batch(rng, 1, 2, 128, [50], [6])
    masks = [(2 << t) - 1 for t in range(6)]
    q = rng.standard_normal((6, 4, 128)).astype(np.float32)
    right, _ = call(gpu, b, q, "f32", masks, [0, 1, 2, 3, 4, 5], 10)
    for bad in ([0, 2, 2, 3, 4, 5], [0, 1, 2, -1, 4, 5], [0, 1, 2, 3, 4, 2 ** 31 - 1], [0, 1, -2 ** 31, 3, 4, 5]):
        got, _ = call(gpu, b, q, "f32", masks, bad, 10)
        assert E.device_status(0, reset=True) == 2
        assert np.array_equal(got, right)
    dq = torch.from_numpy(q).to(gpu)
    t = torch.tensor(masks, dtype=torch.int64, device=gpu)
    d = torch.arange(6, dtype=torch.int32, device=gpu)
    for kw in (dict(depth=d), dict(tree=t, depth=d[:5]), dict(tree=t, depth=d.long()), dict(tree=t, depth=d.cpu())):
        with pytest.raises((E.EakvError, ValueError)):
            E.extend_attention(b.caches, 0, [6], dq, dq, window=4, **kw)
    rows = E._Rows(dq.data_ptr(), 4 * 128, 128, E.EAKV_F32)
    hs, n = (ctypes.c_void_p * 1)(b.caches[0].h), (ctypes.c_int * 1)(6)
    rc = E.lib().eakv_extend_attention_depths(hs, 1, 0, n, ctypes.byref(rows), ctypes.byref(rows), 4, 0.0, 4,
                                              t.data_ptr(), d.data_ptr() + 2, None, None, 0, None)
    assert rc == E.EAKV_ERR_INVALID
    b.free()
    assert E.device_status(0) == 0
