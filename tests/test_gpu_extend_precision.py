"""GPU: how far eakv_extend_attention is off on the whole. Beside the worst case that
test_gpu_extend.py allows stands the root mean square that the kernels' roundings give when
each is as likely up as down; a mistake in one page, group or token passes the first and
not the second."""
import numpy as np
import pytest

import eakv_b200 as E
from test_gpu_extend import CODE, HALF_STEP, Batch, allowed, rounded, run

pytestmark = pytest.mark.gpu

KINDS = [("f32", "auto"), ("f16", "mma"), ("bf16", "mma"), ("f16", "umma"), ("bf16", "umma")]


@pytest.fixture(autouse=True)
def _path(request):
    E.force_splits(0)
    E.force_path(CODE[request.node.callspec.params["path"]])
    yield
    E.force_splits(0)
    E.force_path(0)


def groups(x):
    """(s, b + 8 s) of dequantized rows [n, hd]: a group's smallest value has nibble 0 and
    its largest 15."""
    g = x.reshape(len(x), -1, 64)
    lo, hi = g.min(2), g.max(2)
    s = (hi - lo) / 15
    return s, lo + 8 * s


def expected(b, q, dtype, path, window=0, tree=None, without=None):
    """64-bit outputs and LSE, and the root mean square of their errors.

    A rounding to f16 is off by half a step at most, 2^-11 of the value, evenly spread: 2^-11 / sqrt 3 of
    it at most in the mean square (u below). Independent errors add as squares:
    - scores: the warp-level kernel keeps K's nibbles, f32 sums are off by 2^-18 of sum |q k|. In
      the tcgen05 kernel every k = m s_hi + (m s_lo + r) is rounded once, its second term (below 3/4 s)
      before that, and r (below s/2), which all dims of a group share.
    - a score off by d moves an output by p d (v - o), the LSE by p d.
    - weights: 2^-11 of p (16-bit types) or 2^-22, on s n' in the warp-level kernel, on v in the other,
      where v itself is m s + r with s and r rounded, and then the sum.
    - the output: its type's half step; sums of both kernels 2^-17 of it.
    `without`: (cache, first, last, what) is left out of the oracle: positions of the cache, or of V's
    second half ("v": doubled)."""
    u2 = 2.0 ** -22 / 3
    wide, total, nq = path == "umma", len(q), q.shape[1]
    weight2 = 2.0 ** -44 if dtype == "f32" else u2
    G, scale = nq // b.H, b.hd ** -0.5
    out, lse = np.zeros(q.shape), np.zeros((total, nq))
    var, lvar = np.zeros(q.shape), np.zeros((total, nq))
    first = 0
    for i, (old, n) in enumerate(zip(b.old, b.new)):
        ok = allowed(old, n, window, None if tree is None else tree[first:first + n])
        rows = slice(first, first + n)
        for h in range(nq):
            k, v = b.k[i][0][h // G], b.v[i][0][h // G].copy()
            (ks, _), (vs, vb) = groups(k), groups(v)
            if without and without[0] == i:
                if without[3] == "v":
                    v[without[1]:without[2], b.hd // 2:] *= 2
                else:
                    ok = ok.copy()
                    ok[:, without[1]:without[2]] = False
            x = q[rows, h].astype(np.float64)
            s = np.where(ok, x @ k.T * scale, -np.inf)
            m = s.max(1, keepdims=True)
            p = np.exp(s - m)
            l = p.sum(1, keepdims=True)
            p /= l
            o = p @ v
            out[rows, h], lse[rows, h] = o, (m + np.log(l))[:, 0]
            if wide:
                ksd = np.repeat(ks, 64, axis=1)
                qsum = np.stack([x[:, 64 * g:64 * g + 64].sum(1) for g in range(b.hd // 64)], 1)
                d2 = u2 * scale ** 2 * (x ** 2 @ (k ** 2 + (0.75 * ksd) ** 2).T + qsum ** 2 @ (0.5 * ks).T ** 2)
                held = v ** 2
                vsd = np.repeat(vs, 64, axis=1)
                v2 = u2 * (2 * v ** 2 + (0.5 * vsd) ** 2)
            else:
                d2 = (2.0 ** -18 * scale * np.abs(x) @ np.abs(k).T) ** 2
                held = (v - np.repeat(vb, 64, axis=1)) ** 2
                v2 = 0 * v
            pd = p ** 2 * d2
            var[rows, h] = (pd @ v ** 2 - 2 * o * (pd @ v) + o ** 2 * pd.sum(1, keepdims=True)
                            + weight2 * (p ** 2 @ held) + p ** 2 @ v2 + (HALF_STEP[dtype] ** 2 / 3 + 2.0 ** -34) * o ** 2)
            lvar[rows, h] = pd.sum(1) + 2.0 ** -40
        first += n
    return out, lse, var, lvar


def ratios(got, lse, e):
    """Root mean square errors of outputs and LSE as shares of what is expected, per query head: the worst."""
    out, wl, var, lvar = e
    return (np.sqrt(((got - out) ** 2).mean((0, 2)) / var.mean((0, 2))).max(),
            np.sqrt(((lse - wl) ** 2).mean(0) / lvar.mean(0)).max())


SHAPES = [
    # hd, nq, nkv, old, new, window
    (128, 8, 2, [700], [120], 0),
    (64, 8, 4, [900, 0], [70, 130], 0),
    (128, 4, 4, [2000, 300], [40, 90], 500),
    (64, 14, 2, [63], [200], 0),
]


@pytest.mark.parametrize("dtype,path", KINDS)
@pytest.mark.parametrize("hd,nq,nkv,old,new,window", SHAPES)
def test_root_mean_square(gpu, hd, nq, nkv, old, new, window, dtype, path):
    """Within 5/4 of what is expected (an upper estimate: values spread between the powers of two that
    their steps go by make it 3/4 of that), and far from it when the oracle leaves out 16 positions or
    doubles half of V there."""
    rng = np.random.default_rng(hd + nq)
    b = Batch(rng, 1, nkv, hd, old, new)
    q = rounded(rng.standard_normal((sum(new), nq, hd)).astype(np.float32), dtype)
    got, lse = run(gpu, b, 0, q, dtype, nq, window=window)
    r, rl = ratios(got, lse, expected(b, q, dtype, path, window))
    assert r <= 1.25 and rl <= 1.25, (r, rl)
    at = old[0] - 20
    r, rl = ratios(got, lse, expected(b, q, dtype, path, window, without=(0, at, at + 16, "k")))
    assert r > 3 and rl > 3, (r, rl)
    r, _ = ratios(got, lse, expected(b, q, dtype, path, window, without=(0, at, at + 16, "v")))
    assert r > 3, r
    b.free()
    assert E.device_status(0) == 0


@pytest.mark.parametrize("dtype,path", KINDS)
def test_root_mean_square_of_trees(gpu, dtype, path):
    import torch
    rng = np.random.default_rng(9)
    old, new, nq = [400, 5], [40, 64], 8
    b = Batch(rng, 1, 2, 128, old, new)
    masks = []
    for n in new:
        m = []
        for t in range(n):
            m.append((1 << t) | (m[rng.integers(t)] if t else 0))
        masks += m
    tree = np.array(masks, np.uint64)
    q = rounded(rng.standard_normal((sum(new), nq, 128)).astype(np.float32), dtype)
    got, lse = run(gpu, b, 0, q, dtype, nq, tree=torch.from_numpy(tree.astype(np.int64)).to(gpu))
    r, rl = ratios(got, lse, expected(b, q, dtype, path, tree=tree))
    assert r <= 1.25 and rl <= 1.25, (r, rl)
    wrong = tree.copy()
    wrong[10] ^= np.uint64(1)     # the first new token's bit of one row
    r, _ = ratios(got[10:11], lse[10:11], [a[10:11] for a in expected(b, q, dtype, path, tree=wrong)])
    assert r > 3, r
    b.free()


@pytest.mark.parametrize("dtype,path", [("bf16", "auto"), ("f16", "umma")])
def test_a_build_without_the_tcgen05_kernel(gpu, dtype, path):
    """A register count that the kernel's warpgroups cannot trade: calls of many rows run on the
    warp-level kernel, with its bits."""
    rng = np.random.default_rng(2)
    b = Batch(rng, 1, 2, 128, [300, 10], [100, 3])
    q = rounded(rng.standard_normal((103, 8, 128)).astype(np.float32), dtype)
    here, _ = run(gpu, b, 0, q, dtype, 8)
    E.force_path(CODE["mma"])
    want, wl = run(gpu, b, 0, q, dtype, 8)
    E.force_path(CODE[path])
    E.extend_registers(120)
    try:
        need = E.extend_workspace(b.caches, b.new, getattr(E, "EAKV_" + dtype.upper()), 8)
        got, lse = run(gpu, b, 0, q, dtype, 8)
        assert need >= 0 and np.array_equal(got, want) and np.array_equal(lse, wl)
    finally:
        E.extend_registers(0)
    again, _ = run(gpu, b, 0, q, dtype, 8)
    assert np.array_equal(again, here) and not np.array_equal(again, got)
    b.free()
