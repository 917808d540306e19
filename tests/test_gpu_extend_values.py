"""GPU: eakv_extend_attention over values that stress the powers of two its operands are
held by: unwritten and denormal positions, V near the smallest numbers, groups and rows
of very different sizes, q elements far below their row's largest."""
import numpy as np
import pytest

import eakv_b200 as E
from gpu_util import kv_data
from test_gpu_extend import CODE, HALF_STEP, rounded, run

pytestmark = pytest.mark.gpu

KINDS = [("f32", "auto"), ("f16", "mma"), ("bf16", "mma"), ("f16", "umma"), ("bf16", "umma")]


@pytest.fixture(autouse=True)
def _path(request):
    E.force_splits(0)
    E.force_path(CODE[request.node.callspec.params.get("path", "auto")])
    yield
    E.force_splits(0)
    E.force_path(0)


class Sequence:
    """One cache whose positions are segments in a row, each an array [2, H, n, hd] or a
    number of positions that are advanced over and never written. The last `new` positions are the
    call's new tokens."""

    def __init__(self, H, hd, segments, new):
        n = sum(s if isinstance(s, int) else s.shape[2] for s in segments)
        self.H, self.hd, self.old, self.new = H, hd, [n - new], [new]
        c = E.Cache(1, H, hd, n)
        for s in segments:
            if not isinstance(s, int):
                for kv in (0, 1):
                    assert c.append(np.ascontiguousarray(s[kv]), 0, kv, s.shape[2]) == 0
            assert c.advance(s if isinstance(s, int) else s.shape[2]) == 0
        self.k, self.v = ([[c.dequantize(0, kv, 0, n).astype(np.float64)]] for kv in (0, 1))
        assert c.restore(n - new) == 0
        self.caches = [c]

    def free(self):
        self.caches[0].free()


def data(rng, H, n, hd, k=1.0, v=1.0):
    d = kv_data(rng, 1, H, n, hd)[0]
    d[0] *= np.float32(k)
    d[1] *= np.float32(v)
    return d


def exact(seq, q, scale, window=0):
    """64-bit attention of one sequence -> out [n, nq, hd], lse, and per row: sum_j p_j max|v_j| of
    every 64-dim group [n, nq, groups], the largest sum |q k| scale over attended positions."""
    old, n, hd = seq.old[0], seq.new[0], seq.hd
    nq = q.shape[1]
    i, j = np.arange(n)[:, None], np.arange(old + n)[None, :]
    ok = j <= old + i
    if window:
        ok = ok & (j > old + i - window)
    out, lse = np.zeros((n, nq, hd)), np.zeros((n, nq))
    size, reach = np.zeros((n, nq, hd // 64)), np.zeros((n, nq))
    for h in range(nq):
        k, v = seq.k[0][0][h * seq.H // nq], seq.v[0][0][h * seq.H // nq]
        s = np.where(ok, q[:, h].astype(np.float64) @ k.T * scale, -np.inf)
        m = s.max(1, keepdims=True)
        p = np.exp(s - m)
        total = p.sum(1, keepdims=True)
        out[:, h], lse[:, h] = p / total @ v, (m + np.log(total))[:, 0]
        size[:, h] = p / total @ np.abs(v).reshape(len(v), -1, 64).max(2)
        reach[:, h] = np.where(ok, np.abs(q[:, h]).astype(np.float64) @ np.abs(k).T, 0).max(1) * scale
    return out, lse, size, reach


def meets(gpu, seq, q, dtype, path, window=0):
    """The outputs within what the roundings allow, group by group.
    A score is off by at most d: sums of 128 exact products in f32 2^-16 of the row's sum |q k|; where
    K is held in f16 (tcgen05) two roundings of at most the group's size, 2^-11 each. A weight is
    then off by a factor within e^(2 d), and rounded to 22 bits (f32) or 11; V in f16 is rounded twice, at
    most the group's size each. Then half a step of the output's type; one of its smallest
    denormal number counts for results below the normal range."""
    q = rounded(q, dtype)
    got, lse = run(gpu, seq, 0, q, dtype, q.shape[1], window=window)
    want, wl, size, reach = exact(seq, q, seq.hd ** -0.5, window)
    wide = path == "umma"
    d = reach * (2.0 ** -16 + (2 * 2.0 ** -11 if wide else 0.0))
    w = (2.0 ** -22 if dtype == "f32" else 2.0 ** -11) + (2 * 2.0 ** -11 if wide else 0.0) + 2.0 ** -15
    lim = (2 * d[..., None] + w) * size
    lim = np.repeat(lim, 64, axis=2) + HALF_STEP[dtype] * np.abs(want)
    lim += {"f32": 2.0 ** -140, "bf16": 2.0 ** -133, "f16": 2.0 ** -25}[dtype]
    err = np.abs(got - want)
    assert (err <= lim).all(), f"worst {np.nanmax(err / lim)} of the limit, nan {np.isnan(got).sum()}"
    assert (np.abs(lse - wl) <= d + 2.0 ** -16 + 2.0 ** -22 * np.abs(wl)).all()
    assert E.device_status(0) == 0


def layouts(rng, H, hd):
    """Positions never written, or of denormal size, before, between and behind others."""
    real = lambda n: data(rng, H, n, hd, v=0.3)           # noqa: E731
    tiny = data(rng, H, 256, hd, v=1e-41)
    return {"before": [256, real(256)], "between": [real(100), 200, real(60)],
            "behind": [real(300), 128, real(3)], "alone": [256], "ragged": [70, real(1), 70, real(1), 59],
            "denormal before": [tiny, real(256)], "denormal behind": [real(200), tiny, real(5)]}


@pytest.mark.parametrize("dtype,path", KINDS)
@pytest.mark.parametrize("kind", ["before", "between", "behind", "alone", "ragged", "denormal before",
                                  "denormal behind"])
@pytest.mark.parametrize("hd,new", [(128, 3), (64, 50)])
def test_positions_without_a_scale(gpu, hd, new, kind, dtype, path):
    """Zero and denormal V scales leave every weight its share."""
    rng = np.random.default_rng(len(kind) + hd)
    seq = Sequence(2, hd, layouts(rng, 2, hd)[kind], min(new, 3) if kind == "behind" else new)
    q = rng.standard_normal((seq.new[0], 4, hd)).astype(np.float32)
    meets(gpu, seq, q, dtype, path)
    seq.free()


@pytest.mark.parametrize("dtype,path", [k for k in KINDS if k[0] != "f16"])   # f16 holds no such output
@pytest.mark.parametrize("first,rest", [(1e-35, 1e-35), (1e-37, 1e-37), (1e-37, 1.0), (1.0, 1e-36), (1e-30, 1e30)])
def test_the_smallest_values(gpu, first, rest, dtype, path):
    """V down to the last normal numbers, over a long row, and a small start that larger values follow."""
    rng = np.random.default_rng(3)
    H, hd = 2, 128
    seq = Sequence(H, hd, [data(rng, H, 64, hd, v=first), data(rng, H, 4000, hd, v=rest)], 4)
    meets(gpu, seq, rng.standard_normal((4, 4, hd)).astype(np.float32), dtype, path)
    seq.free()


@pytest.mark.parametrize("dtype,path", KINDS)
@pytest.mark.parametrize("k", [8, 10, 12, 14, 16])
@pytest.mark.parametrize("low", [0, 1])
@pytest.mark.parametrize("window", [1, 0])
def test_groups_of_different_size(gpu, window, low, k, dtype, path):
    """One 64-dim group of V is 2^-k of the other: its dims keep their own precision. A window of one
    makes each output a single position's value."""
    rng = np.random.default_rng(k)
    H, hd, new = 1, 128, 40
    d = data(rng, H, 170, hd)
    d[1, :, :, 64 * low:64 * low + 64] *= np.float32(2.0 ** -k)
    if dtype == "f16":   # into its normal range: 2^-14 .. 2^16
        d[1] *= np.float32(2.0 ** (k - 4))
    seq = Sequence(H, hd, [d], new)
    q = (0.05 * rng.standard_normal((new, 4, hd))).astype(np.float32)
    meets(gpu, seq, q, dtype, path, window)
    seq.free()


@pytest.mark.parametrize("dtype,path", KINDS)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("k", [5, 9, 11, 14])
def test_rows_below_the_first(gpu, hd, k, dtype, path):
    """V rows 2^-k of those of the part's first positions, each seen alone."""
    rng = np.random.default_rng(k)
    new = 70
    seq = Sequence(1, hd, [data(rng, 1, 128, hd, v=2.0 ** (k - 8)), data(rng, 1, 150, hd, v=2.0 ** -8)], new)
    E.force_splits(1)
    q = (0.05 * rng.standard_normal((new, 2, hd))).astype(np.float32)
    meets(gpu, seq, q, dtype, path, window=1)
    meets(gpu, seq, q, dtype, path, window=60)
    seq.free()


@pytest.mark.parametrize("dtype,path", [k for k in KINDS if k[0] != "f16"])
@pytest.mark.parametrize("k", [8, 12, 16])
def test_key_groups_of_different_size(gpu, k, dtype, path):
    """One group of K is 2^-k of the other, and q's dims there 2^k of the others: both groups take
    the same part in the scores."""
    rng = np.random.default_rng(k)
    H, hd, new = 1, 128, 40
    d = data(rng, H, 170, hd)
    d[0, :, :, 64:] *= np.float32(2.0 ** -k)
    seq = Sequence(H, hd, [d], new)
    q = rng.standard_normal((new, 4, hd)).astype(np.float32) * 0.2
    q[..., 64:] *= np.float32(2.0 ** k)
    meets(gpu, seq, q, dtype, path)
    seq.free()


@pytest.mark.parametrize("dtype,path", KINDS)
def test_small_elements_of_q(gpu, dtype, path):
    """Elements of q down to 2^-16 of their row's largest keep their bits: they meet keys as much larger."""
    rng = np.random.default_rng(16)
    H, hd, new = 1, 128, 40
    d = data(rng, H, 170, hd, k=2.0 ** -6)
    d[0, :, :, 64:] *= np.float32(2.0 ** 16)
    seq = Sequence(H, hd, [d], new)
    q = rng.standard_normal((new, 4, hd)).astype(np.float32) * 2.0 ** 5
    q[..., 64:] *= np.float32(2.0 ** -16)
    meets(gpu, seq, q, dtype, path)
    seq.free()


@pytest.mark.parametrize("dtype,path", KINDS)
@pytest.mark.parametrize("splits", [0, 4])
def test_the_same_call_gives_the_same_bits(gpu, splits, dtype, path):
    rng = np.random.default_rng(7)
    seq = Sequence(2, 128, [data(rng, 2, 3000, 128)], 60)
    q = rng.standard_normal((60, 8, 128)).astype(np.float32)
    E.force_splits(splits)
    first, lse = run(gpu, seq, 0, q, dtype, 8)
    for _ in range(20):
        out, l = run(gpu, seq, 0, q, dtype, 8)
        assert np.array_equal(out, first) and np.array_equal(l, lse)
    seq.free()


@pytest.mark.parametrize("dtype,path", KINDS)
@pytest.mark.parametrize("hd,new", [(128, 3), (64, 50)])
@pytest.mark.parametrize("level", [0.0, 3e-4])
def test_groups_of_one_value(gpu, level, hd, new, dtype, path):
    """A group of 64 equal values has a scale of 1 whatever they are: zero vectors, or 3e-4 in all dims,
    among values of 1e-3 do not bring errors of that scale."""
    rng = np.random.default_rng(hd)
    d = data(rng, 2, 300, hd, k=0.1, v=1e-3)
    d[1, :, ::2] = level
    d[1, 1, 1::4, :64] = -level
    d[0, :, 5::7] = level
    d[:, :, 128:192] = level     # a whole page
    seq = Sequence(2, hd, [d], new)
    q = rng.standard_normal((new, 4, hd)).astype(np.float32)
    meets(gpu, seq, q, dtype, path)
    meets(gpu, seq, q, dtype, path, window=3)
    seq.free()


@pytest.mark.parametrize("dtype,path", [k for k in KINDS if k[0] != "f16"])
@pytest.mark.parametrize("size", [1e-12, 1e-3, 1e12])
@pytest.mark.parametrize("kind", ["unwritten", "zeros", "one in three", "scattered", "large ones before"])
@pytest.mark.parametrize("hd,new", [(128, 3), (64, 50), (128, 150)])
def test_rows_of_zeros_among_values_of_any_size(gpu, hd, new, kind, size, dtype, path):
    """V rows of zeros, never written or written, in a part's first tile, in runs of 32 and among others,
    leave values of any size their weights; so do large values before a row's window."""
    rng = np.random.default_rng(hd + len(kind))
    d = data(rng, 2, 300 + new, hd, v=size)
    window = 0
    segments = [d]
    if kind == "unwritten":
        segments = [256, d]
    elif kind == "zeros":
        d[1, :, 32:200] = 0
    elif kind == "one in three":
        d[1, :, ::3] = 0
    elif kind == "scattered":
        d[1, :, rng.integers(0, 300, 5)] = 0
    else:
        window = 40
        d[1, :, :300 + new // 2] *= np.float32(1e15)
        d[1, :, 260 + new // 2:300 + new // 2] = 0
    seq = Sequence(2, hd, segments, new)
    q = rng.standard_normal((new, 4, hd)).astype(np.float32)
    meets(gpu, seq, q, dtype, path, window)
    seq.free()
