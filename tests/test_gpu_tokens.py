"""GPU: the new tokens of a batch of caches (rotary positions, quantization),
positions copied, gathered and compacted, and positions read back."""
import numpy as np
import pytest

import eakv_b200 as E
from gpu_util import assert_blocks_equal, bits, device_blocks, kv_data

pytestmark = pytest.mark.gpu

DT = {"f32": "float32", "f16": "float16", "bf16": "bfloat16"}
HALF_STEP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}


def make(rng, L, H, hd, size, n):
    c = E.Cache(L, H, hd, size)
    if n:
        assert c.load_raw(kv_data(rng, L, H, n, hd), n) == 0
    return c


def rotate64(x, cos, sin, interleaved):
    """f64 rotation of [tokens, heads, hd] by tables [tokens, pairs]."""
    x = x.astype(np.float64).copy()
    n = cos.shape[1]
    a, b = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if interleaved else (slice(0, n), slice(n, 2 * n))
    c, s = cos.astype(np.float64)[:, None], sin.astype(np.float64)[:, None]
    p, q = x[..., a].copy(), x[..., b].copy()
    x[..., a], x[..., b] = p * c - q * s, q * c + p * s
    return x


APPEND = [
    # hd, nq, nkv, counts, dtype, rot, sections, interleaved, strided
    (128, 8, 2, [1], "bf16", 128, [64], False, False),
    (128, 32, 8, [1, 1, 1], "bf16", 128, [64], False, True),
    (64, 32, 4, [5, 0, 70], "f16", 64, [32], True, True),
    (64, 7, 1, [3], "f32", 32, [10, 3, 3], False, True),
    (128, 5, 5, [63, 2], "f32", 64, [20, 7, 5], True, False),
    (128, 4, 4, [129], "bf16", 104, [26, 13, 0, 13], False, True),
    (128, 6, 3, [17], "f16", 8, [4], False, False),
    (64, 3, 3, [2, 66], "bf16", 0, [], False, True),      # no rotation
]


@pytest.mark.parametrize("hd,nq,nkv,counts,dtype,rot,sections,inter,strided", APPEND)
def test_append_rotary(gpu, hd, nq, nkv, counts, dtype, rot, sections, inter, strided):
    """The pages equal eakv_cache_append's on the rotated rows (rounded once to
    f32) bit for bit; q is the rotation within the type's rounding: half a
    step of the result and, for the f32 arithmetic behind it, two roundings
    of |x c| + |y s| <= 2 |largest|."""
    import torch
    rng = np.random.default_rng(sum(counts) + hd + rot)
    B, L, layer, size = len(counts), 2, 1, 200
    old = [0, 61, 64, 7][:B]
    total = sum(counts)
    tdt = getattr(torch, DT[dtype])
    wide = rng.standard_normal((total, nq + 2 * nkv, hd)).astype(np.float32)
    x = torch.from_numpy(wide).to(gpu).to(tdt)
    if not strided:
        q, k, v = (x[:, a:b].contiguous() for a, b in ((0, nq), (nq, nq + nkv), (nq + nkv, nq + 2 * nkv)))
    else:
        q, k, v = x[:, :nq], x[:, nq:nq + nkv], x[:, nq + nkv:]
    xs = x.float().cpu().numpy()
    kw, cosr, sinr = {}, None, None
    if rot:
        rows, pairs = 300, rot // 2
        ang = rng.uniform(0, 300, (rows, pairs))
        cos, sin = np.cos(ang).astype(np.float32), np.sin(ang).astype(np.float32)
        pos = rng.integers(0, rows, (len(sections), total)).astype(np.int32)
        axis = np.repeat(np.arange(len(sections)), sections)
        at = pos[axis].T
        cosr, sinr = cos[at, np.arange(pairs)], sin[at, np.arange(pairs)]
        kw = dict(cos=torch.from_numpy(cos).to(gpu), sin=torch.from_numpy(sin).to(gpu),
                  positions=torch.from_numpy(pos).to(gpu), sections=sections, interleaved=inter)
    caches = [make(np.random.default_rng(b), L, nkv, hd, size, old[b]) for b in range(B)]
    qo = torch.full((total, nq, hd), float("nan"), dtype=tdt, device=gpu)
    torch.cuda.synchronize()
    E.append_rotary(caches, layer, counts, k, v, q=q, q_out=qo, **kw)
    caches[0].synchronize()
    torch.cuda.synchronize()
    want_q, want_k = xs[:, :nq].astype(np.float64), xs[:, nq:nq + nkv].astype(np.float64)
    if rot:
        want_q, want_k = rotate64(want_q, cosr, sinr, inter), rotate64(want_k, cosr, sinr, inter)
    got = qo.double().cpu().numpy()
    lim = HALF_STEP[dtype] * np.abs(want_q) + 3 * 2.0 ** -24 * 2 * np.abs(xs).max()
    if not rot:
        lim = 0.0 * lim
    assert (np.abs(got - want_q) <= lim).all()
    first = 0
    for b in range(B):
        n = counts[b]
        assert caches[b].seq_len == old[b]
        ref = make(np.random.default_rng(b), L, nkv, hd, size, old[b])
        if n:
            sl = slice(first, first + n)
            ref.append(want_k[sl].astype(np.float32).transpose(1, 0, 2), layer, 0, n)
            ref.append(xs[sl, nq + nkv:].transpose(1, 0, 2), layer, 1, n)
            ref.advance(n)
            caches[b].advance(n)
        assert_blocks_equal(device_blocks(caches[b]), device_blocks(ref))
        # the V-scale bound was raised: a decode over the new positions agrees
        if caches[b].seq_len:
            qq = rng.standard_normal(nq * hd).astype(np.float32)
            assert np.array_equal(bits(caches[b].fused(qq, layer, nq, nkv)), bits(ref.fused(qq, layer, nq, nkv)))
        first += n
        ref.free()
        caches[b].free()
    assert E.device_status(0) == 0


def test_append_in_place_q_and_special_values(gpu):
    """q rotated in place; rows of zeros of both signs, constants, NaN and inf
    quantize as eakv_cache_append does."""
    import torch
    rng = np.random.default_rng(3)
    n, H, hd = 6, 2, 128
    k = rng.standard_normal((n, H, hd)).astype(np.float32)
    k[0] = 0.0
    k[1] = -0.0
    k[2, 0, :64] = 3.25
    k[3, 0, 5] = np.nan
    k[3, 1, 64] = np.nan
    k[4, 0, 70] = np.inf
    k[5, 1, ::2] = -0.0
    v = k[::-1].copy()
    c, ref = E.Cache(1, H, hd, 64), E.Cache(1, H, hd, 64)
    dk, dv = (torch.from_numpy(a).to(gpu) for a in (k, v))
    q = torch.from_numpy(rng.standard_normal((n, 4, hd)).astype(np.float32)).to(gpu)
    one, zero = torch.ones(8, 64, device=gpu), torch.zeros(8, 64, device=gpu)
    pos = torch.arange(n, dtype=torch.int32, device=gpu)
    before = q.clone()
    torch.cuda.synchronize()
    # no table: K goes in as it is
    E.append_rotary([c], 0, [n], dk, dv)
    ref.append(k.transpose(1, 0, 2), 0, 0, n)
    ref.append(v.transpose(1, 0, 2), 0, 1, n)
    c.advance(n)
    ref.advance(n)
    assert_blocks_equal(device_blocks(c), device_blocks(ref))
    c.clear()
    # an angle of a quarter turn, q in place: (a, b) -> (-b, a)
    E.append_rotary([c], 0, [n], dk, dv, q=q, cos=zero, sin=one, positions=pos)
    c.synchronize()
    want = torch.cat([-before[..., 64:], before[..., :64]], -1)
    assert torch.equal(q, want)
    c.free()
    ref.free()
    assert E.device_status(0) == 0


def test_append_bad_positions_leave_the_token_out(gpu):
    import torch
    H, hd, n = 2, 64, 5
    c = E.Cache(1, H, hd, 64)
    x = torch.randn(n, H, hd, device=gpu)
    q = torch.randn(n, H, hd, device=gpu)
    qo = torch.full_like(q, 7.0)
    tab = torch.ones(4, 32, device=gpu)
    pos = torch.tensor([0, 4, 2, -1, 3], dtype=torch.int32, device=gpu)
    torch.cuda.synchronize()
    E.append_rotary([c], 0, [n], x, x, q=q, q_out=qo, cos=tab, sin=tab * 0, positions=pos)
    c.synchronize()
    assert E.device_status(0, reset=True) == 2
    for t, p in enumerate(pos.tolist()):
        if 0 <= p < 4:
            assert torch.equal(qo[t], q[t])
        else:
            assert (qo[t] == 7.0).all()
    c.advance(n)
    got = c.dequantize(0, 0, 0, n)
    assert (got[:, [1, 3]] == 0).all() and (got[:, [0, 2, 4]] != 0).any(-1).all()
    c.free()


def test_append_refusals(gpu):
    import torch
    c, d = E.Cache(2, 2, 128, 8), E.Cache(2, 2, 128, 16)
    x = torch.zeros(4, 2, 128, device=gpu)
    tab = torch.zeros(4, 64, device=gpu)
    pos = torch.zeros(1, 4, dtype=torch.int32, device=gpu)
    ok = dict(cos=tab, sin=tab, positions=pos)

    def no(*args, **kw):
        with pytest.raises((E.EakvError, ValueError)):
            E.append_rotary(*args, **kw)

    no([c], 0, [9], torch.zeros(9, 2, 128, device=gpu), torch.zeros(9, 2, 128, device=gpu))
    no([c], 2, [4], x, x)
    no([c], -1, [4], x, x)
    no([c, c], 0, [2, 2], x, x)                      # the same cache twice
    no([c, d], 0, [2, 2], x, x)                      # another shape
    no([c], 0, [4], x, x.half())
    no([c], 0, [4], x, x, q=torch.zeros(4, 3, 128, device=gpu))   # 3 heads over 2
    no([c], 0, [4], x, x, cos=tab[:, :62].contiguous(), sin=tab[:, :62].contiguous(), positions=pos)
    no([c], 0, [4], x, x, **ok, sections=[63])
    no([c], 0, [4], x, x, **ok, sections=[-1])
    no([c], 0, [4], x, x, cos=torch.zeros(4, 68, device=gpu), sin=torch.zeros(4, 68, device=gpu), positions=pos)
    wide = E.Cache(1, 1, 256, 8)
    no([wide], 0, [1], torch.zeros(1, 1, 256, device=gpu), torch.zeros(1, 1, 256, device=gpu))
    assert c.seq_len == 0
    E.append_rotary([c], 0, [0], x[:0], x[:0])       # nothing to do
    for z in (c, d, wide):
        z.free()
    assert E.device_status(0) == 0


# ---- read back -----------------------------------------------------------------


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("hd,H,begins,counts", [
    (128, 3, [0], [1]), (64, 3, [5, 0, 64], [70, 0, 1]), (128, 8, [63, 1], [2, 128]), (64, 1, [0, 3], [3, 97])])
def test_read_positions(gpu, dtype, hd, H, begins, counts):
    """Rows equal eakv_cache_dequantize's, rounded once to the type."""
    import torch
    rng = np.random.default_rng(hd + H)
    L, S = 3, 150
    caches = [make(rng, L, H, hd, 160, S) for _ in counts]
    total = sum(counts)
    tdt = getattr(torch, DT[dtype])
    # strided and odd-addressed destinations beside the plain one
    plain = torch.full((2, 2, total, H, hd), -5.0, dtype=tdt, device=gpu)
    room = torch.full((2, 2, total, H, hd + 3), -5.0, dtype=tdt, device=gpu)
    odd = room[..., 1:hd + 1]
    torch.cuda.synchronize()
    for out in (plain, odd):
        E.read_positions(caches, begins, counts, out, layer=1)
        caches[0].synchronize()
        first = 0
        for c, b, n in zip(caches, begins, counts):
            for l in range(2):
                for kv in range(2):
                    want = torch.from_numpy(c.dequantize(l + 1, kv, b, b + n)).to(gpu).to(tdt)
                    assert torch.equal(out[l, kv, first:first + n], want.transpose(0, 1))
            first += n
    assert (room[..., 0] == -5.0).all() and (room[..., hd + 1:] == -5.0).all()
    for bad in (dict(layer=2), dict(layer=-1)):
        with pytest.raises(E.EakvError):
            E.read_positions(caches, begins, counts, plain, **bad)
    with pytest.raises(E.EakvError):
        E.read_positions(caches, [160 for _ in counts], [max(n, 1) for n in counts],
                         torch.zeros(1, 2, sum(max(n, 1) for n in counts), H, hd, device=gpu))
    for c in caches:
        c.free()
    assert E.device_status(0) == 0


# ---- copies ----------------------------------------------------------------------


def values(c, kv_layer, upto):
    l, kv = kv_layer
    return c.dequantize(l, kv, 0, upto)


@pytest.mark.parametrize("hd,H", [(64, 3), (128, 2), (256, 2)])
@pytest.mark.parametrize("src_pos,dst_pos,n", [(0, 0, 1), (0, 0, 300), (64, 0, 64), (3, 70, 130), (299, 1, 1), (10, 5, 0),
                                               (0, 70, 256), (0, 70, 257)])
def test_copy(gpu, hd, H, src_pos, dst_pos, n):
    """Bits move unchanged to every destination, whatever its size; what is
    around them stays; the V-scale bound follows."""
    rng = np.random.default_rng(hd + n)
    L = 2
    src = make(rng, L, H, hd, 300, 300)
    dsts = [make(rng, L, H, hd, size, 80) for size in (330, 517)]
    whole = [[values(src, (l, kv), 300) for kv in (0, 1)] for l in range(L)]
    before = [[[values(d, (l, kv), 80) for kv in (0, 1)] for l in range(L)] for d in dsts]
    src.synchronize()
    E.copy_positions(dsts, dst_pos, src, src_pos, n)
    src.synchronize()
    for i, d in enumerate(dsts):
        assert d.seq_len == dst_pos + n
        for l in range(L):
            for kv in (0, 1):
                got = values(d, (l, kv), dst_pos + n)
                assert np.array_equal(bits(got[:, dst_pos:]), bits(whole[l][kv][:, src_pos:src_pos + n]))
                assert np.array_equal(bits(got[:, :dst_pos]), bits(before[i][l][kv][:, :dst_pos]))
                d.advance(1)     # the position behind stays as it was
                if dst_pos + n < 80:
                    assert np.array_equal(bits(d.dequantize(l, kv, dst_pos + n, dst_pos + n + 1)),
                                          bits(before[i][l][kv][:, dst_pos + n:dst_pos + n + 1]))
                d.restore(dst_pos + n)
    for c in [src] + dsts:
        c.free()


def test_copy_raises_the_scale_bound(gpu):
    """A copied V of 1e30 decodes (the bound of the V scales came along)."""
    rng = np.random.default_rng(0)
    data = kv_data(rng, 1, 2, 100, 128)
    data[:, 1] *= np.float32(1e30)
    src, dst = E.Cache(1, 2, 128, 100), E.Cache(1, 2, 128, 200)
    assert src.load_raw(data, 100) == 0
    E.copy_positions([dst], 0, src, 0, 100)
    src.synchronize()
    q = rng.standard_normal(4 * 128).astype(np.float32)
    a, b = src.fused(q, 0, 4, 2), dst.fused(q, 0, 4, 2)
    assert np.array_equal(bits(a), bits(b)) and np.isfinite(a).all()
    with src.fork(60, 64) as f:
        assert f.seq_len == 60 and f.max_seq_len == 64
        src.restore(60)
        assert np.array_equal(bits(f.fused(q, 0, 4, 2)), bits(src.fused(q, 0, 4, 2)))
    src.free()
    dst.free()


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("shared", ["none", "layers", "all"])
@pytest.mark.parametrize("S,n", [(1, 1), (65, 40), (700, 257), (700, 600)])
def test_gather_and_compact(gpu, hd, shared, S, n):
    import torch
    rng = np.random.default_rng(S + n)
    L, H, begin = 2, 3, min(7, S - 1)
    n = min(n, S - begin)
    src = make(rng, L, H, hd, S, S)
    whole = [[values(src, (l, kv), S) for kv in (0, 1)] for l in range(L)]
    shape = {"none": (L, H), "layers": (1, H), "all": (1, 1)}[shared]
    keep = np.stack([np.stack([np.sort(rng.choice(np.arange(begin, S), n, replace=False)) for _ in range(shape[1])])
                     for _ in range(shape[0])]).astype(np.int32)
    idx = torch.from_numpy(keep).to(gpu)
    if shared == "all":
        idx = idx[0, 0]
    full = np.broadcast_to(keep, (L, H, n))
    # any order, with repeats, into another cache
    free = torch.from_numpy(rng.integers(0, S, (L, H, n)).astype(np.int32)).to(gpu)
    dst = make(rng, L, H, hd, S + 70, 3)
    head = [[values(dst, (l, kv), 3) for kv in (0, 1)] for l in range(L)]
    torch.cuda.synchronize()
    dst.synchronize()
    E.gather_positions(dst, 3, src, free)
    src.synchronize()
    assert dst.seq_len == 3 + n
    for l in range(L):
        for kv in (0, 1):
            got = values(dst, (l, kv), 3 + n)
            assert np.array_equal(bits(got[:, :3]), bits(head[l][kv]))
            for h in range(H):
                assert np.array_equal(bits(got[h, 3:]), bits(whole[l][kv][h][free[l, h].cpu().numpy()]))
    # ascending, in place
    src.compact(begin, idx)
    assert src.seq_len == begin + n
    for l in range(L):
        for kv in (0, 1):
            got = values(src, (l, kv), begin + n)
            assert np.array_equal(bits(got[:, :begin]), bits(whole[l][kv][:, :begin]))
            for h in range(H):
                assert np.array_equal(bits(got[h, begin:]), bits(whole[l][kv][h][full[l, h]]))
    assert E.device_status(0) == 0
    src.free()
    dst.free()


def test_bad_indexes_are_reported_and_left(gpu):
    import torch
    rng = np.random.default_rng(9)
    src, dst = make(rng, 1, 2, 128, 100, 90), make(rng, 1, 2, 128, 100, 20)
    s0, d0 = values(src, (0, 1), 90), values(dst, (0, 1), 20)
    idx = torch.tensor([5, -1, 90, 7, 2 ** 31 - 1], dtype=torch.int32, device=gpu)
    torch.cuda.synchronize()
    dst.synchronize()
    E.gather_positions(dst, 10, src, idx)
    src.synchronize()
    assert E.device_status(0, reset=True) == 2
    got = values(dst, (0, 1), 15)
    assert np.array_equal(bits(got[:, [10, 13]]), bits(s0[:, [5, 7]]))
    assert np.array_equal(bits(got[:, [11, 12, 14]]), bits(d0[:, [11, 12, 14]]))
    # in place an entry below its own place is refused as well
    idx = torch.tensor([12, 3, 13, 100], dtype=torch.int32, device=gpu)
    torch.cuda.synchronize()
    src.compact(10, idx)
    src.synchronize()
    assert E.device_status(0, reset=True) == 2
    got = values(src, (0, 1), 14)
    assert np.array_equal(bits(got[:, 10:]), bits(s0[:, [12, 11, 13, 13]]))
    src.free()
    dst.free()


def test_move_refusals(gpu):
    import torch
    rng = np.random.default_rng(1)
    src, dst, other = make(rng, 1, 2, 128, 100, 50), make(rng, 1, 2, 128, 100, 10), make(rng, 1, 1, 128, 100, 10)
    idx = torch.zeros(4, dtype=torch.int32, device=gpu)

    def no(f, *args):
        with pytest.raises((E.EakvError, ValueError)):
            f(*args)

    no(E.copy_positions, [dst], 0, src, 0, 51)
    no(E.copy_positions, [dst], 11, src, 0, 5)
    no(E.copy_positions, [dst], 0, src, -1, 5)
    no(E.copy_positions, [dst], 0, src, 0, -1)
    no(E.copy_positions, [src], 0, src, 0, 5)
    no(E.copy_positions, [dst, dst], 0, src, 0, 5)
    no(E.copy_positions, [other], 0, src, 0, 5)
    no(E.gather_positions, src, 0, src, idx)
    no(E.gather_positions, dst, 98, src, idx)
    no(E.gather_positions, other, 0, src, idx)
    no(src.compact, 51, idx)
    no(src.compact, -1, idx)
    no(src.fork, 51)
    no(src.fork, 5, 4)
    assert (src.seq_len, dst.seq_len, other.seq_len) == (50, 10, 10)
    for c in (src, dst, other):
        c.free()
    assert E.device_status(0) == 0
