"""Cases of the cache's multi-token operators, and their plain forms.

append   new tokens of a batch of caches: rotate q and k by their positions, quantise k and v into the pages
extend   attention of several new tokens per cache over the Q4 cache
copy     a range of one cache copied to others (fork), listed positions gathered into another (eviction)
read     ranges of several caches and layers read back as values

The plain forms are elementary torch operations on the same quantised cache, held as (nibbles, scale, bias)
tensors; quantised state is returned as the values it stands for.
"""
import math
import random

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}


def listed():
    return [
        # a short draft on a small model (22-layer shape of the benchmark, 4 KV heads of 64): the smallest call
        dict(name="extend_draft_small", op="extend", B=1, T=2, S=2048, nq=32, nkv=4, hd=64, dtype="bf16", window=0,
             tree=False, ragged=False),
        # drafted tokens of a batch of long sequences being verified: 16 sequences of 32768, five tokens each
        dict(name="extend_draft_batch", op="extend", B=16, T=5, S=32768, nq=32, nkv=8, hd=128, dtype="bf16", window=0,
             tree=False, ragged=True),
        # one chunk of a long prompt: 2048 new tokens behind 32768 cached ones (the largest)
        dict(name="extend_chunk_long", op="extend", B=1, T=2048, S=34816, nq=32, nkv=8, hd=128, dtype="bf16", window=0,
             tree=False, ragged=False),
        # a batch of whole prompts without earlier context, every query head its own KV head, odd lengths
        dict(name="extend_prompts", op="extend", B=4, T=1501, S=1501, nq=32, nkv=32, hd=128, dtype="bf16", window=0,
             tree=False, ragged=True),
        # a drafted tree of tokens with a sliding window, queries and outputs in 32 bits
        dict(name="extend_tree_f32", op="extend", B=4, T=13, S=5003, nq=64, nkv=8, hd=128, dtype="f32", window=4096,
             tree=True, ragged=True),
        # the next token of 16 sequences: latency
        dict(name="append_step", op="append", B=16, T=1, S=4096, nq=32, nkv=8, hd=128, dtype="bf16", axes=1, rot=128,
             interleaved=False, ragged=True),
        # a prompt of images or video (time, height, width), the halves rotated
        dict(name="append_video", op="append", B=1, T=2048, S=8192, nq=32, nkv=8, hd=128, dtype="bf16", axes=3, rot=128,
             interleaved=False, ragged=False),
        # a ragged batch of f32 prompts, interleaved pairs, half of each head rotated
        dict(name="append_prompts_f32", op="append", B=3, T=777, S=2048, nq=32, nkv=4, hd=64, dtype="f32", axes=1, rot=32,
             interleaved=True, ragged=True),
        # a prompt forked to two samples
        dict(name="copy_fork", op="copy", L=2, n=2048, S=2048, nkv=8, hd=128, children=2, shift=0, gather=False),
        # eviction: each head of each layer keeps its own 4096 of 16384 positions
        dict(name="copy_evict", op="copy", L=2, n=4096, S=16384, nkv=8, hd=128, children=1, shift=0, gather=True),
        # the newest positions of a batch, all layers, for a check or a hand-over
        dict(name="read_recent", op="read", B=16, L=4, n=33, S=1000, nkv=4, hd=64, dtype="bf16"),
        # a whole sequence read back
        dict(name="read_whole", op="read", B=1, L=4, n=8192, S=8192, nkv=8, hd=128, dtype="f32"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("extend", "extend", "append", "copy", "read"))
    hd = rng.choice((64, 128))
    nkv, g = rng.choice(((4, 8), (8, 4), (8, 8), (8, 1), (2, 7), (4, 3)))
    if op == "extend":
        T = _log(rng, 1, 1600)
        dtype = rng.choice(("bf16", "bf16", "f32")) if T <= 256 else "bf16"
        B = _log(rng, 1, 16 if T <= 64 else 3)
        S = T + (_log(rng, 1, 24000 if T <= 64 else 8000) if rng.random() < 0.8 else 0)
        return dict(op=op, B=B, T=T, S=S, nq=nkv * g, nkv=nkv, hd=hd, dtype=dtype,
                    window=_log(rng, 16, 8192) if rng.random() < 0.3 else 0, tree=T <= 64 and rng.random() < 0.4,
                    ragged=rng.random() < 0.7)
    if op == "append":
        T = _log(rng, 1, 1500)
        B = _log(rng, 1, 16 if T <= 64 else 4)
        return dict(op=op, B=B, T=T, S=T + rng.randrange(0, 3000), nq=nkv * g, nkv=nkv, hd=hd,
                    dtype=rng.choice(("f32", "f16", "bf16", "bf16")), axes=rng.choice((1, 1, 2, 3)),
                    rot=rng.choice((hd, hd, hd // 2)), interleaved=rng.random() < 0.4, ragged=rng.random() < 0.7)
    if op == "copy":
        S = _log(rng, 65, 16384)
        n = rng.randrange(1, min(S, 6000) + 1)
        gather = rng.random() < 0.5
        return dict(op=op, L=rng.choice((1, 2, 3)), n=n, S=S, nkv=nkv, hd=hd, children=1 if gather else rng.choice((1, 2, 3)),
                    shift=rng.choice((0, 0, 5, 64)), gather=gather)
    n = _log(rng, 1, 6000)
    return dict(op=op, B=_log(rng, 1, 16 if n < 256 else 3), L=rng.choice((1, 2, 4)), n=n, S=n + rng.randrange(0, 500),
                nkv=nkv, hd=hd, dtype=rng.choice(("f32", "f16", "bf16")))


# ---- shapes of a case ---------------------------------------------------------------


def _lengths(case):
    """(cached positions before the new tokens, new tokens) of each cache: a pure function of the case."""
    r = random.Random(case["B"] * 7919 + case["T"] * 31 + case["S"])
    new = [r.randint(max(1, case["T"] // 2), case["T"]) if case["ragged"] else case["T"] for _ in range(case["B"])]
    new[0] = case["T"]
    before = case["S"] - case["T"]
    old = [r.randint(before * 3 // 4, before) if case["ragged"] else before for _ in range(case["B"])]
    old[0] = before
    return old, new


def _sections(case):
    """Rotated pairs that follow each position axis."""
    pairs, axes = case["rot"] // 2, case["axes"]
    rest = [pairs // (axes + 1)] * (axes - 1)
    return [pairs - sum(rest)] + rest


# ---- the quantised cache as tensors ----------------------------------------------------


def _quantise(x):
    """f32 [..., hd] -> nibbles u8 [..., hd/64, 64], scale and bias [..., hd/64]: the cache's rule, each step rounded once."""
    g = x.unflatten(-1, (-1, 64))
    low, high = g.amin(-1), g.amax(-1)
    span = high - low
    fifteen = torch.full_like(span, 15.0)
    scale = torch.where(span > 0, span / fifteen, 1.0)
    inv = torch.where(span > 0, fifteen / span, 0.0)
    n = ((g - low[..., None]) * inv[..., None] + 0.5).floor_().clamp_(0, 15).to(torch.uint8)
    return n, scale, low


def _pack(n):
    return n[..., :32] | (n[..., 32:] << 4)


def _values(w, scale, bias):
    """f32 values [..., hd] of packed groups."""
    n = torch.cat([w & 15, w >> 4], -1).float()
    return (n * scale[..., None] + bias[..., None]).flatten(-2)


def _values64(w, scale, bias):
    n = torch.stack([w.to(torch.int16) % 16, w.to(torch.int16) // 16], -2).flatten(-2).double()
    return (n * scale.double()[..., None] + bias.double()[..., None]).reshape(*w.shape[:-2], -1)


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _kv(gen, L, H, S, hd):
    """K with channels of different sizes, V standard normal: f32 [L, 2, H, S, hd]."""
    x = torch.randn(L, 2, H, S, hd, generator=gen, device="cuda")
    x[:, 0] *= torch.exp(torch.empty(L, H, 1, hd, device="cuda").uniform_(math.log(0.5), math.log(8.0), generator=gen))
    return x


# ---- inputs ----------------------------------------------------------------------------


def _handle(L, nkv, hd, size, raw=None):
    """The user's cache on torch's current stream, filled with `raw`."""
    import eakv_b200 as E

    c = E.Cache(L, nkv, hd, size)
    c.set_stream(torch.cuda.current_stream().cuda_stream or 1)  # 1: the legacy default stream
    if raw is not None:
        assert c.load_raw_device(raw.contiguous(), raw.shape[3]) == 0
    return c


def prepare(case, seed):
    gen = _gen(seed)
    s = dict(case=case)
    op, nkv, hd = case["op"], case["nkv"], case["hd"]
    if op == "extend":
        old, new = _lengths(case)
        B, T, S = case["B"], case["T"], max(a + b for a, b in zip(old, new))
        s["old"], s["new"] = old, new
        s["w"] = torch.zeros(B, 2, nkv, S, hd // 64, 32, dtype=torch.uint8, device="cuda")
        s["scale"], s["bias"] = (torch.zeros(B, 2, nkv, S, hd // 64, device="cuda") for _ in range(2))
        s["caches"] = []
        for b in range(B):
            n = old[b] + new[b]
            raw = _kv(gen, 1, nkv, n, hd)
            q, s["scale"][b, :, :, :n], s["bias"][b, :, :, :n] = _quantise(raw[0])
            s["w"][b, :, :, :n] = _pack(q)
            if own:
                s["caches"].append(_handle(1, nkv, hd, S, raw))
                s["caches"][-1].restore(old[b])  # the new tokens' K and V are appended, not yet advanced over
        total = sum(new)
        s["q"] = torch.randn(total, case["nq"], hd, generator=gen, device="cuda").to(DTYPES[case["dtype"]])
        s["row"] = torch.tensor([[min(sum(new[:b]) + t, total - 1) for t in range(T)] for b in range(B)], device="cuda")
        s["old_"], s["new_"] = torch.tensor(old, device="cuda"), torch.tensor(new, device="cuda")
        s["back"] = torch.tensor([b * T + t for b in range(B) for t in range(new[b])], device="cuda")
        s["tree"] = None
        if case["tree"]:  # each token's ancestors and itself, as bits
            r, bits = random.Random(seed), []
            for n in new:
                mine = []
                for t in range(n):
                    mine.append((1 << t) | (mine[r.randrange(t)] if t else 0))
                bits += [m - (1 << 64) if m >> 63 else m for m in mine]
            s["tree"] = torch.tensor(bits, dtype=torch.int64, device="cuda")
    elif op == "append":
        old, new = _lengths(case)
        s["old"], s["new"] = old, new
        nq, pairs, total = case["nq"], case["rot"] // 2, sum(new)
        # the projections' output: q, k and v of a token side by side
        s["qkv"] = torch.randn(total, (nq + 2 * nkv) * hd, generator=gen, device="cuda").to(DTYPES[case["dtype"]])
        rows = case["S"] + 64
        angle = torch.arange(rows, device="cuda").double()[:, None] * 10000.0 ** (-torch.arange(pairs, device="cuda").double() / pairs)
        s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
        pos = torch.tensor([old[b] + t for b in range(case["B"]) for t in range(new[b])], dtype=torch.int32, device="cuda")
        if case["axes"] > 1:  # a frame's height and width, behind its time
            side = torch.randint(0, 64, (case["axes"] - 1, total), generator=gen, device="cuda", dtype=torch.int32)
            s["pos"] = torch.cat([pos[None], side])
        else:
            s["pos"] = pos[None]
        s["axis"] = torch.tensor([a for a, n in enumerate(_sections(case)) for _ in range(n)], device="cuda")
        s["sections"] = _sections(case)
        s["caches"] = []
        if own:
            for b in range(case["B"]):
                c = _handle(1, nkv, hd, case["S"])
                if old[b]:
                    assert c.advance(old[b]) == 0
                s["caches"].append(c)
    elif op == "copy":
        L, S, n = case["L"], case["S"], case["n"]
        raw = _kv(gen, L, nkv, S, hd)
        q, s["scale"], s["bias"] = _quantise(raw)
        s["w"] = _pack(q)
        if case["gather"]:
            order = torch.rand(L, nkv, S, generator=gen, device="cuda").argsort(-1)[..., :n]
            s["index"] = order.sort(-1).values.to(torch.int32).contiguous()
        s["src"], s["dst"] = None, []
        if own:
            s["src"] = _handle(L, nkv, hd, S, raw)
            for _ in range(case["children"]):
                s["dst"].append(_handle(L, nkv, hd, n + case["shift"] + 64))
                if case["shift"]:
                    s["dst"][-1].advance(case["shift"])
    else:
        B, L, S = case["B"], case["L"], case["S"]
        raws = [_kv(gen, L, nkv, S, hd) for _ in range(B)]
        parts = [_quantise(r) for r in raws]
        s["w"] = torch.stack([_pack(p[0]) for p in parts])
        s["scale"], s["bias"] = torch.stack([p[1] for p in parts]), torch.stack([p[2] for p in parts])
        r = random.Random(S * 31 + case["n"])
        s["begin"] = [r.randint(0, S - case["n"]) for _ in range(B)]
        s["begin_"] = torch.tensor(s["begin"], device="cuda")
        s["caches"] = [_handle(L, nkv, hd, S, x) for x in raws] if own else []
    return s


# ---- one pass ----------------------------------------------------------------------------


def _allowed(s):
    """bool [B, T, S]: the positions that each new token attends."""
    case = s["case"]
    S, T = s["w"].shape[3], case["T"]
    col = torch.arange(S, device="cuda")[None, None, :]
    t = torch.arange(T, device="cuda")[None, :, None]
    old, new = s["old_"][:, None, None], s["new_"][:, None, None]
    at = old + t
    ok = (col <= at) & (t < new)
    if case["window"]:
        ok &= col > at - case["window"]
    if s["tree"] is not None:
        bits = s["tree"][s["row"]][:, :, None]
        ok &= (col < old) | ((bits >> (col - old).clamp(0, 63)) & 1).bool()
    return ok


def _extend_plain(s):
    case = s["case"]
    B, T, H, hd = case["B"], case["T"], case["nkv"], case["hd"]
    G = case["nq"] // H
    k, v = _values(s["w"], s["scale"], s["bias"]).unbind(1)
    q = s["q"].float()[s["row"]].view(B, T, H, G, hd).permute(0, 2, 1, 3, 4).reshape(B, H, T * G, hd)
    sc = (q @ k.transpose(-1, -2)).view(B, H, T, G, -1) / math.sqrt(hd)
    sc.masked_fill_(~_allowed(s)[:, None, :, None, :], -math.inf)
    m = sc.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, 0.0, m)
    p = (sc - m).exp_()
    total = p.sum(-1, keepdim=True)
    o = (p.view(B, H, T * G, -1) @ v).view(B, H, T, G, hd) / torch.where(total > 0, total, 1.0)
    o = o.permute(0, 2, 1, 3, 4).reshape(B * T, H * G, hd)[s["back"]].to(s["q"].dtype)
    if case["dtype"] != "f32":
        return o
    lse = (m + total.log()).permute(0, 2, 1, 3, 4).reshape(B * T, H * G)[s["back"]]
    return {"out": o, "lse": lse}


def _extend_own(s):
    import eakv_b200 as E

    case = s["case"]
    out = torch.empty_like(s["q"])
    lse = torch.empty(s["q"].shape[:2], device="cuda") if case["dtype"] == "f32" else None
    E.extend_attention(s["caches"], 0, s["new"], s["q"], out, window=case["window"], tree=s["tree"], lse=lse)
    return out if lse is None else {"out": out, "lse": lse}


def _rotate(x, c, s, interleaved):
    """Rotates the leading pairs of [tokens, heads, hd] in 64 bits (products of two 24-bit numbers are exact there)."""
    x = x.double()
    r = 2 * c.shape[-1]
    c, s = c.double()[:, None, :], s.double()[:, None, :]
    a, b = (x[..., 0:r:2], x[..., 1:r:2]) if interleaved else (x[..., : r // 2], x[..., r // 2 : r])
    u, v = a * c - b * s, b * c + a * s
    return torch.cat([torch.stack([u, v], -1).flatten(-2) if interleaved else torch.cat([u, v], -1), x[..., r:]], -1)


def _append_plain(s):
    case = s["case"]
    nq, nkv, hd = case["nq"], case["nkv"], case["hd"]
    x = s["qkv"].view(len(s["qkv"]), nq + 2 * nkv, hd)
    pair = torch.arange(len(s["axis"]), device="cuda")
    at = s["pos"].long()[s["axis"]].t()  # [tokens, pairs]
    c, sn = s["cos"][at, pair], s["sin"][at, pair]
    turned = _rotate(x[:, : nq + nkv], c, sn, case["interleaved"])
    kv = torch.stack([turned[:, nq:].float(), x[:, nq + nkv :].float()])
    n, scale, bias = _quantise(kv)
    return {"q": turned[:, :nq].to(x.dtype), "kv": _values(_pack(n), scale, bias)[None]}


def _append_own(s):
    import eakv_b200 as E

    case = s["case"]
    nq, nkv, hd = case["nq"], case["nkv"], case["hd"]
    total = len(s["qkv"])
    x = s["qkv"].view(total, nq + 2 * nkv, hd)
    q = torch.empty(total, nq, hd, dtype=x.dtype, device="cuda")
    E.append_rotary(s["caches"], 0, s["new"], x[:, nq : nq + nkv], x[:, nq + nkv :], q=x[:, :nq], q_out=q, cos=s["cos"],
                    sin=s["sin"], positions=s["pos"], sections=s["sections"], interleaved=case["interleaved"])
    kv = torch.empty(1, 2, total, nkv, hd, device="cuda")  # what the cache holds now, token-major like the projections
    E.read_positions(s["caches"], s["old"], s["new"], kv)
    return {"q": q, "kv": kv}


def _copy_plain(s):
    case = s["case"]
    n = case["n"]
    if case["gather"]:
        at = s["index"].long()[:, None, :, :, None, None].expand(-1, 2, -1, -1, case["hd"] // 64, 1)
        got = [x.gather(3, at.expand(*at.shape[:-1], x.shape[-1])) for x in (s["w"], s["scale"][..., None], s["bias"][..., None])]
    else:
        got = [x[:, :, :, case["S"] - n :].clone() for x in (s["w"], s["scale"][..., None], s["bias"][..., None])]
    v = _values(got[0], got[1][..., 0], got[2][..., 0]).transpose(2, 3)  # [layers, 2, positions, heads, hd]
    return v.repeat(1, 1, case["children"], 1, 1)


def _copy_own(s):
    import eakv_b200 as E

    case, n = s["case"], s["case"]["n"]
    if case["gather"]:
        E.gather_positions(s["dst"][0], case["shift"], s["src"], s["index"])
    else:
        E.copy_positions(s["dst"], case["shift"], s["src"], case["S"] - n, n)
    out = torch.empty(case["L"], 2, case["children"] * n, case["nkv"], case["hd"], device="cuda")
    E.read_positions(s["dst"], [case["shift"]] * case["children"], [n] * case["children"], out)
    return out


def _read_plain(s):
    case = s["case"]
    at = (s["begin_"][:, None] + torch.arange(case["n"], device="cuda"))[:, None, None, None, :, None]
    at = at.expand(-1, case["L"], 2, case["nkv"], -1, case["hd"] // 64)
    w = s["w"].gather(4, at[..., None].expand(*at.shape, 32))
    v = _values(w, s["scale"].gather(4, at), s["bias"].gather(4, at)).to(DTYPES[case["dtype"]])
    return v.permute(1, 2, 0, 4, 3, 5).reshape(case["L"], 2, -1, case["nkv"], case["hd"])


def _read_own(s):
    import eakv_b200 as E

    case = s["case"]
    out = torch.empty(case["L"], 2, case["B"] * case["n"], case["nkv"], case["hd"], dtype=DTYPES[case["dtype"]], device="cuda")
    E.read_positions(s["caches"], s["begin"], [case["n"]] * case["B"], out)
    return out


def run(s):
    op = s["case"]["op"]
    if op == "extend":
        return _extend_own(s) if own else _extend_plain(s)
    if op == "append":
        return _append_own(s) if own else _append_plain(s)
    if op == "copy":
        return _copy_own(s) if own else _copy_plain(s)
    return _read_own(s) if own else _read_plain(s)


# ---- what a pass cannot do without -----------------------------------------------------


def work(case):
    op, nkv, hd = case["op"], case["nkv"], case["hd"]
    pos = 2 * nkv * (hd // 64) * 40  # bytes of one position's K and V in one layer
    if op == "extend":
        old, new = _lengths(case)
        pairs = read = 0
        for a, b in zip(old, new):
            far = case["window"] or 1 << 60
            first = max(0, a - far + 1)
            read += a + b - first
            pairs += sum(min(a + t + 1, far) for t in range(b))
        io = 2 * sum(new) * case["nq"] * hd * SIZE[case["dtype"]]
        return {"bytes": read * pos + io, "flops": 4 * hd * case["nq"] * pairs}
    if op == "append":
        total = sum(_lengths(case)[1])
        kv = total * 2 * nkv * hd
        io = total * hd * (2 * case["nq"] + 2 * nkv) * SIZE[case["dtype"]] + total * case["rot"] * 4
        # the pages are written once and read once, and their values come back in 32 bits
        return {"bytes": io + 2 * kv // 64 * 40 + 4 * kv, "flops": 6 * total * (case["nq"] + 2 * nkv) * hd}
    if op == "copy":
        moved = case["L"] * case["n"] * pos
        values = case["L"] * case["n"] * 2 * nkv * hd * 4
        return {"bytes": moved * (1 + 2 * case["children"]) + values * case["children"], "flops": 0}
    rows = case["B"] * case["L"] * case["n"]
    return {"bytes": rows * pos + rows * 2 * nkv * hd * SIZE[case["dtype"]], "flops": 2 * rows * 2 * nkv * hd}


# ---- the definitions in 64 bits --------------------------------------------------------


def _exact_extend(s):
    case = s["case"]
    G, hd = case["nq"] // case["nkv"], case["hd"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.full(s["q"].shape[:2], -math.inf, dtype=torch.float64, device="cuda")
    first = 0
    for b, (a, n) in enumerate(zip(s["old"], s["new"])):
        i = torch.arange(n, device="cuda")[:, None]
        j = torch.arange(a + n, device="cuda")[None, :]
        ban = j > a + i
        if case["window"]:
            ban |= a + i - j >= case["window"]
        if s["tree"] is not None:
            bits = s["tree"][first : first + n]
            for t in range(n):
                ban[:, a + t] |= bits.bitwise_right_shift(t).bitwise_and(1) == 0
        for h in range(case["nkv"]):
            kk = _values64(s["w"][b, 0, h, : a + n], s["scale"][b, 0, h, : a + n], s["bias"][b, 0, h, : a + n])
            vv = _values64(s["w"][b, 1, h, : a + n], s["scale"][b, 1, h, : a + n], s["bias"][b, 1, h, : a + n])
            for g in range(G):
                z = s["q"][first : first + n, h * G + g].double() @ kk.T * hd ** -0.5
                z[ban] = -math.inf
                l = torch.logsumexp(z, -1)
                p = torch.exp(z - l[:, None])
                p[ban] = 0
                out[first : first + n, h * G + g] = p @ vv
                lse[first : first + n, h * G + g] = l
        first += n
    return {"out": out, "lse": lse} if case["dtype"] == "f32" else out


def _exact_append(s):
    """The rotation in 64 bits; what is held is the rotated key rounded to 32 bits, then quantised by the cache's rule."""
    case = s["case"]
    nq, nkv, hd, pairs = case["nq"], case["nkv"], case["hd"], case["rot"] // 2
    x = s["qkv"].view(-1, nq + 2 * nkv, hd).double().clone()
    first = 0
    for axis, n in enumerate(s["sections"]):
        at = s["pos"][axis].long()
        for i in range(first, first + n):
            lo, hi = (2 * i, 2 * i + 1) if case["interleaved"] else (i, i + pairs)
            c, d = s["cos"][at, i].double()[:, None], s["sin"][at, i].double()[:, None]
            p, q = x[:, : nq + nkv, lo].clone(), x[:, : nq + nkv, hi].clone()
            x[:, : nq + nkv, lo], x[:, : nq + nkv, hi] = p * c - q * d, q * c + p * d
        first += n
    held = []
    for part in (x[:, nq : nq + nkv], x[:, nq + nkv :]):
        g = part.float().reshape(-1, 64)
        low = g.min(1, keepdim=True).values
        span = g.max(1, keepdim=True).values - low
        flat = span == 0
        one = torch.ones_like(span)
        step = torch.where(flat, one, span.div(one * 15))
        n = g.sub(low).mul(torch.where(flat, one * 0, (one * 15).div(span))).add(0.5).to(torch.int32).clamp(0, 15)
        held.append((n.double() * step.double() + low.double()).view(-1, nkv, hd))
    return {"q": x[:, :nq], "kv": torch.stack(held)[None]}


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "extend":
        return _exact_extend(s)
    if op == "append":
        return _exact_append(s)
    v = _values64(s["w"], s["scale"], s["bias"])
    if op == "copy":
        if case["gather"]:
            v = torch.stack([torch.stack([torch.stack([v[l, x, h][s["index"][l, h].long()] for h in range(case["nkv"])]) for x in (0, 1)]) for l in range(case["L"])])
        else:
            v = v[:, :, :, -case["n"] :]
        return torch.cat([v.transpose(2, 3)] * case["children"], 2)
    return torch.cat([v[b, :, :, :, a : a + case["n"]].transpose(2, 3) for b, a in enumerate(s["begin"])], 2)
