"""Timed cases of the decode operators on compressed data: rotary positions per
token, the KV cache held in 8 bits (append, read-back, attention) and products
with 4-bit weights.

Each case is one pass through one operator as a decoder's step makes it. `run`
computes it in elementary torch operations, or, where `own` is true, by the
calls a user makes of alpakann_b200.onHost.nn. Outputs live in buffers that
the program keeps, as a serving loop does.
"""
import math

import torch

own = False

LEVELS = 127  # an 8-bit cache value is a whole number of -127..127


# ---- cases ------------------------------------------------------------------
def _attend(name, b, tq, hq, hkv, d, cap, block, lengths):
    case = {"op": "attend", "b": b, "tq": tq, "hq": hq, "hkv": hkv, "d": d, "cap": cap, "block": block,
            "lengths": lengths}
    return dict(case, name=name) if name else case


def _cache(name, b, tn, hkv, d, cap, block, start):
    case = {"op": "cache", "b": b, "tn": tn, "hkv": hkv, "d": d, "cap": cap, "block": block, "start": start}
    return dict(case, name=name) if name else case


def _rotary(name, b, t, hq, hkv, d, rot, pairs, first, dtype, inverse):
    case = {"op": "rotary", "b": b, "t": t, "hq": hq, "hkv": hkv, "d": d, "rot": rot, "pairs": pairs, "first": first,
            "dtype": dtype, "inverse": inverse}
    return dict(case, name=name) if name else case


def _linear(name, m, k, n, group, bias, act, residual):
    case = {"op": "linear", "m": m, "k": k, "n": n, "group": group, "bias": bias, "act": act, "residual": residual}
    return dict(case, name=name) if name else case


def listed():
    return [
        # a single conversation a few hundred tokens in: a latency-bound call
        _attend("attend 1x300", 1, 1, 32, 8, 128, 512, 64, 300),
        # the decode configuration of batch 8 over 2048 keys, 32 heads of 128, every head with its own keys
        _attend("attend 8x2048 32/32", 8, 1, 32, 32, 128, 2048, 64, "full"),
        # four tokens checked at once in a batch of uneven lengths with an empty slot, heads of 64
        _attend("attend 12x4x4096 ragged", 12, 4, 16, 4, 64, 4096, 16, "ragged"),
        # one very long context: few rows, so the key axis has to be split
        _attend("attend 1x131072", 1, 1, 32, 4, 128, 131072, 128, "full"),
        # the long decode configuration (batch 16, 32768 keys, 64 heads of 128) with eight query heads a KV head
        _attend("attend 16x32768 64/8", 16, 1, 64, 8, 128, 32768, 64, "full"),
        # a serving step's new rows, one a sequence, into part-filled blocks, and a short cache read back
        _cache("cache 8x1", 8, 1, 8, 128, 256, 64, 201),
        # a prompt's chunk appended behind earlier tokens, then read back for the fp32 prefill kernel
        _cache("cache 4x2048", 4, 2048, 8, 128, 4096, 64, 1000),
        # a decode step's queries and keys: half pairs, half of the head, far positions
        _rotary("rotary 16x1 half", 16, 1, 64, 8, 128, 64, "halves", 100000, "float32", False),
        # the prefill configuration of batch 4 x 4096 tokens, 32 heads of 128, interleaved pairs
        _rotary("rotary 4x4096", 4, 4096, 32, 32, 128, 128, "interleaved", 0, "float32", False),
        # gradient with respect to the inputs in fp64: batch 2 x 1024, 16 heads of 64
        _rotary("rotary 2x1024 fp64 grad", 2, 1024, 16, 16, 64, 64, "halves", 0, "float64", True),
        # one token through a 4096-wide output projection, added to the residual stream
        _linear("linear 1x4096x4096", 1, 4096, 4096, 128, False, "none", True),
        # a batch of eight through the 4096 -> 16384 layer of an MLP, bias and silu behind it
        _linear("linear 8x4096x16384", 8, 4096, 16384, 64, True, "silu", False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attend", "attend", "cache", "rotary", "linear", "linear"])
    if op == "attend":
        g = rng.choice([1, 2, 4, 7, 8])
        hkv = _log(rng, 1, 16)
        d = rng.choice([64, 128, 128, 256])
        block = rng.choice([16, 32, 64, 128])
        tq = rng.choice([1, 1, 1, 2, 5])
        b = _log(rng, 1, 64)
        most = 16 * 32768 * 8 * 128 // (b * hkv * d * tq)
        cap = max(8, _log(rng, 8, max(9, min(131072, most))))
        return _attend("", b, tq, g * hkv, hkv, d, cap, block, rng.choice(["full", "ragged"]))
    if op == "cache":
        b, hkv, d = _log(rng, 1, 16), _log(rng, 1, 16), rng.choice([64, 96, 128, 256])
        tn = max(1, min(_log(rng, 1, 2048), 4 * 2048 * 8 * 128 // (b * hkv * d)))
        start = _log(rng, 1, 2048) - 1
        start = min(start, max(0, 4 * 4096 * 8 * 128 // (b * hkv * d) - tn))
        return _cache("", b, tn, hkv, d, start + tn + rng.randrange(64), rng.choice([16, 32, 64, 128]), start)
    if op == "rotary":
        hkv, g = _log(rng, 1, 16), rng.choice([1, 2, 4, 8])
        d = rng.choice([64, 80, 96, 128, 256])
        rot = rng.choice([d, d, d // 2, d // 4])
        b = _log(rng, 1, 16)
        dtype = rng.choice(["float32", "float32", "float64"])
        most = 4 * 4096 * 64 * 128 // (b * hkv * (g + 1) * d * (2 if dtype == "float64" else 1))
        t = _log(rng, 1, max(2, min(8192, most)))
        first = _log(rng, 1, 200000) - 1
        return _rotary("", b, t, g * hkv, hkv, d, rot, rng.choice(["halves", "interleaved"]), first, dtype,
                       rng.random() < 0.3)
    group = rng.choice([32, 64, 128])
    k = 8 * _log(rng, 16, 2048)
    n = min(_log(rng, 64, 32768), 4096 * 16384 // k)
    if rng.random() < 0.8:
        n = 4 * max(1, n // 4)
    return _linear("", rng.choice([1, 1, 2, 3, 5, 8, 16]), k, n, group, rng.random() < 0.5,
                   rng.choice(["none", "none", "relu", "silu", "gelu"]), rng.random() < 0.5)


def _lengths(case):
    """Keys each sequence holds: all of the cache, a number of them, or spread up to it (in a batch of four or more with
    one empty slot)."""
    b, cap = case["b"], case["cap"]
    if case["lengths"] == "full":
        return [cap] * b
    if case["lengths"] != "ragged":
        return [case["lengths"]] * b
    spread = [max(1, cap * (2 * i + 1) // (2 * b)) for i in range(b)]
    return [0] + spread[1:] if b >= 4 else spread


def _starts(case):
    """First new token of each sequence, and how many of the padded rows are real."""
    starts = [max(0, case["start"] - 7 * i) for i in range(case["b"])]
    counts = [max(1, case["tn"] - i % 3) for i in range(case["b"])]
    return starts, counts


# ---- inputs -----------------------------------------------------------------
def _quantised(shape, block, gen):
    """A filled 8-bit cache [B,H,T,D]: normal rows of varying size, and the scale of each block of tokens and head."""
    b, h, t, d = shape
    nb = -(-t // block)
    q = torch.empty(shape, dtype=torch.int8, device="cuda")
    scale = torch.empty((b, h, nb), device="cuda")
    for i in range(b):
        x = torch.randn((h, nb, block, d), device="cuda", generator=gen)
        x *= 0.5 + torch.rand((h, nb, 1, 1), device="cuda", generator=gen)
        s = x.abs().amax((2, 3)) / LEVELS
        q[i] = (x / s[:, :, None, None]).round_().to(torch.int8).view(h, nb * block, d)[:, :t]
        scale[i] = s
    return q, scale


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)

    def randn(*shape, dtype=torch.float32):
        return torch.randn(shape, device="cuda", generator=gen, dtype=dtype)

    op = case["op"]
    if op == "attend":
        shape = (case["b"], case["hkv"], case["cap"], case["d"])
        kc, ks = _quantised(shape, case["block"], gen)
        vc, vs = _quantised(shape, case["block"], gen)
        q = randn(case["b"], case["tq"], case["hq"], case["d"]) * 1.5
        return {"op": op, "q": q, "kc": kc, "ks": ks, "vc": vc, "vs": vs, "lengths": _ints(_lengths(case)),
                "out": torch.empty_like(q), "block": case["block"], "group": case["hq"] // case["hkv"],
                "scale": 1.0 / math.sqrt(case["d"])}
    if op == "cache":
        shape = (case["b"], case["hkv"], case["cap"], case["d"])
        kc, ks = _quantised(shape, case["block"], gen)
        vc, vs = _quantised(shape, case["block"], gen)
        new = (case["b"], case["tn"], case["hkv"], case["d"])
        starts, counts = _starts(case)
        return {"op": op, "kc": kc, "ks": ks, "vc": vc, "vs": vs, "kn": randn(*new), "vn": randn(*new),
                "starts": _ints(starts), "counts": _ints(counts),
                "ends": _ints([s + c for s, c in zip(starts, counts)]), "block": case["block"],
                "ko": torch.zeros(shape, device="cuda"), "vo": torch.zeros(shape, device="cuda")}
    if op == "rotary":
        dtype = getattr(torch, case["dtype"])
        q = randn(case["b"], case["t"], case["hq"], case["d"], dtype=dtype)
        k = randn(case["b"], case["t"], case["hkv"], case["d"], dtype=dtype)
        pair = torch.arange(case["rot"] // 2, dtype=torch.float64, device="cuda")
        first = torch.arange(case["b"], device="cuda")[:, None] * 3 + case["first"]
        positions = (first + torch.arange(case["t"], device="cuda")[None, :]).to(torch.int32)
        return {"op": op, "q": q, "k": k, "positions": positions, "freq": 1e4 ** (-2.0 * pair / case["rot"]),
                "halves": case["pairs"] == "halves", "inverse": case["inverse"], "oq": torch.empty_like(q),
                "ok": torch.empty_like(k)}
    k, n, group = case["k"], case["n"], case["group"]
    packed = torch.randint(-2**31, 2**31, (k // 8, n), device="cuda", generator=gen, dtype=torch.int64).to(torch.int32)
    scales = (0.5 + torch.rand((-(-k // group), n), device="cuda", generator=gen)) * (0.2 / math.sqrt(k))
    return {"op": op, "x": randn(case["m"], k), "packed": packed, "scales": scales, "group": group, "act": case["act"],
            "bias": randn(n) if case["bias"] else None, "res": randn(case["m"], n) if case["residual"] else None,
            "y": torch.empty((case["m"], n), device="cuda")}


# ---- the plain forms ----------------------------------------------------------
def _values(cache, scale, block):
    """What an 8-bit cache stands for: each whole number times its block's scale."""
    t = cache.shape[2]
    return cache.float() * scale.repeat_interleave(block, dim=2)[:, :, :t, None]


def _plain_attend(s):
    q, g = s["q"], s["group"]
    b, tq, hq, d = q.shape
    hkv, t = s["kc"].shape[1], s["kc"].shape[2]
    k, v = _values(s["kc"], s["ks"], s["block"]), _values(s["vc"], s["vs"], s["block"])
    rows = q.view(b, tq, hkv, g, d).permute(0, 2, 1, 3, 4).reshape(b, hkv, tq * g, d)
    scores = (rows @ k.transpose(2, 3)).view(b, hkv, tq, g, t) * s["scale"]
    # query i of the last tq tokens sees the keys up to its own
    seen = s["lengths"][:, None] - tq + 1 + torch.arange(tq, device="cuda")
    keep = torch.arange(t, device="cuda") < seen[:, :, None]
    scores = scores.masked_fill(~keep[:, None, :, None, :], -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = (scores - torch.where(top == -math.inf, 0.0, top)).exp()
    total = p.sum(-1, keepdim=True)
    p = (p / torch.where(total == 0, 1.0, total)).view(b, hkv, tq * g, t)
    s["out"].copy_((p @ v).view(b, hkv, tq, g, d).permute(0, 2, 1, 3, 4).reshape(b, tq, hq, d))
    return s["out"]


def _plain_append(new, cache, scale, starts, counts, block):
    """New rows into the cache: each touched block keeps one scale, its earlier rows are rounded anew where it grows."""
    b, tn, h, d = new.shape
    t, nb = cache.shape[2], scale.shape[2]
    token = torch.arange(nb * block, device="cuda")
    at = token[None, :] - starts[:, None]
    fresh = (at >= 0) & (at < counts[:, None]) & (token < t)
    rows = new.transpose(1, 2).gather(2, at.clamp(0, tn - 1)[:, None, :, None].expand(b, h, nb * block, d))
    rows = torch.where(fresh[:, None, :, None], rows, 0.0).view(b, h, nb, block, d)
    touched = fresh.view(b, 1, nb, block).any(-1)
    begun = (torch.arange(nb, device="cuda") * block)[None, None, :] < starts[:, None, None]
    grown = torch.maximum(rows.abs().amax((3, 4)) / LEVELS, torch.where(begun, scale, 0.0))
    now = torch.where(touched, grown, scale)
    pad = torch.zeros((b, h, nb * block, d), device="cuda")
    pad[:, :, :t] = cache
    # quotients next to a border between two whole numbers need more than 32 bits
    held = (pad.view(b, h, nb, block, d) * scale[..., None, None].double() / now[..., None, None].double()).round()
    fresh_q = (rows.double() / now[..., None, None].double()).round()
    early = (touched[..., None] & (token.view(nb, block)[None, None] < starts[:, None, None, None]))[..., None]
    out = torch.where(early, held, pad.view(b, h, nb, block, d).double())
    out = torch.where(fresh.view(b, 1, nb, block, 1), fresh_q, out).clamp(-LEVELS, LEVELS)
    cache.copy_(out.view(b, h, nb * block, d)[:, :, :t])
    scale.copy_(now)


def _plain_cache(s):
    for new, cache, scale, out in (("kn", "kc", "ks", "ko"), ("vn", "vc", "vs", "vo")):
        _plain_append(s[new], s[cache], s[scale], s["starts"], s["counts"], s["block"])
        valid = torch.arange(s[cache].shape[2], device="cuda")[None, :] < s["ends"][:, None]
        s[out].copy_(torch.where(valid[:, None, :, None], _values(s[cache], s[scale], s["block"]), s[out]))
    return s["ko"], s["vo"], s["ks"], s["vs"]


def _plain_rotary(s):
    angle = s["positions"].double()[..., None] * s["freq"]  # far positions: angles in 64 bits
    if s["inverse"]:
        angle = -angle
    r = 2 * s["freq"].shape[0]
    for name, to in (("q", "oq"), ("k", "ok")):
        x = s[name]
        c, sn = angle.cos().to(x.dtype)[:, :, None, :], angle.sin().to(x.dtype)[:, :, None, :]
        if s["halves"]:
            a, b = x[..., : r // 2], x[..., r // 2 : r]
            turned = torch.cat((a * c - b * sn, a * sn + b * c), -1)
        else:
            a, b = x[..., 0:r:2], x[..., 1:r:2]
            turned = torch.stack((a * c - b * sn, a * sn + b * c), -1).flatten(-2)
        s[to].copy_(torch.cat((turned, x[..., r:]), -1))
    return s["oq"], s["ok"]


def _plain_linear(s):
    k = s["x"].shape[1]
    shifts = torch.arange(0, 32, 4, device="cuda", dtype=torch.int32)
    nibble = (s["packed"][:, None, :] >> shifts[None, :, None]) & 15
    w = (nibble.reshape(k, -1) - 8).float() * s["scales"].repeat_interleave(s["group"], dim=0)[:k]
    y = s["x"] @ w
    if s["bias"] is not None:
        y = y + s["bias"]
    if s["act"] == "relu":
        y = torch.where(y > 0, y, 0.0)
    elif s["act"] == "silu":
        y = y / (1 + (-y).exp())
    elif s["act"] == "gelu":
        y = 0.5 * y * (1 + torch.erf(y / math.sqrt(2)))
    s["y"].copy_(y if s["res"] is None else y + s["res"])
    return s["y"]


def run(state):
    s = state
    if not own:
        return {"attend": _plain_attend, "cache": _plain_cache, "rotary": _plain_rotary,
                "linear": _plain_linear}[s["op"]](s)
    from alpakann_b200.onHost import nn
    if s["op"] == "attend":
        nn.attentionDecodeQ8(None, None, s["q"], s["kc"], s["vc"], s["ks"], s["vs"], s["out"], s["block"],
                             s["lengths"], s["scale"], s["group"])
        return s["out"]
    if s["op"] == "cache":
        nn.kvCacheAppendQ8(None, None, s["kn"], s["vn"], s["kc"], s["vc"], s["ks"], s["vs"], s["starts"], s["block"],
                           s["counts"])
        nn.kvCacheReadQ8(None, None, s["kc"], s["vc"], s["ks"], s["vs"], s["ko"], s["vo"], s["block"], s["ends"])
        return s["ko"], s["vo"], s["ks"], s["vs"]
    if s["op"] == "rotary":
        pairs = nn.RotaryPairs.halves if s["halves"] else nn.RotaryPairs.interleaved
        nn.rotary(None, None, s["q"], s["k"], s["positions"], s["freq"], s["oq"], s["ok"], pairs,
                  inverse=s["inverse"])
        return s["oq"], s["ok"]
    nn.linearQ4(None, None, s["x"], s["packed"], s["scales"], s["y"], s["group"], s["bias"],
                nn.Activation[s["act"]], s["res"])
    return s["y"]


# ---- what a pass cannot do without ---------------------------------------------
def work(case):
    op = case["op"]
    if op == "attend":
        keys, rows = sum(_lengths(case)), case["b"] * case["tq"] * case["hq"] * case["d"]
        per_key = case["hkv"] * 2 * (case["d"] + 4 / case["block"])
        return {"bytes": keys * per_key + 8 * rows, "flops": 4 * case["d"] * case["tq"] * case["hq"] * keys}
    if op == "cache":
        starts, counts = _starts(case)
        row, block = 2 * case["hkv"] * case["d"], case["block"]
        new, total = sum(counts), sum(starts) + sum(counts)
        early = sum(s % block for s in starts)  # earlier rows of a block whose scale grows: read and written
        return {"bytes": row * (new * 5 + early * 2 + total * 5), "flops": row * (new * 3 + early * 2 + total)}
    if op == "rotary":
        values = case["b"] * case["t"] * (case["hq"] + case["hkv"]) * case["d"]
        size = 8 if case["dtype"] == "float64" else 4
        return {"bytes": 2 * size * values, "flops": 3 * values * case["rot"] / case["d"]}
    m, k, n = case["m"], case["k"], case["n"]
    weights = k * n / 2 + 4 * -(-k // case["group"]) * n
    return {"bytes": weights + 4 * m * (k + n * (2 if case["residual"] else 1)) + (4 * n if case["bias"] else 0),
            "flops": 2 * m * k * n}


# ---- the definitions in 64 bits -------------------------------------------------
def _exact_attend(s):
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    tq, g = s["q"].shape[1], s["group"]
    for b, length in enumerate(s["lengths"].tolist()):
        for h in range(s["kc"].shape[1]):
            block = torch.arange(length, device="cuda") // s["block"]
            k = s["kc"][b, h, :length].double() * s["ks"][b, h].double()[block][:, None]
            v = s["vc"][b, h, :length].double() * s["vs"][b, h].double()[block][:, None]
            for i in range(tq):
                n = length - tq + 1 + i
                if n > 0:
                    x = torch.einsum("gd,jd->gj", s["q"][b, i, h * g : (h + 1) * g].double(), k[:n])
                    out[b, i, h * g : (h + 1) * g] = torch.softmax(x * s["scale"], -1) @ v[:n]
    return out


def _exact_cache(s):
    res = []
    for new, cache, scale in (("kn", "kc", "ks"), ("vn", "vc", "vs")):
        n, q, sc = s[new].double(), s[cache].double(), s[scale].clone()
        out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
        for b, (start, count) in enumerate(zip(s["starts"].tolist(), s["counts"].tolist())):
            end, bl = start + count, s["block"]
            for j in range(start // bl, (end - 1) // bl + 1):
                lo, hi = max(start, j * bl), min(end, (j + 1) * bl)
                rows = n[b, lo - start : hi - start].transpose(0, 1)  # [H, rows, D]
                wanted = (rows.abs().amax((1, 2)) / LEVELS).float()  # a scale is stored in 32 bits
                if j * bl < start:
                    wanted = torch.maximum(wanted, sc[b, :, j])
                    held = q[b, :, j * bl : start] * sc[b, :, j, None, None].double()
                    q[b, :, j * bl : start] = torch.round(held / wanted[:, None, None].double())
                sc[b, :, j] = wanted
                q[b, :, lo:hi] = torch.round(rows / wanted[:, None, None].double())
            block = torch.arange(end, device="cuda") // bl
            out[b, :, :end] = q[b, :, :end] * sc[b].double()[:, block][:, :, None]
        res.append((out, sc.double()))
    return res[0][0], res[1][0], res[0][1], res[1][1]


def _exact_rotary(s):
    r = 2 * s["freq"].shape[0]
    sign = -1.0 if s["inverse"] else 1.0
    turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"),
                       sign * torch.einsum("bt,p->btp", s["positions"].double(), s["freq"]))[:, :, None, :]
    res = []
    for x in (s["q"].double(), s["k"].double()):
        out = x.clone()
        first, second = (slice(0, r // 2), slice(r // 2, r)) if s["halves"] else (slice(0, r, 2), slice(1, r, 2))
        z = torch.complex(x[..., first].contiguous(), x[..., second].contiguous()) * turn
        out[..., first], out[..., second] = z.real, z.imag
        res.append(out)
    return tuple(res)


def _exact_linear(s):
    x = s["x"].double()
    y = torch.zeros(s["y"].shape, dtype=torch.float64, device="cuda")
    for j in range(8):  # the j-th nibble of every word is input 8 r + j
        level = torch.bitwise_and(torch.bitwise_right_shift(s["packed"], 4 * j), 15).double() - 8
        group = torch.arange(j, x.shape[1], 8, device="cuda") // s["group"]
        y += x[:, j::8] @ (level * s["scales"].double()[group])
    if s["bias"] is not None:
        y += s["bias"].double()
    if s["act"] == "relu":
        y = y.clamp_min(0)
    elif s["act"] == "silu":
        y = y * torch.sigmoid(y)
    elif s["act"] == "gelu":
        y = y * (0.5 + 0.5 * torch.special.erf(y * math.sqrt(0.5)))
    return y if s["res"] is None else y + s["res"].double()


def exact(case, seed):
    s = prepare(case, seed)
    return {"attend": _exact_attend, "cache": _exact_cache, "rotary": _exact_rotary, "linear": _exact_linear}[s["op"]](s)
