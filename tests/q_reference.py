"""Plain implementations in 64 bits of the operators on compressed data, for
their tests: rotary positions, the 8-bit KV cache, 4-bit weights."""
import numpy as np

U = 2.0 ** -24  # half a step of float32, relative


def rotary(x, positions, freq, halves, magnitude=1.0, inverse=False):
    """x [B,T,H,D] float64; positions [B,T]; freq [P]."""
    p = len(freq)
    a = positions.astype(np.float64)[..., None] * freq * (-1.0 if inverse else 1.0)
    c, s = np.cos(a)[:, :, None], np.sin(a)[:, :, None]
    i0, i1 = (slice(0, p), slice(p, 2 * p)) if halves else (slice(0, 2 * p, 2), slice(1, 2 * p, 2))
    out = x.astype(np.float64).copy()
    x0, x1 = out[..., i0].copy(), out[..., i1].copy()
    out[..., i0] = magnitude * (x0 * c - x1 * s)
    out[..., i1] = magnitude * (x0 * s + x1 * c)
    return out


def rotary_bound(x, freq, halves, magnitude, eps):
    """|x0| + |x1| of every element's pair, times magnitude and eps."""
    p = len(freq)
    i0, i1 = (slice(0, p), slice(p, 2 * p)) if halves else (slice(0, 2 * p, 2), slice(1, 2 * p, 2))
    b = np.zeros(x.shape)
    both = np.abs(x[..., i0]) + np.abs(x[..., i1])
    b[..., i0] = b[..., i1] = both * abs(magnitude) * eps
    return b


def append(x, cache, scale, start, count, block):
    """One sequence and head, in place: x [Tn,D] float32, cache [Tcap,D] int8,
    scale [blocks] float32. Whole numbers from quotients in 64 bits: the quotient
    of two float32 (or of n * float32 by a float32) differs from every tie by far
    more than a 64-bit rounding, unless it is one."""
    lo, end = max(start, 0), min(start + count, cache.shape[0])
    if lo >= end:
        return
    for j in range(lo // block, (end - 1) // block + 1):
        a, b = max(lo, j * block), min(end, (j + 1) * block)
        rows = x[a - start:b - start]
        with np.errstate(all="ignore"):
            top = np.float32(np.nan) if np.isnan(rows).any() else np.abs(rows).max()
            s = np.float32(top * (np.float32(1) / np.float32(127)))
            if j * block < lo:
                old = np.abs(scale[j])
                s = old if np.isnan(old) or (not np.isnan(s) and old > s) else s
                if not (s == old):
                    held = cache[j * block:lo].astype(np.float64) * np.float64(old) / np.float64(s)
                    cache[j * block:lo] = np.clip(np.rint(held), -127, 127) if np.isfinite(s) and s > 0 else 0
            scale[j] = s
            ok = np.isfinite(s) and s > 0
            cache[a:b] = np.clip(np.rint(rows.astype(np.float64) / np.float64(s)), -127, 127) if ok else 0


def make_cache(g, B, H, T, D, block):
    """A filled cache: whole numbers in [-127, 127] and a positive scale per block."""
    q = g.integers(-127, 128, (B, H, T, D)).astype(np.int8)
    s = (g.uniform(0.2, 2.0, (B, H, -(-T // block))) / 127).astype(np.float32)
    return q, s


def attend(q, kc, vc, ks, vs, lengths, block, scale, g, causal=True):
    """q [B,Tq,Hq,D], caches int8 [B,Hkv,T,D]. Returns the output in 64 bits and
    a bound on a float32 implementation's error, whatever its order of sums:
    d = scale * max_j sum_d |q k| * (D u 2 + 2^-20) for a score (products of
    operands split into parts of 22 bits or more among them), 2 d + (n + 8) 2 u of
    sum p |v| for the output. A probability in two fp16 parts, scaled so that the
    row's largest is 2^13 or more, is a multiple of fp16's smallest number 2^-24:
    off by at most 2^-25 / 2^13 = 2^-38 of the largest, which matters where the
    keys of large p have v = 0: n 2^-38 max |v| more (p relative to the largest is
    at least p itself)."""
    B, Tq, Hq, D = q.shape
    T = kc.shape[2]
    blk = np.arange(T) // block
    out, tol = np.zeros(q.shape), np.zeros(q.shape)
    for b in range(B):
        length = T if lengths is None else int(np.clip(lengths[b], 0, T))
        for i in range(Tq):
            n = length - Tq + 1 + i if causal else length
            if n <= 0:
                continue
            for h in range(Hq):
                k = kc[b, h // g, :n].astype(np.float64) * ks[b, h // g].astype(np.float64)[blk[:n], None]
                v = vc[b, h // g, :n].astype(np.float64) * vs[b, h // g].astype(np.float64)[blk[:n], None]
                qq = q[b, i, h].astype(np.float64)
                s = (k @ qq) * scale
                p = np.exp(s - s.max())
                p /= p.sum()
                out[b, i, h] = p @ v
                d = abs(scale) * (np.abs(k) @ np.abs(qq)).max() * (2 * D * U + 2.0 ** -20)
                tol[b, i, h] = (2 * d + (n + 8) * 2 * U) * (p @ np.abs(v)) + n * 2.0 ** -38 * np.abs(v).max(0) + 1e-30
    return out, tol


def quantise_weight(w, group):
    """W [K,N] float32 -> nibbles u [K,N] (0..15) and scales [groups,N]."""
    K, N = w.shape
    G = -(-K // group)
    u, s = np.full((K, N), 8, np.int64), np.zeros((G, N), np.float32)
    for g in range(G):
        rows = slice(g * group, min(K, (g + 1) * group))
        with np.errstate(all="ignore"):
            top = np.abs(w[rows]).max(0)  # NaN wins in numpy's max
            s[g] = (top / np.float32(7)).astype(np.float32)
            ok = np.isfinite(s[g]) & (s[g] > 0)
            n = np.clip(np.rint(w[rows].astype(np.float64) / s[g].astype(np.float64)), -7, 7)
        u[rows] = np.where(ok, n, 0) + 8
    return u, s


def pack_words(u):
    K, N = u.shape
    words = np.zeros((K // 8, N), np.uint32)
    for j in range(8):
        words |= (u[j::8].astype(np.uint32) & 15) << np.uint32(4 * j)
    return words.view(np.int32)


def linear(x, u, s, group, bias=None, act="none", residual=None):
    """Output in 64 bits and a float32 implementation's bound: sums of K products
    in any order, 2 (K + 16) u of sum |x||W| + |bias|, times 1.2 for the slope of
    an activation, and a few roundings of the result."""
    from scipy.special import erf
    K = x.shape[1]
    w = (u - 8).astype(np.float64) * np.repeat(s.astype(np.float64), group, 0)[:K]
    y = x.astype(np.float64) @ w
    size = np.abs(x).astype(np.float64) @ np.abs(w)
    if bias is not None:
        y, size = y + bias, size + np.abs(bias)
    if act == "relu":
        y = np.where(y > 0, y, 0)
    elif act == "silu":
        y = y / (1 + np.exp(-y))
    elif act == "gelu":
        y = 0.5 * y * (1 + erf(y / np.sqrt(2)))
    tol = 1.2 * 2 * (K + 16) * U * size + 8 * U * np.abs(y) + 1e-30
    if residual is not None:
        y = y + residual
        tol = tol + 2 * U * np.abs(y)
    return y, tol


def assert_within(got, want, tol, what=""):
    got = np.asarray(got, np.float64)
    assert np.isfinite(got).all(), f"{what}: not finite"
    off = np.abs(got - want)
    if not (off <= tol).all():
        i = np.unravel_index(np.argmax(off - tol), off.shape)
        raise AssertionError(f"{what}: {got[i]!r} vs {want[i]!r} at {i}, off {off[i]:.3g} of {tol[i]:.3g} "
                             f"({int((off > tol).sum())} of {off.size})")
