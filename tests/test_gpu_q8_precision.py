"""attentionDecodeQ8 where keys add very different amounts to a row: what the softmax
keeps has to come out to fp32 accuracy however large the scales, or the probabilities,
of the keys that add nothing are.

Bounds, u = 2^-24, relative to sum p |v| of the output element unless said:
  * a score s_j (in nats): q and K's products are whole numbers summed exactly, then
    four roundings of their sum, its factor (four roundings) and the difference to the
    maximum: 10 u (|s_j| + |s_max|); q itself to 2^-31 of its largest element, and the
    middle digits' sums (2^-6 of the whole) to u: (2^-31 + 2^-28) scale max|q| sum |k_j|;
  * 2^x: 2^-22 relative, 4 u; times V's scale u; two fp16 parts of it 2^-23, 2 u;
  * sums of a tile: two products of depth 16 whose terms may be cut at 2^-23 of the
    largest of 17, 68 u; a rounding for the tile, one for the maximum's step, one for its
    unit: 3 u for each tile of a warp; 40 u for the merges of warps, CTAs and windows;
  * the divisor: the same score errors, one rounding a tile and the merges, relative to
    the output.
Roundings are independent and most of them cancel, so the root mean square over a row is
held to less: 4 u (the exponential's 2^-22, should it have one sign) and four times that
of the same formulas in float32.
"""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


@pytest.fixture(scope="module")
def nn():
    from tests.helpers import build_library
    build_library()
    from alpakann_b200.onHost import nn
    return nn


def attend(q, kc, vc, ks, vs, block, scale, g):
    """One sequence and one query token, every key seen: q [Hq,D], caches int8 [Hkv,T,D].
    Output in 64 bits, the bound on every element, sum p |v|, and the output in float32."""
    Hq, D = q.shape
    T = kc.shape[1]
    blk = np.arange(T) // block
    tiles = -(-T // 16 // 4) if D == 256 else -(-T // 32 // 4)
    out, tol, size = (np.zeros(q.shape) for _ in range(3))
    single = np.zeros(q.shape, np.float32)
    for h in range(Hq):
        k = kc[h // g].astype(np.float64) * ks[h // g].astype(np.float64)[blk, None]
        v = vc[h // g].astype(np.float64) * vs[h // g].astype(np.float64)[blk, None]
        qq = q[h].astype(np.float64)
        s = (k @ qq) * scale
        p = np.exp(s - s.max())
        p /= p.sum()
        e = 10 * U * (np.abs(s) + abs(s.max())) + abs(scale) * np.abs(qq).max() * np.abs(k).sum(1) * (2.0 ** -31 + 2.0 ** -28)
        out[h] = p @ v
        size[h] = p @ np.abs(v)
        tol[h] = (p * (e + (7 + 68 + 3 * tiles + 40) * U)) @ np.abs(v) + ((p @ e) + (4 + tiles + 40) * U) * np.abs(out[h])
        k, v = k.astype(np.float32), v.astype(np.float32)
        s = (k @ q[h]) * np.float32(scale)
        p = np.exp(s - s.max())
        single[h] = (p / p.sum()) @ v
    return out, tol, size, single


def check(nn, q, kc, vc, ks, vs, block, scale, g, what):
    with np.errstate(under="ignore"):
        want, tol, size, single = attend(q, kc, vc, ks, vs, block, scale, g)
    dev = [torch.from_numpy(np.ascontiguousarray(a)).cuda() for a in (q[None, None], kc[None], vc[None], ks[None], vs[None])]
    out = torch.full(dev[0].shape, float("nan"), device="cuda")
    nn.attentionDecodeQ8(None, None, *dev, out, block, None, scale, g)
    off = np.abs(out.cpu().numpy()[0, 0].astype(np.float64) - want)
    assert np.isfinite(off).all(), what
    worst = (off / np.maximum(tol, 1e-300)).max()
    rms = lambda e: np.sqrt(((e / size) ** 2).mean(1))
    spread = (rms(off) / (4 * rms(single - want) + 4 * U)).max()
    assert worst <= 1 and spread <= 1, f"{what}: {worst:.3g} of the bound, {spread:.3g} of the root mean square's"


def keys(g, Hkv, T, D, levels):
    """K whose score with queries of the same first eight elements is 8 * level plus noise, in units of K's scale."""
    k = g.integers(-10, 11, (Hkv, T, D))
    k[:, :, :8] = np.asarray(levels)[..., None]
    return k.astype(np.int8)


def queries(g, Hq, D):
    q = g.standard_normal((Hq, D)) * 0.05
    q[:, :8] = 1.0
    return q.astype(np.float32)


ROWS = [1, 2, 4, 7, 16]  # query rows of a KV head: one product for four, eight, or sixteen rows


@pytest.mark.parametrize("T,Hkv", [(512, 2), (2000, 3), (40000, 1)])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("rows", ROWS)
def test_large_scales_of_keys_that_are_not_attended_to(nn, rows, D, T, Hkv):
    """The first block's keys, and a block in the middle, score 42 nats below the others,
    under V scales up to 2^40 times theirs."""
    g = np.random.default_rng(rows + D + T)
    for block in (16, 64):
        n = -(-T // block)
        far = np.zeros(n, bool)
        far[[0, n // 2]] = True
        level = np.where(np.repeat(far, block)[:T], -127, 1) + g.integers(-1, 2, (Hkv, T)) * (1 - np.repeat(far, block)[:T])
        kc, q = keys(g, Hkv, T, D, level), queries(g, rows * Hkv, D)
        ks = np.full((Hkv, n), 0.125, np.float32)
        scale = 42 / (0.125 * 8 * 128)
        vc = g.integers(-127, 128, (Hkv, T, D)).astype(np.int8)
        for ratio in (1.0, 1e2, 1e4, 2.0 ** 40):
            vs = (g.uniform(0.5, 1, (Hkv, n)) * np.where(far, ratio, 1) / 127).astype(np.float32)
            check(nn, q, kc, vc, ks, vs, block, scale, rows, f"ratio {ratio} block {block}")


@pytest.mark.parametrize("T", [64, 500, 20000])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("rows", ROWS)
def test_a_key_that_takes_the_softmax_and_adds_nothing(nn, rows, D, T):
    """One key of V = 0 whose score stands 16 to 60 nats above all others: the others
    alone make the output, whatever tile they share with it."""
    g = np.random.default_rng(rows + D + T)
    block, n = 16, -(-T // 16)
    ks = np.full((1, n), 0.125, np.float32)
    for at in (0, 37):
        level = np.full((1, T), -120)
        level[0] += g.integers(-1, 2, T)
        level[0, at] = 0
        kc, q = keys(g, 1, T, D, level), queries(g, rows, D)
        kc[0, at] = 0
        vc = g.integers(-127, 128, (1, T, D)).astype(np.int8)
        vc[0, at] = 0
        vs = (g.uniform(0.5, 1, (1, n)) / 127).astype(np.float32)
        for gap in (16, 18.3, 25, 40, 60):
            check(nn, q, kc, vc, ks, vs, block, gap / 120.0, rows, f"gap {gap} at {at}")


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("rows", ROWS)
def test_columns_that_only_small_contributions_reach(nn, rows, D):
    """Columns of V in which the keys of large p, or of large scales, are 0: three sizes of
    contribution in every tile, down to 2^-60 of the largest."""
    g = np.random.default_rng(rows * D)
    T, block = 700, 16
    n = -(-T // block)
    kind = np.arange(T) % 3
    level = np.array([0, -40, -80])[kind][None] + g.integers(-1, 2, (1, T))
    kc, q = keys(g, 1, T, D, level), queries(g, rows, D)
    ks = np.full((1, n), 0.125, np.float32)
    vc = g.integers(-127, 128, (1, T, D)).astype(np.int8)
    for c in range(D):
        vc[0, kind < c % 3, c] = 0
    for gap in (4, 12, 20):  # nats between the kinds
        for ratio in (1.0, 1e6):
            vs = (g.uniform(0.5, 1, (1, n)) * np.where(np.arange(n) % 2, ratio, 1) / 127).astype(np.float32)
            check(nn, q, kc, vc, ks, vs, block, gap / 40.0, rows, f"gap {gap} ratio {ratio}")


@pytest.mark.parametrize("D,g_,Tq", [(128, 1, 3), (64, 2, 2), (128, 2, 4), (64, 5, 3), (256, 2, 3)])
@pytest.mark.parametrize("T", [90, 15000])
def test_several_tokens_over_scores_far_apart(nn, D, g_, Tq, T):
    """Causal queries of ragged sequences, one key of V = 0 far above the others: every
    query by itself, over the keys that it sees."""
    g = np.random.default_rng(D + Tq + T)
    lengths, block, Hkv = [T, 41, Tq - 1, 0], 16, 2
    B, n = len(lengths), -(-T // block)
    level = np.full((B * Hkv, T), -120) + g.integers(-1, 2, (B * Hkv, T))
    level[:, 7] = 0
    level[:, 20:T:33] = -60
    kc = keys(g, B * Hkv, T, D, level).reshape(B, Hkv, T, D)
    vc = g.integers(-127, 128, (B, Hkv, T, D)).astype(np.int8)
    kc[:, :, 7], vc[:, :, 7] = 0, 0
    vc[:, :, 20:T:33, ::2] = 0
    ks = np.full((B, Hkv, n), 0.125, np.float32)
    vs = (g.uniform(0.5, 1, (B, Hkv, n)) / 127).astype(np.float32)
    q = queries(g, B * Tq * Hkv * g_, D).reshape(B, Tq, Hkv * g_, D)
    dev = [torch.from_numpy(a).cuda() for a in (q, kc, vc, ks, vs)]
    for gap in (10, 22, 50):
        out = torch.full(q.shape, float("nan"), device="cuda")
        nn.attentionDecodeQ8(None, None, *dev, out, block, torch.tensor(lengths, dtype=torch.int32, device="cuda"),
                             gap / 120.0, g_)
        got = out.cpu().numpy().astype(np.float64)
        for b in range(B):
            for i in range(Tq):
                seen = lengths[b] - Tq + 1 + i
                if seen <= 0:
                    assert not got[b, i].any()
                    continue
                want, tol, _, _ = attend(q[b, i], kc[b, :, :seen], vc[b, :, :seen], ks[b], vs[b], block, gap / 120.0, g_)
                off = np.abs(got[b, i] - want)
                assert (off <= np.maximum(tol, 1e-300)).all(), (gap, b, i, (off / np.maximum(tol, 1e-300)).max())
