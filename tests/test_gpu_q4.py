"""linearQ4 and packWeightQ4 against plain implementations in 64 bits, and the
operators on compressed data together as one decode step."""
import math

import numpy as np
import pytest
import torch

from tests import q_reference as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def nn():
    from tests.helpers import build_library
    build_library()
    from alpakann_b200.onHost import nn
    return nn


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def make_weight(g, K, N, group):
    u = g.integers(0, 16, (K, N))
    s = (g.uniform(0.5, 1.5, (-(-K // group), N)) * 0.2 / math.sqrt(K)).astype(np.float32)
    return u, s


def run_linear(nn, M, K, N, group, bias=False, act="none", residual=False, seed=0, size=1.0):
    g = np.random.default_rng(seed)
    u, s = make_weight(g, K, N, group)
    x = (g.standard_normal((M, K)) * size).astype(np.float32)
    b = g.standard_normal(N).astype(np.float32) if bias else None
    r = g.standard_normal((M, N)).astype(np.float32) if residual else None
    y = torch.full((M, N), float("nan"), device="cuda")
    args = (dev(x), dev(ref.pack_words(u)), dev(s), y, group, None if b is None else dev(b), nn.Activation[act],
            None if r is None else dev(r))
    nn.linearQ4(None, None, *args)
    want, tol = ref.linear(x, u, s, group, b, act, r)
    ref.assert_within(y.cpu().numpy(), want, tol, f"linear {M}x{K}x{N}")
    return args


@pytest.mark.parametrize("M", [1, 2, 3, 4, 5, 8, 9, 16, 17, 40])
def test_linear_rows(nn, M):
    run_linear(nn, M, 512, 192, 64)


@pytest.mark.parametrize("K,group", [(8, 32), (32, 32), (40, 32), (64, 128), (136, 64), (1000, 128), (4096, 4096),
                                     (5000, 96), (16384, 128)])
@pytest.mark.parametrize("N", [1, 3, 33, 64, 130])
def test_linear_sizes(nn, K, group, N):
    run_linear(nn, 2, K, N, group)


@pytest.mark.parametrize("N", [4096, 1028, 20001])
@pytest.mark.parametrize("M", [1, 6])
def test_linear_wide(nn, M, N):
    run_linear(nn, M, 1024, N, 128, bias=True)


@pytest.mark.parametrize("act", ["none", "relu", "silu", "gelu"])
@pytest.mark.parametrize("bias,residual", [(False, False), (True, False), (False, True), (True, True)])
def test_linear_epilogue(nn, act, bias, residual):
    run_linear(nn, 3, 256, 100, 32, bias, act, residual)


@pytest.mark.parametrize("size", [1e-30, 1e-6, 1e5, 1e30])
def test_linear_input_ranges(nn, size):
    run_linear(nn, 2, 256, 64, 32, size=size)


def test_linear_rows_of_different_size(nn):
    """A row, and within it a stretch, of far larger values costs the others nothing."""
    g = np.random.default_rng(2)
    u, s = make_weight(g, 512, 64, 64)
    x = g.standard_normal((4, 512)).astype(np.float32)
    x[1] *= 1e12
    x[2, 100:200] *= 1e6
    x[3] = 0
    y = torch.empty((4, 64), device="cuda")
    nn.linearQ4(None, None, dev(x), dev(ref.pack_words(u)), dev(s), y, 64)
    want, tol = ref.linear(x, u, s, 64)
    ref.assert_within(y.cpu().numpy(), want, tol)
    assert not y[3].any()


def test_linear_in_place_residual_and_strides(nn):
    g = np.random.default_rng(3)
    M, K, N, group = 3, 320, 70, 64
    u, s = make_weight(g, K, N, group)
    xs = torch.from_numpy(g.standard_normal((M, 2 * K)).astype(np.float32)).cuda()[:, ::2]
    ps = torch.zeros((K // 8, N + 5), dtype=torch.int32, device="cuda")[:, 2:N + 2]
    ps.copy_(torch.from_numpy(ref.pack_words(u)))
    ss = dev(s.T).t()
    y = torch.zeros((M, 3 * N), device="cuda")[:, N:2 * N]
    r = g.standard_normal((M, N)).astype(np.float32)
    y.copy_(torch.from_numpy(r))
    b = g.standard_normal(N).astype(np.float32)
    nn.linearQ4(None, None, xs, ps, ss, y, group, dev(np.repeat(b, 2))[::2], nn.Activation.relu, y)
    want, tol = ref.linear(xs.cpu().numpy(), u, s, group, b, "relu", r)
    ref.assert_within(y.cpu().numpy(), want, tol)
    # one row for every output row (a broadcast input)
    one = dev(xs.cpu().numpy()[:1]).expand(M, K)
    nn.linearQ4(None, None, one, ps, ss, y, group)
    assert torch.equal(y[0], y[1]) and torch.equal(y[0], y[2])


def test_linear_non_finite(nn):
    """An infinite or NaN input reaches its own row only; a NaN scale its own column."""
    args = run_linear(nn, 3, 256, 64, 64)
    x, p, s, y = args[0].clone(), args[1], args[2].clone(), args[3]
    good = y.clone()
    x[1, 5] = float("nan")
    out = torch.empty_like(y)
    nn.linearQ4(None, None, x, p, s, out, 64)
    assert torch.isnan(out[1]).all() and torch.equal(out[[0, 2]], good[[0, 2]])
    x[1, 5] = float("inf")
    nn.linearQ4(None, None, x, p, s, out, 64)
    assert not torch.isfinite(out[1]).any() and torch.equal(out[[0, 2]], good[[0, 2]])
    s[2, 10] = float("nan")
    nn.linearQ4(None, None, args[0], p, s, out, 64)
    assert torch.isnan(out[:, 10]).all()
    keep = torch.arange(64) != 10
    assert torch.equal(out[:, keep], good[:, keep])


def test_linear_repeats_and_replays(nn):
    args = run_linear(nn, 5, 4096, 512, 128, bias=True, act="silu")
    want = args[3].clone()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [torch.empty_like(want) for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(3):
        for st, o in zip(streams, outs):
            nn.linearQ4(st, None, *args[:3], o, *args[4:])
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        nn.linearQ4(None, None, *args[:3], outs[0], *args[4:])
    args[0].mul_(-1.5)
    graph.replay()
    nn.linearQ4(None, None, *args[:3], outs[1], *args[4:])
    torch.cuda.synchronize()
    assert torch.equal(outs[0], outs[1]) and not torch.equal(outs[0], want)


# ---- packing ------------------------------------------------------------------
@pytest.mark.parametrize("K,N,group", [(8, 1, 32), (64, 40, 32), (136, 129, 64), (4096, 300, 128)])
def test_pack(nn, K, N, group):
    g = np.random.default_rng(K)
    w = g.standard_normal((K, N)).astype(np.float32)
    w[:, 0] = 0
    if N > 4:
        w[3, 1], w[4, 2] = np.nan, np.inf
        top = np.float32(0.7)
        w[:, 3] = (np.float64(np.float32(top / np.float32(7))) * (np.arange(K) % 13 - 6 + 0.5)).astype(np.float32)
        w[::8, 3] = top
    p = torch.zeros((K // 8, N), dtype=torch.int32, device="cuda")
    s = torch.zeros((-(-K // group), N), device="cuda")
    nn.packWeightQ4(None, None, dev(w), p, s, group)
    u, sc = ref.quantise_weight(w, group)
    np.testing.assert_array_equal(s.cpu().numpy(), sc)
    np.testing.assert_array_equal(p.cpu().numpy(), ref.pack_words(u))
    # a transposed (column-major) weight packs alike
    p2, s2 = torch.zeros_like(p), torch.zeros_like(s)
    nn.packWeightQ4(None, None, dev(w.T).t(), p2, s2, group)
    assert torch.equal(p2, p) and torch.equal(s2.nan_to_num(7.0), s.nan_to_num(7.0))


# ---- together -------------------------------------------------------------------
def test_decode_step(nn):
    """One layer's decode step on compressed data, twice, captured and replayed:
    rmsNorm, 4-bit projections, rotary, append, attention, output projection onto
    the residual, MLP layer. Against the same step in 64 bits on the same integers.
    The bound grows along the step: each stage passes on its own bound and at most
    the operand's error times the sums of |W| (linear) or the softmax's slope; the
    measured size of that product stays under 2^-14 of each output's largest value
    (13 bits over float32's own 2^-24 for seven chained sums of up to 512 terms)."""
    g = np.random.default_rng(11)
    B, Hq, Hkv, D, T, block, group = 3, 8, 2, 64, 100, 16, 64
    dm, F = Hq * D, 768
    wq, wk, wv, wo, w1 = (make_weight(g, k, n, group) for k, n in ((dm, Hq * D), (dm, Hkv * D), (dm, Hkv * D),
                                                                  (Hq * D, dm), (dm, F)))
    packed = [(dev(ref.pack_words(u)), dev(s)) for u, s in (wq, wk, wv, wo, w1)]
    norm = (1 + 0.1 * g.standard_normal(dm)).astype(np.float32)
    lengths = np.array([40, 7, 0], np.int32)
    kc, ks = ref.make_cache(g, B, Hkv, T, D, block)
    vc, vs = ref.make_cache(g, B, Hkv, T, D, block)
    dkc, dks, dvc, dvs = dev(kc), dev(ks), dev(vc), dev(vs)
    freq = 1e4 ** (-np.arange(D // 4) / (D // 4))
    h = torch.empty((B, dm), device="cuda")
    dn, dpos, dlen, df = dev(norm), dev(lengths), dev(lengths + 1), dev(freq)
    x, a = torch.empty((B, dm), device="cuda"), torch.empty((B, 1, Hq, D), device="cuda")
    q, k, v = (torch.empty((B, 1, n, D), device="cuda") for n in (Hq, Hkv, Hkv))
    up = torch.empty((B, F), device="cuda")

    def step():
        nn.rmsNorm(None, None, h, dn, x, 1e-6)
        for t, (p, s) in zip((q, k, v), packed):
            nn.linearQ4(None, None, x, p, s, t.view(B, -1), group)
        nn.rotary(None, None, q, k, dpos.view(B, 1), df, q, k, nn.RotaryPairs.halves)
        nn.kvCacheAppendQ8(None, None, k, v, dkc, dvc, dks, dvs, dpos, block)
        nn.attentionDecodeQ8(None, None, q, dkc, dvc, dks, dvs, a, block, dlen, None, Hq // Hkv)
        nn.linearQ4(None, None, a.view(B, -1), *packed[3], h, group, residual=h)
        nn.linearQ4(None, None, h, *packed[4], up, group, None, nn.Activation.silu)
        dpos.add_(1)
        dlen.add_(1)

    hs = [g.standard_normal((B, dm)).astype(np.float32) for _ in range(3)]
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    for n, h0 in enumerate(hs):
        h.copy_(torch.from_numpy(h0))
        torch.cuda.synchronize()
        if n == 0:
            step()
        else:
            if n == 1:
                with torch.cuda.graph(graph, stream=stream):
                    step()
            graph.replay()
        torch.cuda.synchronize()
        # the same step in 64 bits; the cache's integers are the device's own, held to the reference's below
        x64 = h0 * (1 / np.sqrt((h0.astype(np.float64) ** 2).mean(-1, keepdims=True) + 1e-6)) * norm
        rows = [ref.linear(x64, u, s, group)[0] for u, s in (wq, wk, wv)]
        pos = (lengths + n)[:, None]
        q64 = ref.rotary(rows[0].reshape(B, 1, Hq, D), pos, freq, True)
        k64 = ref.rotary(rows[1].reshape(B, 1, Hkv, D), pos, freq, True)
        for c, s, r in ((dkc, dks, k64), (dvc, dvs, rows[2].reshape(B, 1, Hkv, D))):
            c, s = c.cpu().numpy(), s.cpu().numpy()
            for b in range(B):
                t = lengths[b] + n
                step_ = s[b, :, t // block][:, None]
                assert (np.abs(c[b, :, t] * step_ - r[b, 0]) <= 0.501 * step_).all()
        a64, _ = ref.attend(q64, *(t.cpu().numpy() for t in (dkc, dvc, dks, dvs)), lengths + n + 1, block,
                            1 / math.sqrt(D), Hq // Hkv)
        h64 = ref.linear(a64.reshape(B, -1), *wo, group)[0] + h0
        up64 = ref.linear(h64, *w1, group, act="silu")[0]
        for got, want in ((a, a64), (h, h64), (up, up64)):
            assert np.abs(got.cpu().numpy() - want).max() <= 2.0 ** -14 * np.abs(want).max()
