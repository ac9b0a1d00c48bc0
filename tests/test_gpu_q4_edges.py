"""linearQ4 at the ends of its range, and with bounds that see the loss of low bits."""
import math

import numpy as np
import pytest
import torch

from tests import q_reference as ref

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


@pytest.fixture(scope="module")
def nn():
    from tests.helpers import build_library
    build_library()
    from alpakann_b200.onHost import nn
    return nn


def run(nn, x, u, s, group):
    dev = [torch.from_numpy(np.ascontiguousarray(a)).cuda() for a in (x, ref.pack_words(u), s)]
    y = torch.full((x.shape[0], u.shape[1]), float("nan"), device="cuda")
    nn.linearQ4(None, None, *dev, y, group)
    return y.cpu().numpy().astype(np.float64)


@pytest.mark.parametrize("M", [1, 3, 8])
@pytest.mark.parametrize("xs,ss", [(0, 90), (0, 100), (-40, 107), (60, 50), (-90, 60), (100, -110), (126, -125)])
def test_far_sizes(nn, M, xs, ss):
    """Inputs of 2^xs and scales of 2^ss: neither the sums of digits nor their join overflow
    while the scales stay below 2^114 / K, nor does anything underflow that the result holds."""
    g = np.random.default_rng(M)
    K, N, group = 64, 96, 32
    x = (np.ldexp(g.uniform(0.5, 1, (M, K)), xs) * g.choice([-1, 1], (M, K))).astype(np.float32)
    s = np.ldexp(g.uniform(0.5, 1, (K // group, N)), ss).astype(np.float32)
    u = g.integers(0, 16, (K, N))
    want, tol = ref.linear(x, u, s, group)
    ref.assert_within(run(nn, x, u, s, group), want, tol, f"2^{xs} 2^{ss}")


@pytest.mark.parametrize("M,K,N", [(1, 4096, 512), (2, 16384, 256), (8, 4096, 512), (5, 16384, 64)])
def test_error_of_the_whole(nn, M, K, N):
    """The root mean square error over all outputs, to which roundings of either sign add as
    a random walk: at most four times that of numpy's float32 product, whose sums are of
    the same length, and 4 u of the outputs' own root mean square (a rounding each of the
    result, the scale's product and two joins)."""
    g = np.random.default_rng(K)
    group = 128
    x = g.standard_normal((M, K)).astype(np.float32)
    s = (g.uniform(0.5, 1.5, (K // group, N)) * 0.2 / math.sqrt(K)).astype(np.float32)
    u = g.integers(0, 16, (K, N))
    w = (u - 8).astype(np.float32) * np.repeat(s, group, 0)
    want = x.astype(np.float64) @ ((u - 8) * np.repeat(s.astype(np.float64), group, 0))
    rms = lambda e: float(np.sqrt((e ** 2).mean()))
    off, plain = rms(run(nn, x, u, s, group) - want), rms((x @ w).astype(np.float64) - want)
    assert off <= 4 * plain + 4 * U * rms(want), (off / rms(want), plain / rms(want))


@pytest.mark.parametrize("M", [1, 4, 8])
def test_small_inputs_beside_large_ones(nn, M):
    """A stretch of inputs 10^5 times the others whose weights are zero in half of the
    columns: there the others alone make the result, each off by the 2^-31 of the row's
    largest that the definition allows, and by the sums' own roundings."""
    g = np.random.default_rng(M)
    K, N, group = 1024, 128, 64
    x = g.standard_normal((M, K)).astype(np.float32)
    x[:, 128:192] *= 1e5
    u = g.integers(0, 16, (K, N))
    u[128:192, ::2] = 8
    s = (g.uniform(0.5, 1.5, (K // group, N)) / math.sqrt(K)).astype(np.float32)
    w = (u - 8).astype(np.float64) * np.repeat(s.astype(np.float64), group, 0)
    want, size = x.astype(np.float64) @ w, np.abs(x).astype(np.float64) @ np.abs(w)
    tol = 2 * (K + 16) * U * size + 2.0 ** -31 * np.abs(x).max(1, keepdims=True) * np.abs(w).sum(0)
    ref.assert_within(run(nn, x, u, s, group), want, tol, "mixed sizes")


def test_infinite_and_nan_scales_reach_their_columns_only(nn):
    g = np.random.default_rng(1)
    K, N, group = 256, 64, 64
    x, u = g.standard_normal((3, K)).astype(np.float32), g.integers(0, 16, (K, N))
    s = g.uniform(0.5, 1.5, (K // group, N)).astype(np.float32)
    want, tol = ref.linear(x, u, s, group)
    s[1, 5], s[3, 17], s[0, 40] = np.inf, np.nan, -np.inf
    y, bad = run(nn, x, u, s, group), [5, 17, 40]
    assert not np.isfinite(y[:, bad]).any()
    keep = np.setdiff1d(np.arange(N), bad)
    ref.assert_within(y[:, keep], want[:, keep], tol[:, keep], "other columns")
