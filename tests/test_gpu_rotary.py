"""rotary and rotaryFrequencies against the formula in 64 bits."""
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


def frequencies(p, base=1e4):
    return base ** (-np.arange(p) / p) if p else np.zeros(0)


# Rounding of an fp32 pair: the angle is reduced to turns in 64 bits and rounded
# to 2^-26 of a turn (2 pi 2^-26 = 1.6 u), sincospi is good to 2 units of 2 u,
# the magnitude, the products and the sum add 4 u: under 8 u = 2^-21 of |x0| +
# |x1|. In fp64 the angle is the 64-bit product itself, sincos good to 2 units,
# and 4 more roundings: under 2^-50.
EPS = {np.float32: 2.0 ** -21, np.float64: 2.0 ** -50}


@pytest.mark.parametrize("T", [np.float32, np.float64])
@pytest.mark.parametrize("halves", [False, True])
@pytest.mark.parametrize("B,t,hq,hk,D,P", [
    (1, 1, 1, 1, 2, 1), (2, 3, 4, 2, 64, 32), (1, 5, 3, 3, 80, 10), (3, 1, 9, 1, 128, 32), (2, 7, 5, 2, 6, 3),
    (1, 2, 2, 1, 128, 0), (1, 33, 8, 8, 96, 48), (2, 130, 17, 3, 256, 128), (1, 4, 2, 2, 24, 4)])
def test_rotary_matches_formula(nn, T, halves, B, t, hq, hk, D, P):
    g = np.random.default_rng(B + t + D)
    q, k = (g.standard_normal((B, t, h, D)).astype(T) for h in (hq, hk))
    pos = g.integers(0, 200000, (B, t)).astype(np.int32)
    f = frequencies(P)
    dq, dk, dp, df = (torch.from_numpy(a).cuda() for a in (q, k, pos, f))
    oq, ok = torch.full_like(dq, float("nan")), torch.full_like(dk, float("nan"))
    nn.rotary(None, None, dq, dk, dp, df, oq, ok, nn.RotaryPairs(int(halves)), magnitude=1.25)
    for x, o in ((q, oq), (k, ok)):
        want = ref.rotary(x, pos, f, halves, 1.25)
        ref.assert_within(o.cpu().numpy(), want, ref.rotary_bound(x, f, halves, 1.25, EPS[T]), "rotary")
        assert np.array_equal(o.cpu().numpy()[..., 2 * P:], x[..., 2 * P:])  # the rest of the head is copied
    # in place, and each tensor alone: the same bits
    nn.rotary(None, None, dq, dk, dp, df, dq, dk, nn.RotaryPairs(int(halves)), magnitude=1.25)
    assert torch.equal(dq, oq) and torch.equal(dk, ok)
    o1 = torch.empty_like(dk)
    nn.rotary(None, None, torch.from_numpy(k).cuda(), None, dp, df, o1, None, nn.RotaryPairs(int(halves)),
              magnitude=1.25)
    assert torch.equal(o1, ok)


@pytest.mark.parametrize("halves", [False, True])
def test_layouts_strides_and_positions(nn, halves):
    """A fused projection's slices, BHTD, one row of positions for every sequence, negative positions."""
    g = np.random.default_rng(3)
    B, t, hq, hk, D = 3, 6, 4, 2, 64
    f = frequencies(32)
    df = torch.from_numpy(f).cuda()
    fused = torch.from_numpy(g.standard_normal((B, t, hq + 2 * hk, D)).astype(np.float32)).cuda()
    q, k = fused[:, :, :hq], fused[:, :, hq:hq + hk]
    row = np.array([-5, 0, 1, 77777, 3, -100000], np.int32)
    want_q = ref.rotary(q.cpu().numpy(), np.tile(row, (B, 1)), f, halves)
    bound = ref.rotary_bound(q.cpu().numpy(), f, halves, 1.0, EPS[np.float32])
    kept = fused[:, :, hq + hk:].clone()
    pairs = nn.RotaryPairs(int(halves))
    nn.rotary(None, None, q, k, torch.from_numpy(row).cuda(), df, q, k, pairs)
    ref.assert_within(q.cpu().numpy(), want_q, bound, "slice of a fused projection")
    assert torch.equal(fused[:, :, hq + hk:], kept)
    # BHTD views of BTHD memory, with element strides that rule out vectors
    x = torch.from_numpy(g.standard_normal((B, t, hq, 2 * D)).astype(np.float32)).cuda()[..., ::2]
    o = torch.zeros((B, hq, t, D + 1), device="cuda")[..., 1:]
    pos = torch.from_numpy(np.tile(row, (B, 1))).cuda().t().contiguous().t()
    nn.rotary(None, None, x.transpose(1, 2), None, pos, df, o, None, pairs, layout=1)
    xn = np.ascontiguousarray(x.cpu().numpy())
    ref.assert_within(o.transpose(1, 2).cpu().numpy(), ref.rotary(xn, np.tile(row, (B, 1)), f, halves),
                      ref.rotary_bound(xn, f, halves, 1.0, EPS[np.float32]), "strided BHTD")


@pytest.mark.parametrize("halves", [False, True])
def test_inverse_is_the_gradient(nn, halves):
    """inverse=True against autograd of the formula, and against differences, in fp64."""
    g = torch.Generator().manual_seed(1)
    B, t, h, D, P = 2, 3, 2, 24, 8
    x = torch.randn((B, t, h, D), generator=g, dtype=torch.float64)
    w = torch.randn((B, t, h, D), generator=g, dtype=torch.float64)
    pos = torch.randint(0, 5000, (B, t), generator=g, dtype=torch.int32)
    f = torch.from_numpy(frequencies(P))
    pairs = nn.RotaryPairs(int(halves))

    def turn(v, inverse=False):
        o = torch.empty_like(v, device="cuda")
        nn.rotary(None, None, v.cuda(), None, pos.cuda(), f.cuda(), o, None, pairs, magnitude=0.75, inverse=inverse)
        return o.cpu()

    grad = turn(w, inverse=True)
    a = (pos.double()[..., None] * f)[:, :, None]
    y = x.clone().requires_grad_()
    i0, i1 = (slice(0, P), slice(P, 2 * P)) if halves else (slice(0, 2 * P, 2), slice(1, 2 * P, 2))
    loss = (0.75 * ((y[..., i0] * a.cos() - y[..., i1] * a.sin()) * w[..., i0] +
                    (y[..., i0] * a.sin() + y[..., i1] * a.cos()) * w[..., i1])).sum() + \
        (y[..., 2 * P:] * w[..., 2 * P:]).sum()
    loss.backward()
    bound = ref.rotary_bound(w.numpy(), f.numpy(), halves, 1.0, 2.0 ** -49)
    ref.assert_within(grad.numpy(), y.grad.numpy(), bound + 0, "gradient")
    # the map is linear: a difference quotient is exact up to its roundings
    step = torch.randn((B, t, h, D), generator=g, dtype=torch.float64)
    diff = ((turn(x + step) - turn(x - step)) * w).sum() / 2
    size = (w.abs() * 4 * (x.abs() + step.abs())).sum().item()
    assert abs(diff.item() - (grad * step).sum().item()) <= 2.0 ** -44 * size


def test_frequencies(nn):
    """Plain, divided and by parts, against the formula: powers good to 2 units, three more roundings."""
    P = 64
    f = torch.empty(P, dtype=torch.float64, device="cuda")
    base = 5e5 ** (-np.arange(P) / P)
    nn.rotaryFrequencies(None, None, f, 5e5)
    np.testing.assert_allclose(f.cpu().numpy(), base, rtol=2.0 ** -48)
    nn.rotaryFrequencies(None, None, f, 5e5, 4.0)
    np.testing.assert_allclose(f.cpu().numpy(), base / 4, rtol=2.0 ** -48)
    nn.rotaryFrequencies(None, None, f, 5e5, 8.0, 4096, 1.0, 32.0)
    r = 4096 * base / (2 * np.pi)
    w = np.clip((r - 1) / 31, 0, 1)
    assert (w == 0).any() and (w == 1).any() and ((w > 0) & (w < 1)).any()
    np.testing.assert_allclose(f.cpu().numpy(), base * (w + (1 - w) / 8), rtol=2.0 ** -44)
    strided = torch.zeros(2 * P, dtype=torch.float64, device="cuda")
    nn.rotaryFrequencies(None, None, strided[::2], 5e5)
    np.testing.assert_allclose(strided[::2].cpu().numpy(), base, rtol=2.0 ** -48)
    assert not strided[1::2].any()


def test_non_finite_stays_in_its_pair(nn):
    x = torch.zeros((1, 1, 1, 16), device="cuda")
    x[0, 0, 0, 2] = float("nan")
    x[0, 0, 0, 9] = float("inf")
    o = torch.empty_like(x)
    nn.rotary(None, None, x, None, torch.ones(1, dtype=torch.int32, device="cuda"),
              torch.from_numpy(frequencies(8)).cuda(), o, None)
    bad = ~torch.isfinite(o[0, 0, 0])
    assert bad.nonzero().flatten().tolist() == [2, 3, 8, 9]
