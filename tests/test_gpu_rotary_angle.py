"""rotary's angles in float32: as good as cosine and sine taken in 64 bits."""
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


@pytest.mark.parametrize("first", [0, 100000, 2**30])
@pytest.mark.parametrize("halves", [False, True])
def test_error_beside_64_bit_angles(nn, halves, first):
    """Plain form: cosine and sine in 64 bits, rounded, two products and a sum in float32:
    half a step each. The kernel rounds the angle, within an eighth of a turn of a whole
    quarter, to 2^-28 turns (0.4 u, root mean square 0.2 u), its functions are good to one
    unit, and it saves one rounding: at most 1.2 times the plain form's root mean square."""
    g = np.random.default_rng(first % 97)
    T, H, D = 512, 4, 128
    x = g.standard_normal((1, T, H, D)).astype(np.float32)
    pos = (first + np.arange(T)).astype(np.int32)[None]
    f = 1e4 ** (-np.arange(D // 2) / (D // 2))
    want = ref.rotary(x, pos, f, halves)
    a = pos.astype(np.float64)[..., None] * f
    c, s = (fn(a).astype(np.float32)[:, :, None] for fn in (np.cos, np.sin))
    i0, i1 = (slice(0, D // 2), slice(D // 2, D)) if halves else (slice(0, D, 2), slice(1, D, 2))
    plain = x.copy()
    plain[..., i0], plain[..., i1] = x[..., i0] * c - x[..., i1] * s, x[..., i0] * s + x[..., i1] * c
    out = torch.empty(x.shape, device="cuda")
    nn.rotary(None, None, torch.from_numpy(x).cuda(), None, torch.from_numpy(pos).cuda(), torch.from_numpy(f).cuda(), out,
              None, nn.RotaryPairs.halves if halves else nn.RotaryPairs.interleaved)
    rms = lambda e: float(np.sqrt((e ** 2).mean()))
    off, base = rms(out.cpu().numpy().astype(np.float64) - want), rms(plain.astype(np.float64) - want)
    assert off <= 1.2 * base, (off, base)


def test_whole_and_half_quarters(nn):
    """Positions that turn by multiples of an eighth of a turn, both ways: every quarter, its
    borders, and inverse back to the input."""
    T, D = 64, 8
    pos = np.arange(-32, 32).astype(np.int32)
    f = np.array([np.pi / 4, np.pi / 2, np.pi, 2 * np.pi])
    x = np.random.default_rng(3).standard_normal((1, T, 2, D)).astype(np.float32)
    dev = [torch.from_numpy(t).cuda() for t in (x, pos, f)]
    out, back = torch.empty(x.shape, device="cuda"), torch.empty(x.shape, device="cuda")
    nn.rotary(None, None, dev[0], None, dev[1], dev[2], out, None)
    nn.rotary(None, None, out, None, dev[1], dev[2], back, None, inverse=True)
    want = ref.rotary(x, pos[None], f, False)
    tol = ref.rotary_bound(x, f, False, 1.0, 2.0 ** -21)
    ref.assert_within(out.cpu().numpy(), want, tol)
    ref.assert_within(back.cpu().numpy(), x.astype(np.float64), 3 * tol)
