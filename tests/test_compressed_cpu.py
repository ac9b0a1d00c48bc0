"""Refusals of the operators on compressed data (rotary, 8-bit KV cache, 4-bit
weights): every call here fails on the host before anything is enqueued."""
import numpy as np
import pytest
import torch

from tests import q_reference as ref


@pytest.fixture(scope="module")
def capi():
    from tests.helpers import build_library
    build_library()
    from alpakann_b200 import _capi
    return _capi


def refused(capi, name, *args, code=None):
    rc = getattr(capi.lib, name)(None, *args)
    assert rc == (capi.ANN_EINVAL if code is None else code), (rc, capi.lib.ann_last_error())
    return capi.lib.ann_last_error().decode()


@pytest.mark.parametrize("sfx,T", [("f32", np.float32), ("f64", np.float64)])
def test_rotary_refusals(capi, sfx, T):
    r = capi.ref
    q, k = np.zeros((2, 3, 4, 8), T), np.zeros((2, 3, 2, 8), T)
    pos, f = np.zeros((2, 3), np.int32), np.zeros(4, np.float64)

    def call(q=q, k=k, pos=pos, f=f, oq=q, ok=k, pairs=0, layout=0):
        return refused(capi, f"ann_rotary_{sfx}", r(q), None if k is None else r(k), r(pos), r(f), r(oq),
                       None if ok is None else r(ok), pairs, layout, 1.0, 0)

    assert "come together" in call(k=None)
    assert "come together" in call(ok=None)
    assert "pairs" in call(pairs=2)
    assert "layout" in call(layout=2)
    assert "same extents" in call(oq=np.zeros((2, 3, 4, 6), T))
    assert "same extents" in call(q=np.zeros((3, 4, 8), T), oq=np.zeros((3, 4, 8), T), k=None, ok=None)
    assert "differ" in call(k=np.zeros((2, 4, 2, 8), T), ok=np.zeros((2, 4, 2, 8), T))
    assert "positions" in call(pos=np.zeros((3, 2), np.int32))
    assert "positions" in call(pos=np.zeros(2, np.int32))
    assert "frequencies" in call(f=np.zeros(5, np.float64))
    assert "frequencies" in call(f=np.zeros((2, 2), np.float64))
    odd = np.zeros((2, 3, 4, 7), T)
    assert "even" in call(q=odd, oq=odd, k=None, ok=None, f=np.zeros(2, np.float64))
    assert "zero pitch" in call(oq=np.broadcast_to(np.zeros((1, 3, 4, 8), T), (2, 3, 4, 8)))
    # BHTD: tokens are axis 2
    assert "positions" in call(k=None, ok=None, layout=1)


def test_rotary_frequencies_refusals(capi):
    f = capi.ref(np.zeros(8, np.float64))
    for args in [(0.0, 1.0, 0.0, 1.0, 32.0), (-1.0, 1.0, 0.0, 1.0, 32.0), (1e4, 0.0, 0.0, 1.0, 32.0),
                 (np.inf, 1.0, 0.0, 1.0, 32.0), (1e4, np.nan, 0.0, 1.0, 32.0)]:
        assert "positive and finite" in refused(capi, "ann_rotary_frequencies", f, *args)
    assert "trained length" in refused(capi, "ann_rotary_frequencies", f, 1e4, 2.0, -1.0, 1.0, 32.0)
    assert "lowTurns" in refused(capi, "ann_rotary_frequencies", f, 1e4, 2.0, 4096.0, 32.0, 32.0)
    assert "lowTurns" in refused(capi, "ann_rotary_frequencies", f, 1e4, 2.0, 4096.0, 1.0, np.nan)
    assert "rank-1" in refused(capi, "ann_rotary_frequencies", capi.ref(np.zeros((2, 4))), 1e4, 1.0, 0.0, 1.0, 32.0)


def cache_args(B=2, H=3, T=40, D=64, block=16):
    return (np.zeros((B, H, T, D), np.int8), np.zeros((B, H, T, D), np.int8),
            np.zeros((B, H, -(-T // block)), np.float32), np.zeros((B, H, -(-T // block)), np.float32))


def test_append_refusals(capi):
    r = capi.ref
    kc, vc, ks, vs = cache_args()
    x, pos = np.zeros((2, 5, 3, 64), np.float32), np.zeros(2, np.int32)

    def call(kn=x, vn=x, kc=kc, vc=vc, ks=ks, vs=vs, pos=pos, counts=None, block=16, layout=1):
        return refused(capi, "ann_kv_cache_append_q8_f32", r(kn), r(vn), r(kc), r(vc), r(ks), r(vs), r(pos),
                       None if counts is None else r(counts), block, layout)

    assert "tokensPerScale" in call(block=0)
    assert "layout" in call(layout=7)
    assert "scales" in call(block=32)
    assert "scales" in call(layout=0)
    assert "differ" in call(vc=vc[:, :, :39])
    assert "same extents" in call(vn=x[:, :4])
    assert "do not match" in call(kn=x[..., :32], vn=x[..., :32])
    assert "do not match" in call(kn=x[:1], vn=x[:1])
    assert "positions" in call(pos=np.zeros(3, np.int32))
    assert "counts" in call(counts=np.zeros((2, 1), np.int32))
    shared = np.broadcast_to(np.zeros((1, 3, 40, 64), np.int8), (2, 3, 40, 64))
    assert "zero pitch" in call(kc=shared)
    assert "zero pitch" in call(vs=np.broadcast_to(np.zeros((1, 3, 3), np.float32), (2, 3, 3)))


def test_read_refusals(capi):
    r = capi.ref
    kc, vc, ks, vs = cache_args()
    o = np.zeros((2, 3, 40, 64), np.float32)

    def call(ko=o, vo=o, lengths=None, block=16, layout=1):
        return refused(capi, "ann_kv_cache_read_q8_f32", r(kc), r(vc), r(ks), r(vs), r(ko), r(vo),
                       None if lengths is None else r(lengths), block, layout)

    assert "tokensPerScale" in call(block=0)
    assert "output" in call(ko=np.zeros((2, 3, 41, 64), np.float32))
    assert "output" in call(vo=np.zeros((2, 2, 40, 64), np.float32))
    assert "differ" in call(vo=o[:, :, :39])
    assert "lengths" in call(lengths=np.zeros(1, np.int32))
    assert "zero pitch" in call(ko=np.broadcast_to(o[:1], o.shape))


def test_attention_refusals(capi):
    r = capi.ref
    kc, vc, ks, vs = cache_args()
    q = np.zeros((2, 1, 6, 64), np.float32)

    def call(q=q, kc=kc, vc=vc, ks=ks, vs=vs, lengths=None, out=None, g=2, block=16, layout=1, code=None):
        out = np.zeros(q.shape, np.float32) if out is None else out
        return refused(capi, "ann_attention_decode_q8_f32", r(q), r(kc), r(vc), r(ks), r(vs),
                       None if lengths is None else r(lengths), r(out), 0.1, g, block, layout, 1, code=code)

    assert "queriesPerKvGroup" in call(g=0)
    assert "tokensPerScale" in call(block=0)
    assert "layout" in call(layout=2)
    assert "scales" in call(block=8)
    assert "does not match" in call(g=1)  # 6 query heads over 3 KV heads need g >= 2
    assert "does not match" in call(q=np.zeros((3, 1, 6, 64), np.float32))
    assert "extents of Q" in call(out=np.zeros((2, 1, 6, 32), np.float32))
    assert "extents differ" in call(vc=vc[:, :, :39])
    assert "lengths" in call(lengths=np.zeros(3, np.int32))
    assert "zero pitch" in call(out=np.broadcast_to(np.zeros((1, 1, 6, 64), np.float32), (2, 1, 6, 64)))
    no = capi.ANN_ENOTSUP
    kc, vc, ks, vs = cache_args(D=80)
    assert "head dim" in call(q=np.zeros((2, 1, 6, 80), np.float32), kc=kc, vc=vc, ks=ks, vs=vs, code=no)
    kc, vc, ks, vs = cache_args(T=48, block=24)
    assert "power of two" in call(kc=kc, vc=vc, ks=ks, vs=vs, block=24, code=no)
    kc, vc, ks, vs = cache_args(block=8)
    assert "power of two" in call(kc=kc, vc=vc, ks=ks, vs=vs, block=8, code=no)
    wide = np.zeros((2, 3, 40, 72), np.int8)[..., :64]  # rows of 72 bytes
    kc, vc, ks, vs = cache_args()
    assert "aligned" in call(kc=wide, vc=wide, ks=ks, vs=vs, code=no)


def test_linear_refusals(capi):
    r = capi.ref
    x, p, s = np.zeros((2, 64), np.float32), np.zeros((8, 12), np.int32), np.zeros((2, 12), np.float32)
    y = np.zeros((2, 12), np.float32)

    def call(x=x, p=p, s=s, b=None, res=None, y=y, group=32, act=0):
        return refused(capi, "ann_linear_q4_f32", r(x), r(p), r(s), None if b is None else r(b),
                       None if res is None else r(res), r(y), group, act)

    assert "multiple of 32" in call(group=0)
    assert "multiple of 32" in call(group=48)
    assert "scales" in call(group=64)
    assert "shape mismatch" in call(x=np.zeros((2, 56), np.float32))
    assert "shape mismatch" in call(y=np.zeros((3, 12), np.float32))
    assert "activation" in call(act=4)
    assert "bias" in call(b=np.zeros(11, np.float32))
    assert "residual" in call(res=np.zeros((2, 11), np.float32))
    assert "zero pitch" in call(y=np.broadcast_to(np.zeros((1, 12), np.float32), (2, 12)))

    def pack(w, p=p, s=s, group=32):
        return refused(capi, "ann_pack_weight_q4_f32", r(w), r(p), r(s), group)

    assert "does not match" in pack(np.zeros((63, 12), np.float32))
    assert "multiple of 32" in pack(np.zeros((64, 12), np.float32), group=16)
    assert "zero pitch" in pack(np.zeros((64, 12), np.float32), p=np.broadcast_to(p[:1], p.shape))


def test_empty_calls_enqueue_nothing(capi):
    """Extents of zero are valid and need no device."""
    r = capi.ref
    q = np.zeros((2, 0, 4, 8), np.float32)
    assert capi.lib.ann_rotary_f32(None, r(q), None, r(np.zeros((2, 0), np.int32)), r(np.zeros(4)), r(q), None, 0, 0,
                                   1.0, 0) == capi.ANN_OK
    kc, vc, ks, vs = cache_args()
    x = np.zeros((2, 0, 3, 64), np.float32)
    assert capi.lib.ann_kv_cache_append_q8_f32(None, r(x), r(x), r(kc), r(vc), r(ks), r(vs), r(np.zeros(2, np.int32)),
                                               None, 16, 1) == capi.ANN_OK
    q = np.zeros((2, 0, 6, 64), np.float32)
    assert capi.lib.ann_attention_decode_q8_f32(None, r(q), r(kc), r(vc), r(ks), r(vs), None, r(q), 0.1, 2, 16, 1,
                                                1) == capi.ANN_OK
    assert capi.lib.ann_linear_q4_f32(None, r(np.zeros((0, 64), np.float32)), r(np.zeros((8, 12), np.int32)),
                                      r(np.zeros((2, 12), np.float32)), None, None, r(np.zeros((0, 12), np.float32)),
                                      32, 0) == capi.ANN_OK


def test_python_refuses_types_and_host_tensors(capi):
    from alpakann_b200.onHost import nn
    kc, vc, ks, vs = (torch.from_numpy(a) for a in cache_args())
    q = torch.zeros((2, 1, 6, 64))
    with pytest.raises(TypeError):
        nn.attentionDecodeQ8(None, None, q, kc.float(), vc, ks, vs, q, 16)
    with pytest.raises(TypeError):
        nn.attentionDecodeQ8(None, None, q.double(), kc, vc, ks, vs, q.double(), 16)
    with pytest.raises(TypeError):
        nn.attentionDecodeQ8(None, None, q, kc, vc, ks, vs, q, 16, torch.zeros(2, dtype=torch.int64))
    with pytest.raises(ValueError, match="CUDA"):
        nn.attentionDecodeQ8(None, None, q, kc, vc, ks, vs, q, 16)
    with pytest.raises(TypeError):
        nn.rotary(None, None, q, None, torch.zeros((2, 1), dtype=torch.int32), torch.zeros(4), q, None)
    with pytest.raises(TypeError):
        nn.rotary(None, None, q, None, torch.zeros((2, 1)), torch.zeros(4, dtype=torch.float64), q, None)
    with pytest.raises(ValueError, match="CUDA"):
        nn.linearQ4(None, None, torch.zeros((1, 32)), torch.zeros((4, 8), dtype=torch.int32), torch.zeros((1, 8)),
                    torch.zeros((1, 8)), 32)


def test_reference_rounding_is_exact():
    """The 64-bit quotients of the tests' plain form give the nearest whole number
    of the exact quotient (rational arithmetic), ties included."""
    from fractions import Fraction
    g = np.random.default_rng(5)
    s = np.float32(0.37)
    halves = (np.arange(-126, 127) + 0.5).astype(np.float64)
    near = (halves * np.float64(s)).astype(np.float32)  # float32 values next to the ties
    xs = np.concatenate([near, np.nextafter(near, np.float32(100)), np.nextafter(near, np.float32(-100)),
                         (g.standard_normal(2000) * 10).astype(np.float32), np.float32([2.5, 3.5, -0.5])])
    for scale in (s, np.float32(1.0), np.float32(2.0 ** -40), np.float32(0.1)):
        for x in xs.astype(np.float32):
            want = round(Fraction(float(x)) / Fraction(float(scale)))  # ties to even
            assert int(np.rint(np.float64(x) / np.float64(scale))) == want
    assert ref.U == 2.0 ** -24
