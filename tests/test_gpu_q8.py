"""The 8-bit KV cache -- append, read-back, attention -- against plain
implementations in 64 bits."""
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


make_cache = ref.make_cache


# ---- append -----------------------------------------------------------------
def run_append(nn, B, H, T, D, block, Tn, starts, counts=None, layout=1, seed=0, grow=3.0):
    g = np.random.default_rng(seed)
    caches = [make_cache(g, B, H, T, D, block) for _ in range(2)]
    new = [(g.standard_normal((B, Tn, H, D)) * grow).astype(np.float32) for _ in range(2)]
    starts = np.asarray(starts, np.int32)
    want = []
    for (q, s), x in zip(caches, new):
        q, s = q.copy(), s.copy()
        for b in range(B):
            n = Tn if counts is None else int(np.clip(counts[b], 0, Tn))
            for h in range(H):
                ref.append(x[b, :, h], q[b, h], s[b, h], int(starts[b]), n, block)
        want.append((q, s))
    dc = [(dev(q if layout else q.transpose(0, 2, 1, 3)), dev(s)) for q, s in caches]
    args = [dev(new[0]), dev(new[1]), dc[0][0], dc[1][0], dc[0][1], dc[1][1], dev(starts), block]
    nn.kvCacheAppendQ8(None, None, *args, None if counts is None else dev(np.asarray(counts, np.int32)), layout)
    for (q, s), (wq, ws) in zip(dc, want):
        q = q.cpu().numpy() if layout else q.cpu().numpy().transpose(0, 2, 1, 3)
        np.testing.assert_array_equal(s.cpu().numpy(), ws)
        np.testing.assert_array_equal(q, wq)
    return args


@pytest.mark.parametrize("layout", [1, 0])
@pytest.mark.parametrize("D", [128, 64, 96, 5])
@pytest.mark.parametrize("T,block,Tn,starts", [
    (64, 16, 1, [0, 15, 16]),      # first row, last of a block, first of the next
    (70, 32, 1, [69, 33, 1]),      # the short last block
    (200, 64, 100, [3, 100, 64]),  # several blocks, begun and whole
    (33, 7, 5, [28, 2, 6]),        # a block size that is no power of two
    (16, 128, 16, [0, 0, 0]),      # a block longer than the cache
    (300, 1, 9, [0, 100, 291]),    # a scale per token
])
def test_append(nn, layout, D, T, block, Tn, starts):
    run_append(nn, 3, 2, T, D, block, Tn, starts, layout=layout)


def test_append_padded_batch(nn):
    """Counts of none, some, all and more than all of the padded rows."""
    run_append(nn, 5, 2, 96, 64, 16, 12, [4, 50, 0, 84, 20], counts=[0, 5, 12, 99, -3])


def test_append_same_rows_again_changes_nothing(nn):
    args = run_append(nn, 2, 2, 64, 64, 16, 3, [5, 30])
    before = [t.clone() for t in args[2:6]]
    nn.kvCacheAppendQ8(None, None, *args)
    for a, b in zip(before, args[2:6]):
        assert torch.equal(a, b)


def test_append_rows_that_do_not_raise_the_scale(nn):
    run_append(nn, 2, 2, 64, 64, 16, 3, [5, 30], grow=1e-3)


def test_append_outside_the_cache_is_dropped_and_reported(nn):
    import alpakann_b200 as ann
    from alpakann_b200 import _capi
    queue = ann.Queue()
    queue.take_device_error()
    run_append(nn, 4, 1, 40, 64, 16, 8, [36, -3, 40, 2 ** 31 - 4])
    assert queue.take_device_error() == _capi.ANN_DEVERR_CACHE_RANGE
    run_append(nn, 2, 1, 40, 64, 16, 8, [32, 0])
    assert queue.take_device_error() == 0


def test_append_ties_zeros_and_tiny_values(nn):
    """Values on and next to the borders between whole numbers, an all-zero
    block, and amplitudes down to subnormals."""
    block, D = 16, 128
    for amp in (127.0, 12.7, 3e38, 1e-25, 1e-33, 1e-38, 1e-43, 0.0):
        with np.errstate(all="ignore"):
            s = np.float32(np.float32(amp) * (np.float32(1) / np.float32(127)))
            n = np.arange(-64, 64) + 0.5
            x = np.tile((n * np.float64(s)).astype(np.float32), (block, 1))
            x[1] = np.nextafter(x[0], np.float32(np.inf))
            x[2] = np.nextafter(x[0], np.float32(-np.inf))
            x[3, 0] = amp
        q = np.zeros((block, D), np.int8)
        sc = np.zeros(1, np.float32)
        ref.append(x, q, sc, 0, block, block)
        kc, vc = torch.ones((1, 1, block, D), dtype=torch.int8, device="cuda"), torch.ones((1, 1, block, D),
                                                                                         dtype=torch.int8, device="cuda")
        ks, vs = torch.ones((1, 1, 1), device="cuda"), torch.ones((1, 1, 1), device="cuda")
        rows = dev(x[None, :, None])
        nn.kvCacheAppendQ8(None, None, rows, rows, kc, vc, ks, vs, dev(np.zeros(1, np.int32)), block)
        assert ks.item() == sc[0] and vs.item() == sc[0]
        np.testing.assert_array_equal(kc.cpu().numpy()[0, 0], q, err_msg=str(amp))
        assert torch.equal(kc, vc)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_append_non_finite_poisons_its_block_only(nn, bad):
    g = np.random.default_rng(1)
    B, H, T, D, block = 1, 2, 64, 64, 16
    kc, ks = make_cache(g, B, H, T, D, block)
    x = g.standard_normal((1, 20, H, D)).astype(np.float32)
    x[0, 3, 1, 7] = bad
    dkc, dks, dvc, dvs = dev(kc), dev(ks), dev(kc), dev(ks)
    nn.kvCacheAppendQ8(None, None, dev(x), dev(x), dkc, dvc, dks, dvs, dev(np.array([10], np.int32)), block)
    out = torch.zeros((B, H, T, D), device="cuda")
    out2 = torch.zeros_like(out)
    nn.kvCacheReadQ8(None, None, dkc, dvc, dks, dvs, out, out2, block)
    finite = torch.isfinite(out).all(-1).cpu().numpy()
    assert finite[0, 0].all()
    assert not finite[0, 1, :16].any()  # NaN or infinity * 0, never a wrong finite value; token 13 lies in block 0
    assert finite[0, 1, 16:].all()
    # a later finite row does not hide it
    nn.kvCacheAppendQ8(None, None, dev(x[:, 4:5]), dev(x[:, 4:5]), dkc, dvc, dks, dvs, dev(np.array([15], np.int32)),
                       block)
    assert not math.isfinite(dks[0, 1, 0].item())


# ---- read-back ----------------------------------------------------------------
@pytest.mark.parametrize("D,T,Tout,block,lengths", [(128, 100, 100, 16, [0, 1, 100]), (64, 65, 40, 64, [70, 40, 39]),
                                                    (7, 30, 30, 4, None), (256, 2048, 2048, 128, [2048, 5, -1])])
@pytest.mark.parametrize("layout", [1, 0])
def test_read_back(nn, D, T, Tout, block, lengths, layout):
    g = np.random.default_rng(2)
    kc, ks = make_cache(g, 3, 2, T, D, block)
    vc, vs = make_cache(g, 3, 2, T, D, block)
    flip = (lambda a: a) if layout else (lambda a: a.transpose(0, 2, 1, 3))
    outs = [torch.full(flip(np.zeros((3, 2, Tout, D))).shape, 7.0, device="cuda") for _ in range(2)]
    nn.kvCacheReadQ8(None, None, dev(flip(kc)), dev(flip(vc)), dev(ks), dev(vs), *outs, block,
                     None if lengths is None else dev(np.array(lengths, np.int32)), layout)
    blk = np.arange(T) // block
    for o, q, s in zip(outs, (kc, vc), (ks, vs)):
        want = (q.astype(np.float32) * s[:, :, blk, None])[:, :, :Tout].copy()
        if lengths is not None:
            for b, n in enumerate(lengths):
                want[b, :, max(0, n):] = 7.0
        np.testing.assert_array_equal(flip(o.cpu().numpy()), want)  # one rounding: equal bits


# ---- attention ----------------------------------------------------------------
def run_attend(nn, B, Tq, g_, Hkv, D, T, block, lengths=None, causal=True, layout=1, seed=0, scale=None, qs=1.0):
    g = np.random.default_rng(seed)
    kc, ks = make_cache(g, B, Hkv, T, D, block)
    vc, vs = make_cache(g, B, Hkv, T, D, block)
    q = (g.standard_normal((B, Tq, Hkv * g_, D)) * qs).astype(np.float32)
    scale = 1 / math.sqrt(D) if scale is None else scale
    flip = (lambda a: a) if layout else (lambda a: a.transpose(0, 2, 1, 3))
    out = torch.full(q.shape, float("nan"), device="cuda")
    ln = None if lengths is None else dev(np.asarray(lengths, np.int32))
    args = (dev(q), dev(flip(kc)), dev(flip(vc)), dev(ks), dev(vs), out, block, ln, scale, g_, layout, causal)
    nn.attentionDecodeQ8(None, None, *args)
    want, tol = ref.attend(q, kc, vc, ks, vs, lengths, block, scale, g_, causal)
    ref.assert_within(out.cpu().numpy(), want, tol, "attention")
    for b in range(B):  # rows without a key are exactly zero
        n = T if lengths is None else int(np.clip(lengths[b], 0, T))
        for i in range(Tq):
            if (n - Tq + 1 + i if causal else n) <= 0:
                assert not out[b, i].any()
    return args, out


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("block", [16, 64])
@pytest.mark.parametrize("T,lengths", [
    (1, None), (16, [16, 1, 0]), (17, [17, 2, 16]), (33, [33, 32, 31]), (200, [200, 65, 129]), (1000, [999, 500, 8]),
    (4099, [4099, 4096, 7])])
def test_attention_lengths(nn, D, block, T, lengths):
    run_attend(nn, 3, 1, 4, 2, D, T, block, lengths)


@pytest.mark.parametrize("g_", [1, 2, 3, 5, 8, 9, 16, 33])
def test_attention_group_sizes(nn, g_):
    run_attend(nn, 2, 1, g_, 2, 128, 150, 32, [150, 47])


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("Tq,g_", [(2, 1), (5, 3), (8, 1), (17, 2), (40, 1)])
def test_attention_several_tokens(nn, Tq, g_, causal):
    run_attend(nn, 3, Tq, g_, 2, 64, 90, 16, [90, 5, 0], causal)  # 5 keys: the first queries see none


@pytest.mark.parametrize("layout", [0, 1])
def test_attention_layouts_and_lengths_past_the_cache(nn, layout):
    run_attend(nn, 3, 1, 2, 3, 128, 77, 128, [1000, -4, 2 ** 31 - 1], layout=layout)


@pytest.mark.parametrize("qs,scale", [(1e-20, 1e19), (3e4, 1e-4), (1.0, 0.0), (1.0, -0.1), (40.0, 0.5)])
def test_attention_ranges(nn, qs, scale):
    """Queries far from 1, a peaked softmax, zero and negative scales."""
    run_attend(nn, 2, 1, 4, 2, 128, 300, 64, [300, 299], scale=scale, qs=qs)


def test_attention_strided_views(nn):
    """Q and out inside fused tensors, caches as a layer of a larger one with a head pitch."""
    g = np.random.default_rng(7)
    B, Hkv, g_, D, T, block = 2, 2, 4, 128, 130, 32
    big = torch.from_numpy(g.integers(-127, 128, (B, 3, Hkv + 1, T + 3, D)).astype(np.int8)).cuda()
    kc, vc = big[:, 0, :Hkv, 1:T + 1], big[:, 2, 1:, 2:T + 2]
    sc = torch.from_numpy((g.uniform(0.2, 2, (B, Hkv, 5, 2)) / 127).astype(np.float32)).cuda()
    ks, vs = sc[..., 0], sc[..., 1]
    fused = torch.from_numpy(g.standard_normal((B, 1, 3 * Hkv * g_, D)).astype(np.float32)).cuda()
    q = fused[:, :, ::3]
    o = torch.zeros((B, 1, Hkv * g_, 2 * D), device="cuda")[..., ::2]
    nn.attentionDecodeQ8(None, None, q, kc, vc, ks, vs, o, block, None, 0.1, g_)
    want, tol = ref.attend(*(t.cpu().numpy() for t in (q, kc, vc, ks, vs)), None, block, 0.1, g_)
    ref.assert_within(o.cpu().numpy(), want, tol, "strided")


def test_attention_long_cache_and_far_offsets(nn):
    """KV heads more than 2^31 bytes apart, and enough keys for every split."""
    Hkv, D, T, block = 2, 128, 20000, 64
    pitch = 2 ** 31 + 4096
    g = np.random.default_rng(9)
    store = torch.zeros(pitch + T * D, dtype=torch.int8, device="cuda")
    view = store.as_strided((1, Hkv, T, D), (0, pitch, D, 1))
    kc, ks = make_cache(g, 1, Hkv, T, D, block)
    view.copy_(torch.from_numpy(kc))
    q = g.standard_normal((1, 1, 8, D)).astype(np.float32)
    out = torch.empty((1, 1, 8, D), device="cuda")
    nn.attentionDecodeQ8(None, None, dev(q), view, view, dev(ks), dev(ks), out, block, None, None, 4)
    want, tol = ref.attend(q, kc, kc, ks, ks, None, block, 1 / math.sqrt(D), 4)
    ref.assert_within(out.cpu().numpy(), want, tol, "far heads")
    # appended and read back there too
    x = g.standard_normal((1, 3, Hkv, D)).astype(np.float32)
    v2, s2 = dev(kc), dev(ks)
    s1 = dev(ks)
    nn.kvCacheAppendQ8(None, None, dev(x), dev(x), view, v2, s1, s2, dev(np.array([T - 5], np.int32)), block)
    assert torch.equal(view, v2) and torch.equal(s1, s2)


@pytest.mark.parametrize("D,g_,Tq", [(64, 1, 1), (64, 8, 1), (128, 4, 1), (128, 3, 2), (128, 5, 3), (256, 2, 1),
                                     (256, 4, 5)])
@pytest.mark.parametrize("block", [16, 128])
def test_attention_few_long_sequences(nn, D, g_, Tq, block):
    """Few KV heads over long caches: shares of keys that cut sequences anywhere, empty and
    single-key sequences between them, and parts merged."""
    run_attend(nn, 4, Tq, g_, 2, D, 20011, block, [20011, 0, 1, 7777])


@pytest.mark.parametrize("g_", [4, 8])
def test_attention_many_ragged_sequences(nn, g_):
    """More sequences than lanes, most of them short, in caches of 20000 tokens."""
    g = np.random.default_rng(g_)
    lengths = g.integers(0, 300, 130)
    lengths[[0, 3, 31, 32, 64, 129]] = [0, 20000, 0, 4096, 12001, 0]
    run_attend(nn, 130, 1, g_, 1, 64, 20000, 64, lengths)


def test_attention_shares_replayed_and_side_by_side(nn):
    """Calls whose parts are merged: captured with their scratch and replayed with new lengths, two graphs at once."""
    args, out = run_attend(nn, 2, 1, 8, 1, 128, 30000, 64, [30000, 12345])
    streams, graphs, outs = [torch.cuda.Stream() for _ in range(2)], [], [torch.empty_like(out) for _ in range(2)]
    torch.cuda.synchronize()
    for st, o in zip(streams, outs):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=st):
            nn.attentionDecodeQ8(None, None, *args[:5], o, *args[6:])
            nn.attentionDecodeQ8(None, None, *args[:5], o, *args[6:])
        graphs.append(graph)
    for n in ([30000, 12345], [1, 29999], [0, 0], [16384, 64]):
        args[7].copy_(torch.tensor(n, dtype=torch.int32))
        want = torch.empty_like(out)
        nn.attentionDecodeQ8(None, None, *args[:5], want, *args[6:])
        torch.cuda.synchronize()
        for _ in range(3):
            for st, graph in zip(streams, graphs):
                with torch.cuda.stream(st):
                    graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, want) for o in outs)


def test_attention_scales_of_every_size_and_sign(nn):
    """V's and K's scales over 2^40 and of both signs: sums whose reference moves along the sequence."""
    g = np.random.default_rng(12)
    for g_, T in ((2, 2000), (8, 2000), (4, 40000)):
        B, Hkv, D, block = 1, 2, 128, 16
        kc, ks = make_cache(g, B, Hkv, T, D, block)
        vc, vs = make_cache(g, B, Hkv, T, D, block)
        vs *= (2.0 ** g.integers(-20, 20, vs.shape)).astype(np.float32) * g.choice([-1, 1], vs.shape)
        vs[0, 0, :3], vs[0, 1, 5] = 0, np.float32(1e-42)
        ks *= g.choice([-1, 1], ks.shape)
        q = g.standard_normal((B, 1, Hkv * g_, D)).astype(np.float32)
        out = torch.empty(q.shape, device="cuda")
        nn.attentionDecodeQ8(None, None, dev(q), dev(kc), dev(vc), dev(ks), dev(vs), out, block, None, 0.05, g_)
        want, tol = ref.attend(q, kc, vc, ks, vs, None, block, 0.05, g_)
        ref.assert_within(out.cpu().numpy(), want, tol, f"scales {g_} {T}")


def test_attention_growing_scores(nn):
    """Keys in rising and in falling order of score: the running maximum moves at every tile, or never."""
    D, T, block = 128, 3000, 64
    g = np.random.default_rng(3)
    q = np.ones((1, 1, 4, D), np.float32)
    for order in (1, -1):
        level = np.linspace(-127, 127, T)[::order]
        kc = np.clip(np.rint(level[:, None] + g.uniform(-1, 1, (T, D))), -127, 127).astype(np.int8)[None, None]
        ks = np.full((1, 1, -(-T // block)), 0.01, np.float32)
        vc, vs = make_cache(g, 1, 1, T, D, block)
        for scale in (0.01, 0.3):
            out = torch.empty(q.shape, device="cuda")
            nn.attentionDecodeQ8(None, None, dev(q), dev(kc), dev(vc), dev(ks), dev(vs), out, block, None, scale, 4)
            want, tol = ref.attend(q, kc, vc, ks, vs, None, block, scale, 4)
            ref.assert_within(out.cpu().numpy(), want, tol, f"order {order} scale {scale}")


def test_attention_ignores_what_lies_behind_the_last_key(nn):
    """Stale integers and NaN / infinite scales past the length change nothing."""
    args, out = run_attend(nn, 2, 1, 4, 2, 128, 200, 16, [100, 33])
    ks, vs = args[3].clone(), args[4].clone()
    for s, n in ((0, 100), (1, 33)):
        ks[s, :, -(-n // 16):] = float("nan")
        vs[s, :, -(-n // 16):] = float("inf")
    again = torch.empty_like(out)
    nn.attentionDecodeQ8(None, None, *args[:3], ks, vs, again, *args[6:])
    assert torch.equal(out, again)


def test_attention_non_finite_reaches_its_rows_only(nn):
    args, out = run_attend(nn, 2, 1, 4, 2, 128, 200, 16, [100, 33])
    vs = args[4].clone()
    vs[0, 1, 2] = float("nan")
    got = torch.empty_like(out)
    nn.attentionDecodeQ8(None, None, *args[:4], vs, got, *args[6:])
    assert torch.isnan(got[0, 0, 4:]).all()
    assert torch.equal(got[0, 0, :4], out[0, 0, :4]) and torch.equal(got[1], out[1])
    q = args[0].clone()
    q[1, 0, 2, 5] = float("nan")
    nn.attentionDecodeQ8(None, None, q, *args[1:5], got, *args[6:])
    assert torch.isnan(got[1, 0, 2]).all()
    rest = torch.ones(8, dtype=torch.bool)
    rest[2] = False
    assert torch.equal(got[1, 0, rest], out[1, 0, rest]) and torch.equal(got[0], out[0])


def test_attention_is_repeatable_and_shares_inputs_across_streams(nn):
    """The same bits on every call, on two streams at once, and from a replayed graph with new lengths."""
    args, out = run_attend(nn, 4, 1, 8, 2, 128, 5000, 64, [5000, 3, 2500, 4999])
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [torch.empty_like(out) for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(3):
        for s, o in zip(streams, outs):
            nn.attentionDecodeQ8(s, None, *args[:5], o, *args[6:])
    torch.cuda.synchronize()
    assert all(torch.equal(o, out) for o in outs)
    got = torch.empty_like(out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        nn.attentionDecodeQ8(None, None, *args[:5], got, *args[6:])
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, out)
    args[7].copy_(torch.tensor([17, 0, 4000, 64], dtype=torch.int32))
    want = torch.empty_like(out)
    nn.attentionDecodeQ8(None, None, *args[:5], want, *args[6:])
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, want) and not torch.equal(got, out)


@pytest.mark.parametrize("D", [64, 128])
def test_cached_prefix_feeds_the_prefill_kernel(nn, D):
    """A prompt appended in chunks, read back, and attended to by attentionPrefill:
    the last token agrees with attentionDecodeQ8 on the same cache. Both compute
    from the same float32 rows; the bound is the two sides' together."""
    g = np.random.default_rng(4)
    B, H, T, block = 2, 4, 96, 32
    kc, vc = (torch.zeros((B, H, T, D), dtype=torch.int8, device="cuda") for _ in range(2))
    ks, vs = (torch.zeros((B, H, T // block), device="cuda") for _ in range(2))
    x = [g.standard_normal((B, T, H, D)).astype(np.float32) for _ in range(3)]
    for lo, hi in ((0, 40), (40, 41), (41, 96)):
        nn.kvCacheAppendQ8(None, None, dev(x[0][:, lo:hi]), dev(x[1][:, lo:hi]), kc, vc, ks, vs,
                           dev(np.full(B, lo, np.int32)), block)
    ko, vo = (torch.empty((B, H, T, D), device="cuda") for _ in range(2))
    nn.kvCacheReadQ8(None, None, kc, vc, ks, vs, ko, vo, block)
    # Every rounding is off by at most half of its step, and a block's step only
    # grows. Tokens 32..39 lie in a block that three appends touch: rounded once
    # and anew at most twice, 3 * 0.5 = 1.5 steps of the final scale.
    step = np.repeat(ks.cpu().numpy(), block, 2)[..., None]
    assert bool((np.abs(ko.cpu().numpy() - x[0].transpose(0, 2, 1, 3)) <= 1.501 * step).all())
    full = torch.empty((B, T, H, D), device="cuda")
    nn.attentionPrefill(None, None, dev(x[2]), ko, vo, full, None, 1, 1, True)
    last = torch.empty((B, 1, H, D), device="cuda")
    nn.attentionDecodeQ8(None, None, dev(x[2][:, -1:]), kc, vc, ks, vs, last, block)
    want, tol = ref.attend(x[2][:, -1:], *(t.cpu().numpy() for t in (kc, vc, ks, vs)), None, block,
                           1 / math.sqrt(D), 1)
    ref.assert_within(last.cpu().numpy(), want, tol)
    ref.assert_within(full[:, -1:].cpu().numpy(), want, tol)
