"""The decode operators on compressed data at the ends of their ranges: inputs by the
hundred thousand, group sizes past the heads, a first call that is captured,
integer arguments outside their types."""
import math
import subprocess
import sys

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


@pytest.mark.parametrize("M,K,N,group", [(8, 57344, 40, 128), (8, 57472, 40, 128), (5, 130000, 33, 64),
                                         (3, 240000, 36, 4096), (1, 253952, 36, 32), (11, 58368, 2048, 128),
                                         (2, 253952, 2048, 128), (1, 364544, 36, 32), (3, 300000, 2052, 96)])
def test_linear_many_inputs(nn, M, K, N, group):
    """Rows that do not fit a CTA's memory eight at a time are taken fewer at a
    time. The sums in 64 bits are formed on the device, columns in slices."""
    g = torch.Generator("cuda").manual_seed(K)
    packed = torch.randint(-2**31, 2**31, (K // 8, N), generator=g, device="cuda", dtype=torch.int64).to(torch.int32)
    s = (torch.rand(-(-K // group), N, generator=g, device="cuda") + 0.5) * 0.2 / math.sqrt(K)
    x = torch.randn(M, K, generator=g, device="cuda")
    y = torch.full((M, N), float("nan"), device="cuda")
    nn.linearQ4(None, None, x, packed, s, y, group)
    shifts = torch.arange(0, 32, 4, device="cuda", dtype=torch.int32)
    for n in range(0, N, 256):
        u = (packed[:, None, n:n + 256] >> shifts[:, None] & 15).reshape(K, -1)
        w = (u - 8).double() * s[:, n:n + 256].double().repeat_interleave(group, 0)[:K]
        want, size = x.double() @ w, x.double().abs() @ w.abs()
        # x in digits: 2^-31 of the largest input each; then at most K sums and products in fp32
        tol = 2 * (K + 16) * ref.U * size + 2.0 ** -30 * x.abs().max() * w.abs().sum(0)
        ref.assert_within(y[:, n:n + 256].cpu().numpy(), want.cpu().numpy(), tol.cpu().numpy(), f"linear {M}x{K}x{N}")


def test_linear_refuses_more_inputs_than_fit(nn):
    K = 1 << 20
    x, y = torch.zeros(1, K, device="cuda"), torch.zeros(1, 4, device="cuda")
    packed, s = torch.zeros(K // 8, 4, dtype=torch.int32, device="cuda"), torch.zeros(K // 32, 4, device="cuda")
    with pytest.raises(Exception, match="inputs"):
        nn.linearQ4(None, None, x, packed, s, y, 32)


@pytest.mark.parametrize("group", [6, 7, 1000, 2**32 - 1])
def test_attention_groups_past_the_heads(nn, group):
    """Every query head reads KV head 0, as with a group of exactly the heads."""
    g = torch.Generator("cuda").manual_seed(1)
    kc, vc = (torch.randint(-127, 128, (2, 2, 100, 64), generator=g, device="cuda").to(torch.int8) for _ in range(2))
    ks, vs = (torch.rand(2, 2, 7, generator=g, device="cuda") * 0.01 for _ in range(2))
    q = torch.randn(2, 3, 6, 64, generator=g, device="cuda")
    want, out = torch.empty_like(q), torch.empty_like(q)
    nn.attentionDecodeQ8(None, None, q, kc, vc, ks, vs, want, 16, queriesPerKvGroup=6)
    nn.attentionDecodeQ8(None, None, q, kc, vc, ks, vs, out, 16, queriesPerKvGroup=group)
    assert torch.equal(out, want) and want.isfinite().all()


@pytest.mark.parametrize("B,Tq,g_,Hkv,D,T", [(2, 5, 5, 8, 128, 4096), (4, 4, 4, 4, 64, 16384), (2, 8, 2, 2, 128, 60000)])
def test_attention_many_rows_of_a_head(nn, B, Tq, g_, Hkv, D, T):
    """Sixteen rows a CTA, in clusters and in even shares."""
    from tests.test_gpu_q8 import run_attend
    run_attend(nn, B, Tq, g_, Hkv, D, T, 64, [T - 37 * b for b in range(B)])


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("which", ["K", "V"])
@pytest.mark.parametrize("g_,D", [(1, 64), (2, 128), (4, 64), (8, 128), (2, 256), (12, 256)])
def test_attention_scale_that_an_earlier_query_does_not_see(nn, g_, D, which, bad):
    """Two queries: the last block has one key, which only the second sees."""
    g = np.random.default_rng(D + g_)
    kc, vc = (g.integers(-127, 128, (1, 2, 40, D)).astype(np.int8) for _ in range(2))
    kc[:, :, 32] = np.abs(kc[:, :, 32])
    ks, vs = (g.uniform(0.005, 0.01, (1, 2, 3)).astype(np.float32) for _ in range(2))
    q = np.abs(g.standard_normal((1, 2, 2 * g_, D))).astype(np.float32)
    want, tol = ref.attend(q, kc, vc, ks, vs, [33], 16, 0.1, g_)
    (ks if which == "K" else vs)[:, :, 2] = bad
    dev = [torch.from_numpy(a).cuda() for a in (q, kc, vc, ks, vs)]
    out = torch.zeros_like(dev[0])
    nn.attentionDecodeQ8(None, None, *dev, out, 16, torch.tensor([33], dtype=torch.int32, device="cuda"), 0.1, g_)
    ref.assert_within(out[:, 0].cpu().numpy(), want[:, 0], tol[:, 0], "the first query")
    assert torch.isnan(out[:, 1]).all()


def test_integers_outside_their_type_are_refused(nn):
    q, kc = torch.zeros(1, 1, 1, 64, device="cuda"), torch.zeros(1, 1, 16, 64, dtype=torch.int8, device="cuda")
    s = torch.zeros(1, 1, 1, device="cuda")
    for block, group, layout in [(2**32 + 16, 1, 1), (16, -1, 1), (16, 2**40, 1), (16, 1, 2**32)]:
        with pytest.raises(OverflowError):
            nn.attentionDecodeQ8(None, None, q, kc, kc, s, s, q.clone(), block, queriesPerKvGroup=group, kvLayout=layout)


CAPTURED_FIRST = """
import torch
from alpakann_b200.onHost import nn
q = torch.randn(2, 1, 8, 128, device="cuda")
k = torch.randint(-127, 128, (2, 1, 40000, 128), device="cuda").to(torch.int8)
s = torch.rand(2, 1, 625, device="cuda") * 0.01
w, ws = torch.randint(0, 2**31, (512, 4096), device="cuda", dtype=torch.int32), torch.rand(32, 4096, device="cuda")
x, outs, ys = torch.randn(8, 4096, device="cuda"), [torch.zeros_like(q) for _ in range(2)], [torch.zeros(8, 4096, device="cuda") for _ in range(2)]
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    nn.attentionDecodeQ8(None, None, q, k, k, s, s, outs[0], 64, queriesPerKvGroup=8)
    nn.linearQ4(None, None, x, w, ws, ys[0], 128)
graph.replay()
nn.attentionDecodeQ8(None, None, q, k, k, s, s, outs[1], 64, queriesPerKvGroup=8)
nn.linearQ4(None, None, x, w, ws, ys[1], 128)
torch.cuda.synchronize()
assert outs[0].abs().sum() > 0 and torch.equal(*outs) and torch.equal(*ys)
print("equal")
"""


def test_first_call_of_a_process_is_captured(nn):
    """Kernel attributes and the scratch pool are made under the capture."""
    r = subprocess.run([sys.executable, "-c", CAPTURED_FIRST], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "equal" in r.stdout, r.stdout + r.stderr


def test_streams_devices_and_leaves(nn):
    """The current stream by default, a given one as a queue, and tensors that require gradients."""
    x, w, s = torch.randn(1, 4096, device="cuda"), torch.randint(0, 2**31, (512, 512), dtype=torch.int32, device="cuda"), \
        torch.rand(32, 512, device="cuda")
    want = torch.zeros(1, 512, device="cuda")
    nn.linearQ4(None, None, x, w, s, want, 128)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    for queue in (None, side, side.cuda_stream):
        out = torch.zeros_like(want)
        late = x.clone().zero_()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):  # the input comes late on the side stream
            torch.cuda._sleep(10_000_000)
            late.copy_(x)
            if queue is None:
                nn.linearQ4(None, None, late, w, s, out, 128)
        if queue is not None:
            nn.linearQ4(queue, None, late, w, s, out, 128)
        side.synchronize()
        assert torch.equal(out, want)
    leaf, out = torch.nn.Parameter(x), torch.zeros_like(want)
    nn.linearQ4(None, None, leaf, w, s, out, 128)
    assert torch.equal(out, want)


def test_chained_calls_wait_for_their_inputs(nn):
    """Every operator right behind the kernel that writes its input, on one stream, replayed, and
    behind a joined stream: launches overlap the end of the kernels before them, their reads must not."""
    B, D, T = 2, 128, 2048
    g = torch.Generator("cuda").manual_seed(2)
    rnd = lambda *shape: torch.randn(*shape, generator=g, device="cuda")
    x, w4 = rnd(B, 4096), torch.randint(-2**31, 2**31, (512, 4096), generator=g, device="cuda").to(torch.int32)
    ws, freq = torch.rand(32, 4096, generator=g, device="cuda") * 0.01, torch.rand(64, dtype=torch.float64, device="cuda")
    pos, lens = torch.tensor([1900, 7], dtype=torch.int32, device="cuda"), torch.tensor([1901, 8], dtype=torch.int32, device="cuda")
    kc0, vc0 = (torch.randint(-127, 128, (B, 8, T, D), generator=g, device="cuda").to(torch.int8) for _ in range(2))
    sc0 = torch.rand(B, 8, T // 64, generator=g, device="cuda") * 0.01
    kn0 = rnd(B, 1, 8, D)
    side = torch.cuda.Stream()

    def chain(join, sync):
        wait = torch.cuda.synchronize if sync else (lambda: None)
        kc, vc, ks, vs = kc0.clone(), vc0.clone(), sc0.clone(), sc0.clone()
        y, q, kn, out, back = (torch.zeros(n, device="cuda") for n in (B * 4096, B * 4096, B * 8 * D, B * 4096, 2 * B * 8 * T * D))
        back = back.view(2, B, 8, T, D)
        x1 = torch.zeros_like(x)
        if join:
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                x1.copy_(x)
            torch.cuda.current_stream().wait_stream(side)
        else:
            x1.copy_(x)
        for _ in range(3):
            wait()
            nn.linearQ4(None, None, x1, w4, ws, y.view(B, 4096), 128)
            wait()
            nn.rotary(None, None, y.view(B, 1, 32, D), kn0, pos.view(B, 1), freq, q.view(B, 1, 32, D), kn.view(B, 1, 8, D))
            wait()
            nn.kvCacheAppendQ8(None, None, kn.view(B, 1, 8, D), kn.view(B, 1, 8, D), kc, vc, ks, vs, pos, 64)
            wait()
            nn.attentionDecodeQ8(None, None, q.view(B, 1, 32, D), kc, vc, ks, vs, out.view(B, 1, 32, D), 64, lens,
                                 queriesPerKvGroup=4)
            wait()
            nn.linearQ4(None, None, out.view(B, 4096), w4, ws, x1, 128)
            wait()
            nn.kvCacheReadQ8(None, None, kc, vc, ks, vs, back[0], back[1], 64)
        return x1, out, back

    want = chain(False, True)
    for join in (False, True):
        for _ in range(20):
            got = chain(join, False)
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(got, want))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = chain(join, False)
        for _ in range(20):
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_slices_of_one_sequence_keep_odd_strides(nn):
    """One sequence, token or row of a tensor whose stride along that axis is odd: extent 1, no matter."""
    g = torch.Generator("cuda").manual_seed(3)

    def odd(t, *axes):
        """t's values under odd strides along axes of extent 1."""
        strides = [7 if i in axes else s for i, s in enumerate(t.stride())]
        return t.as_strided(t.shape, strides)

    q = torch.randn(1, 1, 4, 64, generator=g, device="cuda")
    kc, vc = (torch.randint(-127, 128, (1, 2, 48, 64), generator=g, device="cuda").to(torch.int8) for _ in range(2))
    ks = torch.rand(1, 2, 3, generator=g, device="cuda") * 0.01
    want, out = torch.zeros_like(q), torch.zeros_like(q)
    nn.attentionDecodeQ8(None, None, q, kc, vc, ks, ks, want, 16, queriesPerKvGroup=2)
    nn.attentionDecodeQ8(None, None, odd(q, 0, 1), odd(kc, 0), odd(vc, 0), odd(ks, 0), ks, odd(out, 0, 1), 16,
                         queriesPerKvGroup=2)
    assert torch.equal(out, want) and want.any()
    back = torch.zeros(2, 2, 1, 2, 48, 64, device="cuda")
    nn.kvCacheReadQ8(None, None, kc, vc, ks, ks, back[0, 0], back[0, 1], 16)
    nn.kvCacheReadQ8(None, None, odd(kc, 0), odd(vc, 0), odd(ks, 0), ks, odd(back[1, 0], 0), back[1, 1], 16)
    assert torch.equal(back[0], back[1])
    x, w = torch.randn(1, 256, generator=g, device="cuda"), torch.randint(0, 2**31, (32, 64), generator=g, device="cuda",
                                                                        dtype=torch.int32)
    s, y = torch.rand(1, 64, generator=g, device="cuda"), torch.zeros(2, 1, 64, device="cuda")
    nn.linearQ4(None, None, x, w, s, y[0], 256)
    nn.linearQ4(None, None, odd(x, 0), w, odd(s, 0), odd(y[1], 0), 256)
    assert torch.equal(y[0], y[1])
    f, pos = torch.rand(32, dtype=torch.float64, generator=g, device="cuda"), torch.tensor([[5]], dtype=torch.int32, device="cuda")
    turned = torch.zeros(2, 1, 1, 4, 64, device="cuda")
    nn.rotary(None, None, q, None, pos, f, turned[0], None)
    nn.rotary(None, None, odd(q, 0, 1), None, odd(pos, 0, 1), f, odd(turned[1], 0, 1), None)
    assert torch.equal(turned[0], turned[1])
