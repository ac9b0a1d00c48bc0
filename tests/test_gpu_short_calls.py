"""The short calls through ctypes give what the compiled module gives."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def short():
    from tests.helpers import build_library
    build_library()
    from alpakann_b200 import _short
    return _short


def test_through_ctypes_as_through_the_module(short, monkeypatch):
    from alpakann_b200.onHost import nn
    assert not isinstance(short.binding, short.ThroughCtypes)
    slow = short._through_ctypes()
    g = torch.Generator("cuda").manual_seed(0)
    rnd = lambda *shape, **kw: torch.randn(*shape, generator=g, device="cuda", **kw)
    ints = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")
    x, w = rnd(2, 256), torch.randint(0, 2**31, (32, 64), generator=g, device="cuda", dtype=torch.int32)
    ws, bias = torch.rand(2, 64, generator=g, device="cuda"), rnd(64)
    freq, new = torch.rand(32, dtype=torch.float64, generator=g, device="cuda"), rnd(2, 3, 2, 64)

    def everything(queue):
        y = torch.zeros(2, 64, device="cuda")
        nn.linearQ4(queue, None, x, w, ws, y, 128, bias=bias, activation=nn.Activation.silu, residual=y)
        q, q64 = torch.zeros(2, 1, 4, 64, device="cuda"), torch.zeros(2, 1, 4, 64, device="cuda", dtype=torch.float64)
        nn.rotary(queue, None, y.view(2, 1, 1, 64).expand(2, 1, 4, 64), None, ints(3, 9).view(2, 1), freq, q, None,
                  nn.RotaryPairs.halves)
        nn.rotary(queue, None, q.double(), None, ints(5), freq, q64, None, inverse=True, magnitude=0.5)
        kc, vc = (torch.zeros(2, 2, 48, 64, device="cuda", dtype=torch.int8) for _ in range(2))
        ks, vs = (torch.zeros(2, 2, 3, device="cuda") for _ in range(2))
        nn.kvCacheAppendQ8(queue, None, new, new, kc, vc, ks, vs, ints(0, 14), 16, counts=ints(3, 2))
        back = torch.zeros(2, 2, 2, 48, 64, device="cuda")
        nn.kvCacheReadQ8(queue, None, kc, vc, ks, vs, back[0], back[1], 16, lengths=ints(3, 16))
        out = torch.zeros(2, 1, 4, 64, device="cuda")
        nn.attentionDecodeQ8(queue, None, q, kc, vc, ks, vs, out, 16, ints(3, 16), queriesPerKvGroup=2)
        torch.cuda.synchronize()
        return y, q, q64, kc, vc, ks, vs, back, out

    for queue in (None, torch.cuda.current_stream(), torch.cuda.current_stream().cuda_stream):
        want = everything(queue)
        with monkeypatch.context() as m:
            m.setattr(nn, "binding", slow)
            got = everything(queue)
            q, kc, ks = got[1], got[3], got[5]
            for block, group, layout in [(2**32 + 16, 1, 1), (16, -1, 1), (16, 2**40, 1), (16, 1, 2**32)]:
                with pytest.raises(OverflowError):
                    nn.attentionDecodeQ8(queue, None, q, kc, kc, ks, ks, q.clone(), block, queriesPerKvGroup=group,
                                         kvLayout=layout)
            with pytest.raises(ValueError, match="scales"):
                nn.attentionDecodeQ8(queue, None, q, kc, kc, ks, ks, q.clone(), 32, queriesPerKvGroup=2)
            with pytest.raises(TypeError, match="kCache"):
                nn.attentionDecodeQ8(queue, None, q, kc.float(), kc, ks, ks, q.clone(), 16, queriesPerKvGroup=2)
        assert all(torch.equal(a, b) for a, b in zip(got, want)) and all(t.any() for t in want)
