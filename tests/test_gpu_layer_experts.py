"""The experts' step of test_gpu_layer_i8's run of operators against the 64-bit value of the int8 rows, ids and
coefficients that the steps before it made."""
from types import SimpleNamespace

import pytest

from test_gpu_layer_i8 import Layer, stream_rows
from test_gpu_moe_i8 import check, oracle

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def be():
    import lbhip
    if not torch.cuda.is_available():
        pytest.fail("no GPU visible")
    b = lbhip.HipBackend(0)
    yield b
    b.close()


class Keeping:
    """A backend that keeps the raw weights of what it uploads."""

    def __init__(self, be):
        self.be, self.raw = be, {}

    def __getattr__(self, name):
        return getattr(self.be, name)

    def upload_i8(self, w, s):
        m = self.be.upload_i8(w, s)
        self.raw[m] = ((w, s),)
        return m

    def upload_i8_gated(self, g, gs, u, us):
        m = self.be.upload_i8_gated(g, gs, u, us)
        self.raw[m] = ((g, gs), (u, us))
        return m


@pytest.mark.parametrize("tokens,n,wide,experts,ffn,shared,top_k", [
    (1, 512, 1024, 8, 256, 512, 2), (6, 256, 300, 40, 96, 33, 6), (16, 768, 512, 12, 520, 64, 4), (50, 512, 768, 20, 128, 256, 8),
    (1, 2304, 256, 8, 200, 300, 3), (7, 2304, 256, 10, 96, 64, 4), (30, 2304, 256, 12, 64, 128, 4)])
@pytest.mark.parametrize("ty", [torch.float32, torch.bfloat16])
def test_experts_of_the_routed_rows(be, tokens, n, wide, experts, ffn, shared, top_k, ty):
    keeping = Keeping(be)
    la = Layer(keeping, n, wide, experts, ffn, shared, seed=n)
    routed, both = la.moe._keep
    raw = SimpleNamespace(n=n, raw=[keeping.raw[up] + keeping.raw[down] for up, down in routed],
                          shared=keeping.raw[both[0]] + keeping.raw[both[1]])
    b = la.buffers(be, tokens, ty, top_k)
    la.run(be, *stream_rows(tokens, la, ty, tokens), b)
    torch.cuda.synchronize()
    want = oracle(raw, b.q1, b.s1, b.ids, b.coefs, None)
    assert bool((want[1] > 0).any(1).all())
    check(b.y, want)
