"""The operators around a layer's int8 experts at the edges of what they take: the longest rows, with the largest sums that
32-bit integers hold, rows far apart, and one workspace for calls of different sizes."""
import numpy as np
import pytest

from test_gpu_moe_i8 import Layer, check, forward, oracle, routes, rows_of
from test_gpu_route_rows import check as check_routes, oracle as routes64

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
LONGEST = 131071


@pytest.fixture(scope="module")
def be():
    import lbhip
    if not torch.cuda.is_available():
        pytest.fail("no GPU visible")
    b = lbhip.HipBackend(0)
    yield b
    b.close()


@pytest.mark.parametrize("tokens", [2, 40])
@pytest.mark.parametrize("n,ffn", [(LONGEST, 20), (20, LONGEST)])
def test_longest_rows(be, n, ffn, tokens):
    """131071 products of -128 and -128 are 2^31 - 16384; tokens of 40 are more than 64 (token, slot) pairs."""
    layer = Layer(be, 3, n, ffn, 0, seed=7)
    (g, u, d) = layer.raw[1]
    g[0][3] = -128
    d[0][5] = -128
    layer.m.close()
    layer.m = be.moe_i8_create([(be.upload_i8_gated(*a, *b), be.upload_i8(*c)) for a, b, c in layer.raw])
    q, s = rows_of(tokens, n, 3)
    q[0] = -128
    ids, coefs = routes(tokens, 3, 2, 4)
    ids[0] = torch.tensor([1, 2], dtype=torch.int32, device="cuda")
    want = oracle(layer, q, s, ids, coefs, None)
    check(forward(be, layer, q, s, ids, coefs, torch.zeros(tokens, n, device="cuda")), want)


@pytest.mark.parametrize("tokens", [2, 20])
def test_experts_of_rows_far_apart(be, tokens):
    """Rows 2^23 - 48 apart, the furthest but for the alignment: what lies between them is left alone."""
    n, far = 160, (1 << 23) - 48
    layer = Layer(be, 6, n, 96, 40, seed=2)
    q, s = rows_of(tokens, n, 5)
    ids, coefs = routes(tokens, 6, 4, 6)
    wide = torch.full((tokens, far), 99, dtype=torch.int8, device="cuda")
    wide[:, :n] = q
    want = forward(be, layer, q, s, ids, coefs, torch.zeros(tokens, n, device="cuda"))
    check(want, oracle(layer, q, s, ids, coefs, None))
    out = torch.zeros(tokens, far, dtype=torch.float16, device="cuda")
    forward(be, layer, wide[:, :n], s, ids, coefs, out[:, :n])
    assert torch.equal(out[:, :n], want.half()) and not bool(out[:, n:].any())


def routed(be, r, x, space, top_k=4):
    n = x.shape[0]
    ids, coefs = torch.zeros(n, top_k, dtype=torch.int32, device="cuda"), torch.zeros(n, top_k, device="cuda")
    logits = torch.zeros(n, r.n_experts, device="cuda")
    be.route_rows(r, x, ids, coefs, space, logits=logits)
    torch.cuda.synchronize()
    return ids.cpu().numpy(), coefs.cpu().numpy(), logits.cpu().numpy()


def test_routing_of_rows_far_apart_in_one_workspace(be):
    """The larger of two sizes serves every call up to it; bytes behind what a call takes are left alone."""
    import lbhip
    rng = np.random.default_rng(4)
    w = rng.standard_normal((24, 512)).astype(np.float32)
    r = be.router(w)
    need = be.route_rows_workspace_bytes
    most = 300
    space = torch.full((max(need(r, most), need(r, 256)),), 0x55, dtype=torch.uint8, device="cuda")
    x = torch.from_numpy(rng.standard_normal((most, 512)).astype(np.float32)).cuda()
    far = torch.zeros(most, (1 << 20) + 3, device="cuda")
    far[:, 1:513] = x
    for n in (1, 300, 17, 256, 257, 64):
        want = routes64(x[:n], w, None, 4, 0, 1.0)
        space.fill_(0x55)
        check_routes(routed(be, r, far[:n, 1:513], space), want)
        assert bool((space[need(r, n):] == 0x55).all())
    few = torch.zeros(need(r, most), dtype=torch.uint8, device="cuda")
    with pytest.raises(lbhip.BackendError):
        routed(be, r, x[:256], few)
