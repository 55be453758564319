"""The routed and shared experts of a layer over int8 matrices against a plain 64-bit implementation.

The kernels round twice (h to 32 bits, y to 32 bits) and once to y's type; the oracle rounds h the same way, so the
int8 rows between the two products are the same but where h lies within 2^-39 of a border of 32 bits and the value
that gives within 2^-24 of a border of the int8 rounding (the sigmoid is good to 2^-39): about one value in 2^30.  y is
then off by its own roundings, half a step each, and by some 1e-13 of its terms."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
TYPES = [torch.float32, torch.float16, torch.bfloat16]


@pytest.fixture(scope="module")
def be():
    import lbhip
    if not torch.cuda.is_available():
        pytest.fail("no GPU visible")
    b = lbhip.HipBackend(0)
    yield b
    b.close()


class Layer:
    def __init__(self, be, experts, n, ffn, shared, seed):
        g = torch.Generator(device="cuda").manual_seed(seed)

        def mat(rows, k):
            return (torch.randint(-127, 128, (rows, k), dtype=torch.int8, device="cuda", generator=g),
                    (torch.rand(rows, device="cuda", generator=g) + 0.5) / (73 * k ** 0.5))

        def expert(f):
            return mat(f, n), mat(f, n), mat(n, f)

        def upload(e):
            return be.upload_i8_gated(*e[0], *e[1]), be.upload_i8(*e[2])

        self.n, self.raw = n, [expert(ffn) for _ in range(experts)]
        self.shared = expert(shared) if shared else None
        self.m = be.moe_i8_create([upload(e) for e in self.raw], upload(self.shared) if shared else None)


def rows_of(tokens, n, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randint(-127, 128, (tokens, n), dtype=torch.int8, device="cuda", generator=g),
            (torch.rand(tokens, device="cuda", generator=g) + 0.5) / 40)


def routes(tokens, experts, top_k, seed, hot=0):
    g = torch.Generator(device="cuda").manual_seed(seed + 1)
    rank = torch.rand(tokens, experts, device="cuda", generator=g)
    rank[:, :hot] += 2
    return rank.topk(top_k, 1).indices.to(torch.int32), torch.rand(tokens, top_k, device="cuda", generator=g) - 0.2


def expert64(q, s, e):
    def prod(q, s, m):
        return (q.double() @ m[0].double().t().contiguous()) * s.double()[:, None] * m[1].double()

    g = prod(q, s, e[0])
    h = (g * torch.sigmoid(g) * prod(q, s, e[1])).float().double()
    hs = (h.abs().amax(1) / 127).float()
    hs = torch.where(hs < 2.0 ** -126, torch.zeros_like(hs), hs)
    hq = torch.where(hs[:, None] > 0, torch.round(h / torch.where(hs > 0, hs, 1.0).double()[:, None]), 0.0)
    return prod(hq, hs, e[2])


def oracle(layer, q, s, ids, coefs, residual):
    """(y, the sum of its terms' magnitudes)"""
    y = torch.zeros(q.shape[0], layer.n, dtype=torch.float64, device="cuda")
    size = torch.zeros_like(y)
    for e in torch.unique(ids).tolist():
        if not 0 <= e < len(layer.raw):
            continue
        t, slot = (ids == e).nonzero(as_tuple=True)
        out = expert64(q[t], s[t], layer.raw[e]) * coefs[t, slot].double()[:, None]
        y.index_add_(0, t, out)
        size.index_add_(0, t, out.abs())
    if layer.shared:
        out = expert64(q, s, layer.shared)
        y, size = y + out, size + out.abs()
    if residual is not None:
        y, size = y + residual.double(), size + residual.double().abs()
    return y, size


def forward(be, layer, q, s, ids, coefs, y, residual=None):
    space = torch.full((be.moe_i8_workspace_bytes(layer.m, *ids.shape),), 0x7f, dtype=torch.uint8, device="cuda")
    be.moe_i8_forward(layer.m, q, s, ids, coefs, y, space, residual=residual)
    torch.cuda.synchronize()
    return y


def check(got, want):
    y, size = want
    half = 2.0 ** -24 + (0 if got.dtype == torch.float32 else torch.finfo(got.dtype).eps / 2 * (1 + 2.0 ** -24))
    bad = (got.double() - y).abs() > y.abs() * half + size * 1e-12 + torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps
    assert not bool(bad.any()), f"{int(bad.sum())} of {bad.numel()}"


# (tokens, experts, top_k, n, ffn, shared): one token; up to 64 pairs and more; 16, 32 and 64 tokens a tile and
# beyond; widths that are no multiples of anything; rows longer than a workgroup's registers; a thousand experts
SHAPES = [(1, 4, 1, 64, 48, 0), (1, 12, 8, 512, 1536, 1024), (2, 3, 2, 100, 33, 7), (3, 20, 5, 1, 1, 1), (5, 40, 8, 300, 130, 256),
          (8, 30, 8, 256, 512, 0), (9, 16, 8, 272, 96, 80), (16, 8, 4, 1040, 200, 300), (17, 9, 4, 130, 520, 64), (33, 6, 3, 257, 100, 33),
          (64, 5, 5, 96, 64, 160), (65, 4, 2, 80, 300, 0), (100, 10, 4, 512, 256, 512), (256, 3, 1, 48, 32, 16), (256, 12, 8, 144, 64, 48),
          (128, 20, 16, 64, 48, 0), (4, 1024, 6, 32, 16, 0), (200, 1024, 10, 32, 16, 32), (2, 4, 2, 64, 5000, 9000), (30, 6, 2, 5000, 64, 0)]


@pytest.mark.parametrize("tokens,experts,top_k,n,ffn,shared", SHAPES)
def test_layers(be, tokens, experts, top_k, n, ffn, shared):
    layer = Layer(be, experts, n, ffn, shared, seed=n + ffn)
    q, s = rows_of(tokens, n, tokens)
    ids, coefs = routes(tokens, experts, top_k, tokens)
    want = None
    for ty in TYPES:
        res = torch.randn(tokens, n, device="cuda").to(ty)
        want = oracle(layer, q, s, ids, coefs, None) if want is None else want
        y = torch.full((tokens, n), 3.0, dtype=ty, device="cuda")
        check(forward(be, layer, q, s, ids, coefs, y, res), (want[0] + res.double(), want[1] + res.double().abs()))
        check(forward(be, layer, q, s, ids, coefs, y), want)


@pytest.mark.parametrize("tokens", [1, 7, 40, 150])
def test_hot_experts_repeated_experts_and_empty_slots(be, tokens):
    layer = Layer(be, 7, 160, 96, 64, seed=1)
    q, s = rows_of(tokens, 160, 2)
    _, coefs = routes(tokens, 7, 4, 3)
    cases = [torch.full((tokens, 4), 6), torch.tensor([3, 3, 1, 3]).repeat(tokens, 1), torch.full((tokens, 4), -1),
             torch.tensor([7, 2, 2 ** 31 - 1, -5]).repeat(tokens, 1), torch.arange(4 * tokens).reshape(tokens, 4) % 9 - 1]
    for ids in cases:
        ids = ids.to(torch.int32).cuda()
        c = torch.where((ids < 0) | (ids > 6), float("nan"), coefs) if tokens != 7 else coefs   # an empty slot's is not used
        res = torch.randn(tokens, 160, device="cuda")
        want = oracle(layer, q, s, ids, torch.nan_to_num(c), res)
        check(forward(be, layer, q, s, ids, c, torch.zeros(tokens, 160, device="cuda"), res), want)


def test_all_slots_empty_without_a_shared_expert(be):
    layer = Layer(be, 3, 64, 32, 0, seed=1)
    for tokens in (1, 5, 70):
        q, s = rows_of(tokens, 64, 1)
        ids = torch.full((tokens, 2), -1, dtype=torch.int32, device="cuda")
        coefs = torch.full((tokens, 2), float("inf"), device="cuda")
        res = torch.randn(tokens, 64, device="cuda")
        assert torch.equal(forward(be, layer, q, s, ids, coefs, torch.ones(tokens, 64, device="cuda"), res), res)
        assert not bool(forward(be, layer, q, s, ids, coefs, torch.ones(tokens, 64, device="cuda")).any())


def test_a_token_s_bits_do_not_depend_on_the_batch(be):
    layer = Layer(be, 24, 320, 512, 256, seed=4)
    q, s = rows_of(200, 320, 5)
    ids, coefs = routes(200, 24, 6, 6, hot=1)
    res = torch.randn(200, 320, device="cuda")
    whole = forward(be, layer, q, s, ids, coefs, torch.zeros(200, 320, device="cuda"), res)
    for at, n in ((0, 1), (77, 2), (10, 10), (60, 11), (100, 33), (3, 90)):
        part = [t[at:at + n].contiguous() for t in (q, s, ids, coefs)]
        assert torch.equal(forward(be, layer, *part, torch.zeros(n, 320, device="cuda"), res[at:at + n]), whole[at:at + n])
    order = torch.randperm(200, device="cuda")
    again = forward(be, layer, q[order], s[order], ids[order], coefs[order], torch.zeros(200, 320, device="cuda"), res[order])
    assert torch.equal(again, whole[order])


@pytest.mark.parametrize("tokens", [3, 40])
def test_rows_that_are_zero_or_not_finite(be, tokens):
    """A scale of NaN reaches its own token alone; zeros stay zeros; a coefficient that is not finite shows."""
    layer = Layer(be, 5, 128, 64, 32, seed=8)
    q, s = rows_of(tokens, 128, 1)
    ids, coefs = routes(tokens, 5, 3, 2)
    s[1] = float("nan")
    q[0] = 0
    y = forward(be, layer, q, s, ids, coefs, torch.zeros(tokens, 128, device="cuda"))
    assert bool(torch.isnan(y[1]).all()) and not bool(y[0].any())
    s[1], coefs[2, 1] = 1.0, float("inf")
    y = forward(be, layer, q, s, ids, coefs, torch.zeros(tokens, 128, device="cuda"))
    assert not bool(torch.isfinite(y[2]).any()) and bool(torch.isfinite(y[1]).all())
    s[1] = 1e30                                       # h is not finite: scale NaN, as the row quantizer has it
    y = forward(be, layer, q, s, ids, coefs, torch.zeros(tokens, 128, device="cuda"))
    assert bool(torch.isnan(y[1]).all())


@pytest.mark.parametrize("tokens", [2, 30])
def test_in_place_strides_and_odd_addresses(be, tokens):
    layer = Layer(be, 6, 200, 72, 40, seed=3)
    q, s = rows_of(tokens, 200, 4)
    ids, coefs = routes(tokens, 6, 2, 5)
    res = torch.randn(tokens, 200, device="cuda").bfloat16()
    want = forward(be, layer, q, s, ids, coefs, torch.zeros_like(res), res)
    check(want, oracle(layer, q, s, ids, coefs, res))
    wide = torch.full((tokens, 333), 77, dtype=torch.int8, device="cuda")
    wide[:, 5:205] = q
    buf = torch.full((tokens, 301), 9.0, dtype=torch.bfloat16, device="cuda")
    view = buf[:, 3:203]
    view.copy_(res)
    forward(be, layer, wide[:, 5:205], s, ids, coefs, view, view)
    assert torch.equal(view, want)
    assert bool((buf[:, :3] == 9).all()) and bool((buf[:, 203:] == 9).all())


def test_steps_of_the_dense_block(be):
    """One expert with coefficient 1 is the dense block's gated product, quantization and product."""
    layer = Layer(be, 1, 512, 384, 0, seed=2)
    q, s = rows_of(9, 512, 3)
    pair, down = layer.m._keep[0][0]
    h, hq, hs = torch.zeros(9, 384, device="cuda"), torch.zeros(9, 384, dtype=torch.int8, device="cuda"), torch.zeros(9, device="cuda")
    want = torch.zeros(9, 512, device="cuda")
    be.gemm_i8_swiglu(pair, q, s, h)
    be.quantize_i8_rows(h, hq, hs)
    be.gemm_i8(down, hq, hs, want)
    ids, one = torch.zeros(9, 1, dtype=torch.int32, device="cuda"), torch.ones(9, 1, device="cuda")
    got = forward(be, layer, q, s, ids, one, torch.zeros(9, 512, device="cuda"))
    # the 32-bit gated product is a few roundings off, which moves int8 values next to borders by one step
    step = hs.double()[:, None] * (layer.raw[0][2][0].double().abs().amax(1) * layer.raw[0][2][1].double())
    assert bool(((got.double() - want.double()).abs() <= 4 * step).all())


def test_matrices_are_kept_alive_and_layers_share_them(be):
    a = Layer(be, 3, 64, 32, 0, seed=5)
    second = be.moe_i8_create(a.m._keep[0][::-1])
    q, s = rows_of(4, 64, 1)
    ids, coefs = routes(4, 3, 2, 1)
    space = torch.zeros(be.moe_i8_workspace_bytes(second, 4, 2), dtype=torch.uint8, device="cuda")
    x, y = forward(be, a, q, s, ids, coefs, torch.zeros(4, 64, device="cuda")), torch.zeros(4, 64, device="cuda")
    a.m.close()
    be.moe_i8_forward(second, q, s, 2 - ids, coefs, y, space)
    assert torch.equal(x, y)
