"""The half of a mixture-of-experts layer around its experts as a program runs it: the attention's output through its
projection with a bias, into the stream with the norms around it, routing, experts into the stream, the next norm.  Each
step is held to the 64-bit value of what it was given; the run is repeated as a captured graph, on another stream, and
in two contexts at once."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
EPS = 1e-5
U = 2.0 ** -24


@pytest.fixture(scope="module")
def be():
    import lbhip
    if not torch.cuda.is_available():
        pytest.fail("no GPU visible")
    b = lbhip.HipBackend(0)
    yield b
    b.close()


class Layer:
    def __init__(self, be, n, wide, experts, ffn, shared, seed):
        g = torch.Generator(device="cuda").manual_seed(seed)

        def mat(rows, k):
            w = torch.randint(-127, 128, (rows, k), dtype=torch.int8, device="cuda", generator=g)
            return w, (torch.rand(rows, device="cuda", generator=g) + 0.5) / (73 * k ** 0.5)

        self.n, self.wide, self.experts = n, wide, experts
        self.out_w, self.bias = mat(n, wide), 0.1 * torch.randn(n, device="cuda", generator=g)
        self.out = be.upload_i8(*self.out_w)
        self.post, self.pre, self.post2, self.pre2 = (torch.rand(n, device="cuda", generator=g) + 0.5 for _ in range(4))
        self.gate = torch.randn(1, n, device="cuda", generator=g)
        rng = np.random.default_rng(seed)
        self.router_w = (rng.standard_normal((experts, n)) / n ** 0.5).astype(np.float32)
        self.router_b = (0.1 * rng.standard_normal(experts)).astype(np.float32)
        self.router = be.router(self.router_w, self.router_b)
        pairs = [(be.upload_i8_gated(*mat(ffn, n), *mat(ffn, n)), be.upload_i8(*mat(n, ffn))) for _ in range(experts)]
        both = (be.upload_i8_gated(*mat(shared, n), *mat(shared, n)), be.upload_i8(*mat(n, shared)))
        self.moe = be.moe_i8_create(pairs, both)

    def buffers(self, be, tokens, ty, top_k):
        class B:
            pass
        b = B()
        new = lambda dt, *shape: torch.zeros(*shape, dtype=dt, device="cuda")   # noqa: E731
        b.q0, b.s0 = new(torch.int8, tokens, self.wide), new(torch.float32, tokens)
        b.o, b.h1, b.h2 = new(ty, tokens, self.n), new(ty, tokens, self.n), new(ty, tokens, self.n)
        b.v, b.q1, b.s1 = new(torch.float32, tokens, self.n), new(torch.int8, tokens, self.n), new(torch.float32, tokens)
        b.ids, b.coefs = new(torch.int32, tokens, top_k), new(torch.float32, tokens, top_k)
        b.y, b.q2, b.s2 = new(torch.float32, tokens, self.n), new(torch.int8, tokens, self.n), new(torch.float32, tokens)
        b.space_p = new(torch.uint8, be.gemm_i8_workspace_bytes(self.out, tokens))
        b.space_r = new(torch.uint8, be.route_rows_workspace_bytes(self.router, tokens))
        b.space_m = new(torch.uint8, be.moe_i8_workspace_bytes(self.moe, tokens, top_k))
        return b

    def run(self, be, attended, hidden, b):
        gate = self.gate.to(hidden.dtype)
        be.quantize_i8_rows(attended, b.q0, b.s0)
        be.gemm_i8_act(self.out, b.q0, b.s0, b.o, "none", b.space_p, bias=self.bias)
        be.block_norm_rows(b.o, hidden, b.h1, post_weight=self.post, post_eps=EPS, gate=gate, gate_act="sigmoid", scale=0.5,
                           weight=self.pre, eps=EPS, y=b.v, q=b.q1, scales=b.s1)
        be.route_rows(self.router, b.v, b.ids, b.coefs, b.space_r, mode=1, weight_scale=2.5)
        be.moe_i8_forward(self.moe, b.q1, b.s1, b.ids, b.coefs, b.y, b.space_m)
        be.block_norm_rows(b.y.to(hidden.dtype), b.h1, b.h2, post_weight=self.post2, post_eps=EPS, weight=self.pre2, eps=EPS,
                           q=b.q2, scales=b.s2)


NAMES = ("q0", "s0", "o", "h1", "v", "q1", "s1", "ids", "coefs", "y", "h2", "q2", "s2")


def stream_rows(tokens, layer, ty, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return ((torch.randn(tokens, layer.wide, device="cuda", generator=g)).to(ty),
            (2 * torch.randn(tokens, layer.n, device="cuda", generator=g)).to(ty))


@pytest.mark.parametrize("tokens,n,wide,experts,ffn,shared,top_k", [
    (1, 512, 1024, 8, 256, 512, 2), (6, 256, 300, 40, 96, 33, 6), (16, 768, 512, 12, 520, 64, 4), (50, 512, 768, 20, 128, 256, 8)])
@pytest.mark.parametrize("ty", [torch.float32, torch.bfloat16])
def test_each_step(be, tokens, n, wide, experts, ffn, shared, top_k, ty):
    la = Layer(be, n, wide, experts, ffn, shared, seed=n)
    attended, hidden = stream_rows(tokens, la, ty, tokens)
    b = la.buffers(be, tokens, ty, top_k)
    la.run(be, attended, hidden, b)
    torch.cuda.synchronize()
    half = 0.0 if ty == torch.float32 else torch.finfo(ty).eps / 2

    def rows8(v, q, s):
        scale = (v.abs().amax(1) / 127).float()
        assert torch.equal(scale, s)
        assert torch.equal(torch.round(v / scale.double()[:, None]).to(torch.int8), q)

    def norm(v, w):
        return v * w.double() / torch.sqrt((v * v).mean(1, keepdim=True) + EPS)

    rows8(attended.double(), b.q0, b.s0)
    p = (b.q0.double() @ la.out_w[0].double().t().contiguous()) * b.s0.double()[:, None] * la.out_w[1].double()
    o = p + la.bias.double()
    assert bool(((b.o.double() - o).abs() <= (3.001 * U * p.abs() + 2.001 * U * o.abs()) * (1 + half) + o.abs() * half * 1.0001 + 1e-37).all())
    moved = 0.5 * norm(b.o.double(), la.post) * torch.sigmoid(la.gate.to(ty).double())
    h1 = hidden.double() + moved
    assert bool(((b.h1.double() - h1).abs() <= h1.abs() * (U + half) * 1.0001 + moved.abs() * 2.0 ** -38).all())
    v = norm(b.h1.double(), la.pre)
    assert bool(((b.v.double() - v).abs() <= v.abs() * U * 1.0001).all())
    rows8(v, b.q1, b.s1)
    l = b.v.double().cpu().numpy() @ la.router_w.astype(np.float64).T
    sig = 1 / (1 + np.exp(-l))
    ids = np.sort(np.argsort(-(sig + la.router_b), axis=1, kind="stable")[:, :top_k], axis=1)
    np.testing.assert_array_equal(b.ids.cpu().numpy(), ids)
    c = np.take_along_axis(sig, ids, 1)
    np.testing.assert_allclose(b.coefs.cpu().numpy(), 2.5 * c / c.sum(1, keepdims=True), rtol=2.0 ** -23.9)
    y2 = b.y.to(ty).double()
    h2 = b.h1.double() + norm(y2, la.post2)
    assert bool(((b.h2.double() - h2).abs() <= h2.abs() * (U + half) * 1.0001 + 1e-37).all())
    rows8(norm(b.h2.double(), la.pre2), b.q2, b.s2)


@pytest.mark.parametrize("tokens,top_k", [(1, 4), (5, 6), (40, 6)])
def test_captured_layer_replays(be, tokens, top_k):
    """The run in a graph, replayed with new inputs, eager work and synchronizations between the replays."""
    ty = torch.bfloat16
    la = Layer(be, 512, 300, 16, 160, 96, seed=3)
    attended, hidden = stream_rows(tokens, la, ty, 0)
    b, e = la.buffers(be, tokens, ty, top_k), la.buffers(be, tokens, ty, top_k)
    stream, before = torch.cuda.Stream(), torch.cuda.current_stream()
    stream.wait_stream(before)
    be.set_stream(stream)
    try:
        with torch.cuda.stream(stream):
            la.run(be, attended, hidden, b)
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            la.run(be, attended, hidden, b)
    finally:
        be.set_stream(before)
    for i in range(4):
        na, nh = stream_rows(tokens, la, ty, 10 + i)
        attended.copy_(na), hidden.copy_(nh)
        for name in NAMES:
            getattr(b, name).zero_()
        la.run(be, na, nh, e)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for name in NAMES:
            assert torch.equal(getattr(b, name), getattr(e, name)), (i, name)


def test_two_contexts_at_once(be):
    """Two contexts on two streams, each with its own buffers, over the same weights, and two captured graphs."""
    import lbhip
    la = Layer(be, 512, 512, 24, 256, 128, seed=5)
    inputs = [stream_rows(t, la, torch.float32, t) for t in (7, 60)]
    want = []
    for x in inputs:
        b = la.buffers(be, x[0].shape[0], torch.float32, 6)
        la.run(be, *x, b)
        want.append(b)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    bes = [lbhip.HipBackend(0, stream=s) for s in streams]
    got = [la.buffers(bes[i], x[0].shape[0], torch.float32, 6) for i, x in enumerate(inputs)]
    torch.cuda.synchronize()
    for _ in range(10):
        for i, x in enumerate(inputs):
            with torch.cuda.stream(streams[i]):
                la.run(bes[i], *x, got[i])
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        for name in NAMES:
            assert torch.equal(getattr(a, name), getattr(b, name)), name
    graphs = []
    for i, x in enumerate(inputs):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=streams[i]):
            la.run(bes[i], *x, got[i])
        graphs.append(g)
    for _ in range(8):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i].h2.zero_()
                graphs[i].replay()
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        for name in NAMES:
            assert torch.equal(getattr(a, name), getattr(b, name)), name
    for c in bes:
        c.close()


def test_empty_calls_leave_everything(be):
    """No token: nothing happens, with empty tensors (whose address is null) as with none."""
    la = Layer(be, 256, 64, 3, 32, 16, seed=1)
    b = la.buffers(be, 0, torch.float32, 2)
    la.run(be, torch.zeros(0, 64, device="cuda"), torch.zeros(0, 256, device="cuda"), b)
    torch.cuda.synchronize()


def test_experts_from_packed_matrices(be):
    """int8 experts made from uploaded K-quant and IQ matrices, as a model's are."""
    from lbhip import synth
    experts, n, ffn = 4, 512, 256
    pairs = []
    for e in range(experts):
        g, u = (be.upload(synth.IQ2_S, ffn, n, synth.random_matrix(synth.IQ2_S, ffn, n, 10 * e + i)) for i in range(2))
        d = be.upload(synth.IQ3_S, n, ffn, synth.random_matrix(synth.IQ3_S, n, ffn, 10 * e + 2))
        pairs.append((be.i8_from_packed(g, u), be.i8_from_packed(d)))
    moe = be.moe_i8_create(pairs)
    x = torch.randn(3, n, device="cuda")
    q, s = torch.zeros(3, n, dtype=torch.int8, device="cuda"), torch.zeros(3, device="cuda")
    be.quantize_i8_rows(x, q, s)
    ids = torch.tensor([[0, 2], [3, 1], [2, 3]], dtype=torch.int32, device="cuda")
    coefs = torch.rand(3, 2, device="cuda")
    y = torch.zeros(3, n, device="cuda")
    be.moe_i8_forward(moe, q, s, ids, coefs, y, torch.zeros(be.moe_i8_workspace_bytes(moe, 3, 2), dtype=torch.uint8, device="cuda"))
    torch.cuda.synchronize()
    want = torch.zeros(3, n, dtype=torch.float64)
    for t in range(3):
        for k in range(2):
            pair, down = pairs[int(ids[t, k])]
            (gw, gs), (uw, us), (dw, ds) = pair.read(0), pair.read(1), down.read()
            xq, xs = q[t].cpu().numpy().astype(np.float64), float(s[t])
            g, u = gw.astype(np.float64) @ xq * xs * gs, uw.astype(np.float64) @ xq * xs * us
            h = (g / (1 + np.exp(-g)) * u).astype(np.float32).astype(np.float64)
            hs = float(np.float32(np.abs(h).max() / 127))
            want[t] += torch.from_numpy(float(coefs[t, k]) * (dw.astype(np.float64) @ np.rint(h / hs)) * hs * ds)
    assert bool(((y.cpu().double() - want).abs() <= want.abs() * U * 1.0001 + 1e-12).all())
