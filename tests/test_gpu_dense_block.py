"""A dense feed-forward block in 8-bit integers as a program runs it: norm with the residual, the gated product, the
quantization of its rows, the product into the residual.  Each call is held to the 64-bit value of what it was given;
the run is repeated as a captured graph, on other streams, and in two contexts at once."""
import numpy as np
import pytest

from lbhip import synth

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


class Block:
    """Weights of one block, and the buffers of one call in flight."""

    def __init__(self, be, hidden, ffn, seed):
        g = torch.Generator(device="cuda").manual_seed(seed)

        def mat(rows, k):
            w = torch.randint(-127, 128, (rows, k), dtype=torch.int8, device="cuda", generator=g)
            return w, (torch.rand(rows, device="cuda", generator=g) + 0.5) / (73 * k ** 0.5)

        self.gate, self.up, self.down = mat(ffn, hidden), mat(ffn, hidden), mat(hidden, ffn)
        self.weight = torch.rand(hidden, device="cuda", generator=g) + 0.5
        self.pair, self.m = be.upload_i8_gated(*self.gate, *self.up), be.upload_i8(*self.down)
        self.hidden, self.ffn = hidden, ffn

    def buffers(self, be, tokens, ty):
        class B:
            pass
        b = B()
        b.after = torch.zeros(tokens, self.hidden, dtype=ty, device="cuda")
        b.q = torch.zeros(tokens, self.hidden, dtype=torch.int8, device="cuda")
        b.h = torch.zeros(tokens, self.ffn, dtype=ty, device="cuda")
        b.hq = torch.zeros(tokens, self.ffn, dtype=torch.int8, device="cuda")
        b.s, b.hs = torch.zeros(tokens, device="cuda"), torch.zeros(tokens, device="cuda")
        b.out = torch.zeros(tokens, self.hidden, dtype=ty, device="cuda")
        size = max(be.gemm_i8_workspace_bytes(x, tokens) for x in (self.pair, self.m))
        b.space = torch.zeros(size, dtype=torch.uint8, device="cuda")
        return b

    def run(self, be, x, delta, b):
        be.rms_norm_i8_rows(x, self.weight, EPS, b.q, b.s, delta=delta, hidden_out=b.after)
        be.gemm_i8_swiglu(self.pair, b.q, b.s, b.h, b.space)
        be.quantize_i8_rows(b.h, b.hq, b.hs)
        be.gemm_i8(self.m, b.hq, b.hs, b.out, b.space, residual=b.after)


def stream_rows(tokens, n, ty, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [(torch.randn(tokens, n, device="cuda", generator=g) * 2).to(ty) for _ in range(2)]


@pytest.mark.parametrize("tokens,hidden,ffn", [(1, 512, 1536), (9, 256, 700), (40, 1040, 520), (150, 300, 333),
                                               (300, 512, 1100)])
@pytest.mark.parametrize("ty", [torch.float32, torch.bfloat16])
def test_each_step_of_the_block(be, tokens, hidden, ffn, ty):
    blk = Block(be, hidden, ffn, seed=hidden)
    x, delta = stream_rows(tokens, hidden, ty, tokens)
    b = blk.buffers(be, tokens, ty)
    blk.run(be, x, delta, b)
    torch.cuda.synchronize()
    half = 0.0 if ty == torch.float32 else torch.finfo(ty).eps / 2

    def prod(q, s, m):
        return (q.double() @ m[0].double().t().contiguous()) * s.double()[:, None] * m[1].double()

    after = (x.float() + delta.float()).to(ty)
    assert torch.equal(after, b.after)
    d = after.double()
    v = d * blk.weight.double() / torch.sqrt((d * d).mean(1, keepdim=True) + EPS)
    for rows, q, s in ((v, b.q, b.s), (b.h.double(), b.hq, b.hs)):
        scale = (rows.abs().amax(1) / 127).float()
        assert torch.equal(scale, s)
        assert torch.equal(torch.round(rows / scale.double()[:, None]).to(torch.int8), q)
    g, u = prod(b.q, b.s, blk.gate), prod(b.q, b.s, blk.up)
    h = g * torch.sigmoid(g) * u
    off = h.abs() * (3 * (1 + g.abs()) + 8) * 1.01 * U
    assert bool(((b.h.double() - h).abs() <= off * (1 + half) + h.abs() * half * 1.0001 + 1e-37).all())
    p = prod(b.hq, b.hs, blk.down)
    y = p + after.double()
    off = p.abs() * 3.001 * U * (1 + U) + y.abs() * U
    assert bool(((b.out.double() - y).abs() <= off * (1 + half) + y.abs() * half * 1.0001 + 1e-37).all())


@pytest.mark.parametrize("tokens,hidden,ffn", [(1, 512, 1024), (20, 500, 333), (200, 512, 600)])
def test_captured_block_replays(be, tokens, hidden, ffn):
    """The block in a graph, replayed with new inputs, eager work and synchronizations between the replays."""
    ty = torch.bfloat16
    blk = Block(be, hidden, ffn, seed=3)
    x, delta = stream_rows(tokens, hidden, ty, 0)
    b, e = blk.buffers(be, tokens, ty), blk.buffers(be, tokens, ty)
    stream, before = torch.cuda.Stream(), torch.cuda.current_stream()
    stream.wait_stream(before)
    be.set_stream(stream)
    try:
        with torch.cuda.stream(stream):
            blk.run(be, x, delta, b)
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            blk.run(be, x, delta, b)
    finally:
        be.set_stream(before)
    for i in range(4):
        nx, nd = stream_rows(tokens, hidden, ty, 10 + i)
        x.copy_(nx), delta.copy_(nd)
        for t in (b.out, b.h, b.q, b.hq):
            t.zero_()
        blk.run(be, nx, nd, e)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for name in ("after", "q", "s", "h", "hq", "hs", "out"):
            assert torch.equal(getattr(b, name), getattr(e, name)), (i, name)


def test_two_contexts_at_once(be):
    """Two contexts on two streams, each with its own buffers, over the same weights."""
    import lbhip
    ty = torch.float32
    blk = Block(be, 768, 1200, seed=5)
    inputs = [stream_rows(37 + 60 * i, 768, ty, i) for i in range(2)]
    want = []
    for x, d in inputs:
        b = blk.buffers(be, x.shape[0], ty)
        blk.run(be, x, d, b)
        want.append(b)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    bes = [lbhip.HipBackend(0, stream=s) for s in streams]
    got = [blk.buffers(bes[i], x.shape[0], ty) for i, (x, _) in enumerate(inputs)]
    torch.cuda.synchronize()
    for _ in range(20):
        for i, (x, d) in enumerate(inputs):
            blk.run(bes[i], x, d, got[i])
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        assert torch.equal(a.out, b.out) and torch.equal(a.h, b.h)
    for c in bes:
        c.close()


def test_block_from_packed_weights_next_to_the_q8_k_path(be):
    """One normed row through both of the framework's paths: the Q8_K matvec of a Q5_K matrix and the int8 product of
    its int8 form.  Each path rounds the row and the weights on its own, by at most half a step of its scales."""
    rows, k = 512, 1024
    raw = synth.random_matrix(synth.Q5_K, rows, k, 9)
    m = be.upload(synth.Q5_K, rows, k, raw)
    m8 = be.i8_from_packed(m)
    x, delta = stream_rows(1, k, torch.float32, 7)
    weight = torch.ones(k, device="cuda")
    enc = torch.zeros(k // 256 * 292, dtype=torch.uint8, device="cuda")
    v = torch.zeros(1, k, device="cuda")
    be.rms_norm_q8_k_rows(x, weight, EPS, enc, y=v, delta=delta)
    y = torch.zeros(rows, device="cuda")
    be.gemv_q8_k(m, enc, y)
    q, s = torch.zeros(1, k, dtype=torch.int8, device="cuda"), torch.zeros(1, device="cuda")
    be.rms_norm_i8_rows(x, weight, EPS, q, s, delta=delta)
    y8 = torch.zeros(1, rows, device="cuda")
    be.gemm_i8(m8, q, s, y8)
    f = torch.zeros(rows, device="cuda")
    be.gemv_dequant_into(m, v[0], f)               # the decoded weights on the float row
    torch.cuda.synchronize()
    w8, ws = m8.read()
    absv, absw = np.abs(v[0].cpu().numpy().astype(np.float64)), np.abs(w8.astype(np.float64)) * ws[:, None]
    d8 = enc.cpu().numpy().reshape(-1, 292)[:, :4].copy().view(np.float32).reshape(-1)
    step_q = np.repeat(np.abs(d8.astype(np.float64)), 256)          # Q8_K may round by a whole step at -127 / max
    step_i = float(s[0])
    wide = absw + ws[:, None] / 2                                   # |decoded weight| is at most this
    tiny = (wide * absv).sum(1) * k * 2.0 ** -23                    # the sequential 32-bit sums
    off_q = (wide * step_q).sum(1) + tiny
    off_i = (wide * step_i / 2).sum(1) + (ws[:, None] / 2 * (absv + step_i / 2)).sum(1) + tiny
    fv = f.cpu().numpy().astype(np.float64)
    assert (np.abs(y.cpu().numpy() - fv) <= off_q).all()
    assert (np.abs(y8[0].cpu().numpy() - fv) <= off_i).all()


def test_empty_calls_leave_everything(be):
    """No token: nothing happens, with empty tensors (whose address is null) as with none."""
    blk = Block(be, 64, 48, seed=1)
    x, b = torch.zeros(0, 64, device="cuda"), blk.buffers(be, 0, torch.float32)
    blk.run(be, x, x, b)
    be.rms_norm_rows(x, blk.weight, EPS, torch.zeros_like(x))
    be.rms_norm_q8_k_rows(torch.zeros(0, 256, device="cuda"), torch.ones(256, device="cuda"), EPS,
                          torch.zeros(0, dtype=torch.uint8, device="cuda"))
    torch.cuda.synchronize()


def test_calls_on_a_side_stream_wait_for_their_own_stream_alone(be):
    """The context's stream orders the work: a run on a side stream over inputs written there just before."""
    ty, tokens = torch.float32, 130
    blk = Block(be, 512, 640, seed=6)
    x, d = stream_rows(tokens, 512, ty, 9)
    want, got = blk.buffers(be, tokens, ty), blk.buffers(be, tokens, ty)
    blk.run(be, x, d, want)
    torch.cuda.synchronize()
    side, before = torch.cuda.Stream(), torch.cuda.current_stream()
    be.set_stream(side)
    try:
        with torch.cuda.stream(side):
            a, c = torch.zeros_like(x), torch.zeros_like(d)
            for _ in range(5):
                a.copy_(x), c.copy_(d)
                blk.run(be, a, c, got)
                a.zero_()
        side.synchronize()
    finally:
        be.set_stream(before)
    assert torch.equal(want.out, got.out) and torch.equal(want.hq, got.hq)


def test_two_graphs_with_workspaces_of_their_own(be):
    """Rows off 16 bytes go through the workspace: two captured runs, each with its own, replayed on two streams at once."""
    import lbhip
    ty, tokens = torch.float32, 24
    blk = Block(be, 300, 333, seed=8)
    runs = []
    for i in range(2):
        x, d = stream_rows(tokens, 300, ty, 20 + i)
        want, b, stream = blk.buffers(be, tokens, ty), blk.buffers(be, tokens, ty), torch.cuda.Stream()
        blk.run(be, x, d, want)
        torch.cuda.synchronize()
        own = lbhip.HipBackend(0, stream=stream)
        with torch.cuda.stream(stream):
            blk.run(own, x, d, b)
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            blk.run(own, x, d, b)
        runs.append((graph, stream, want, b, own, x, d))
    for _ in range(10):
        for graph, stream, _, b, *_ in runs:
            with torch.cuda.stream(stream):
                b.out.zero_()
                graph.replay()
    torch.cuda.synchronize()
    for _, _, want, b, own, *_ in runs:
        assert torch.equal(want.out, b.out)
        own.close()
