"""The experts of layers of more than 2048 channels, whose down product has sixteen channels a workgroup, against the 64-bit
implementation of test_gpu_moe_i8 (which holds narrower layers to it, eight channels a workgroup): with a shared
expert, with int8 rows made in the down product, by a launch of their own and behind a plan, and with the
most rows that a workgroup holds sums of."""
import threading

import pytest

from test_gpu_moe_i8 import TYPES, Layer, check, forward, oracle, routes, rows_of

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


# (tokens, experts, top_k, n, ffn, shared)
SHAPES = [(1, 6, 2, 2049, 300, 500), (1, 9, 8, 4096, 256, 1024), (2, 5, 4, 2064, 96, 33),         # up to 16 steps of 512
          (5, 20, 8, 2049, 130, 256), (3, 6, 4, 4096, 1536, 2048), (8, 10, 8, 2064, 600, 40),     # up to 64 slots
          (16, 12, 8, 2064, 64, 48), (40, 7, 3, 2049, 200, 96), (100, 9, 4, 4096, 96, 80), (65, 4, 2, 2560, 520, 0),
          (256, 12, 8, 2064, 32, 48), (128, 20, 16, 2049, 33, 16), (256, 3, 1, 5000, 16, 20)]     # the first: every row


@pytest.mark.parametrize("tokens,experts,top_k,n,ffn,shared", SHAPES)
def test_wide_layers(be, tokens, experts, top_k, n, ffn, shared):
    layer = Layer(be, experts, n, ffn, shared, seed=n + ffn)
    q, s = rows_of(tokens, n, tokens)
    ids, coefs = routes(tokens, experts, top_k, tokens, hot=1)
    want = oracle(layer, q, s, ids, coefs, None)
    for ty in TYPES:
        res = torch.randn(tokens, n, device="cuda").to(ty)
        y = torch.full((tokens + 1, n), 3.0, dtype=ty, device="cuda")
        check(forward(be, layer, q, s, ids, coefs, y[:tokens], res), (want[0] + res.double(), want[1] + res.double().abs()))
        check(forward(be, layer, q, s, ids, coefs, y[:tokens]), want)
        assert bool((y[tokens] == 3.0).all())


@pytest.mark.parametrize("n", [2049, 2064])
@pytest.mark.parametrize("tokens", [1, 7, 40, 150])
def test_hot_experts_repeated_experts_and_empty_slots(be, tokens, n):
    layer = Layer(be, 7, n, 96, 64, seed=1)
    q, s = rows_of(tokens, n, 2)
    _, coefs = routes(tokens, 7, 4, 3)
    cases = [torch.full((tokens, 4), 6), torch.tensor([3, 3, 1, 3]).repeat(tokens, 1), torch.full((tokens, 4), -1),
             torch.tensor([7, 2, 2 ** 31 - 1, -5]).repeat(tokens, 1), torch.arange(4 * tokens).reshape(tokens, 4) % 9 - 1]
    for ids in cases:
        ids = ids.to(torch.int32).cuda()
        c = torch.where((ids < 0) | (ids > 6), float("nan"), coefs)   # an empty slot's is not used
        res = torch.randn(tokens, n, device="cuda")
        want = oracle(layer, q, s, ids, torch.nan_to_num(c), res)
        check(forward(be, layer, q, s, ids, c, torch.zeros(tokens, n, device="cuda"), res), want)


def test_a_token_s_bits_do_not_depend_on_the_batch(be):
    n = 2320
    layer = Layer(be, 24, n, 512, 256, seed=4)
    q, s = rows_of(200, n, 5)
    ids, coefs = routes(200, 24, 6, 6, hot=1)
    res = torch.randn(200, n, device="cuda")
    whole = forward(be, layer, q, s, ids, coefs, torch.zeros(200, n, device="cuda"), res)
    check(whole, oracle(layer, q, s, ids, coefs, res))
    for at, count in ((0, 1), (77, 2), (10, 10), (60, 11), (100, 33), (3, 90)):
        part = [t[at:at + count].contiguous() for t in (q, s, ids, coefs)]
        assert torch.equal(forward(be, layer, *part, torch.zeros(count, n, device="cuda"), res[at:at + count]), whole[at:at + count])
    order = torch.randperm(200, device="cuda")
    again = forward(be, layer, q[order], s[order], ids[order], coefs[order], torch.zeros(200, n, device="cuda"), res[order])
    assert torch.equal(again, whole[order])


@pytest.mark.parametrize("tokens", [1, 2, 30])
def test_in_place_strides_and_odd_addresses(be, tokens):
    n = 2061
    layer = Layer(be, 6, n, 72, 40, seed=3)
    q, s = rows_of(tokens, n, 4)
    ids, coefs = routes(tokens, 6, 2, 5)
    res = torch.randn(tokens, n, device="cuda").bfloat16()
    want = forward(be, layer, q, s, ids, coefs, torch.zeros_like(res), res)
    check(want, oracle(layer, q, s, ids, coefs, res))
    wide = torch.full((tokens, n + 133), 77, dtype=torch.int8, device="cuda")
    wide[:, 5:n + 5] = q
    buf = torch.full((tokens, n + 100), 9.0, dtype=torch.bfloat16, device="cuda")
    view = buf[:, 3:n + 3]
    view.copy_(res)
    forward(be, layer, wide[:, 5:n + 5], s, ids, coefs, view, view)
    assert torch.equal(view, want)
    assert bool((buf[:, :3] == 9).all()) and bool((buf[:, n + 3:] == 9).all())


def test_the_most_rows_captured(be):
    """2048 slots and 256 shared rows in a graph, replayed with new inputs, eager work and synchronizations between."""
    n, tokens = 2064, 256
    layer = Layer(be, 12, n, 32, 48, seed=6)
    q, s = rows_of(tokens, n, 1)
    ids, coefs = routes(tokens, 12, 8, 1)
    y, e = (torch.zeros(tokens, n, device="cuda") for _ in range(2))
    space, other = (torch.zeros(be.moe_i8_workspace_bytes(layer.m, tokens, 8), dtype=torch.uint8, device="cuda") for _ in range(2))
    stream, before = torch.cuda.Stream(), torch.cuda.current_stream()
    stream.wait_stream(before)
    be.set_stream(stream)
    try:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            be.moe_i8_forward(layer.m, q, s, ids, coefs, y, space)
    finally:
        be.set_stream(before)
    for i in range(4):
        nq, ns = rows_of(tokens, n, 10 + i)
        nids, nc = routes(tokens, 12, 8, 10 + i)
        for a, b in ((q, nq), (s, ns), (ids, nids), (coefs, nc)):
            a.copy_(b)
        y.zero_()
        be.moe_i8_forward(layer.m, nq, ns, nids, nc, e, other)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, e), i
    check(e, oracle(layer, nq, ns, nids, nc, None))


def test_two_threads_with_different_numbers_of_rows(be):
    """Two host threads, a context and a stream each, over one layer: calls whose sums take different amounts of LDS,
    both above what a launch has without asking."""
    import lbhip
    n, sizes = 2064, ((128, 16), (100, 12))
    layer = Layer(be, 20, n, 32, 48, seed=9)
    inputs, want = [], []
    for tokens, top_k in sizes:
        x = (*rows_of(tokens, n, tokens), *routes(tokens, 20, top_k, tokens))
        inputs.append(x)
        want.append(forward(be, layer, *x, torch.zeros(tokens, n, device="cuda")))
        check(want[-1], oracle(layer, *x, None))
    streams = [torch.cuda.Stream() for _ in sizes]
    bes = [lbhip.HipBackend(0, stream=st) for st in streams]
    got = [torch.zeros_like(w) for w in want]
    spaces = [torch.zeros(be.moe_i8_workspace_bytes(layer.m, *size), dtype=torch.uint8, device="cuda") for size in sizes]
    torch.cuda.synchronize()
    errors = []
    start = threading.Barrier(2)

    def calls(i):
        try:
            start.wait()
            for _ in range(200):
                bes[i].moe_i8_forward(layer.m, *inputs[i], got[i], spaces[i])
        except Exception as e:   # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=calls, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not errors, errors
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    for b in bes:
        b.close()
