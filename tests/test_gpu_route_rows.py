"""Routing of a batch of rows against a plain 64-bit implementation: ids equal, coefficients and logits within their one
rounding to 32 bits (half a step, 2^-24 of the value) and what precedes it (2^-37 of the value: the exponentials are
good to 2^-39, a quotient has two of them; sums of 64-bit products are some 2^-50 of the terms' magnitudes off)."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def be():
    import lbhip
    if not torch.cuda.is_available():
        pytest.fail("no GPU visible")
    b = lbhip.HipBackend(0)
    yield b
    b.close()


def oracle(x, w, bias, top_k, mode, scale):
    """(ids, coefs, logits, the logits' terms) of rows x in 64 bits."""
    x, w = x.double().cpu().numpy(), w.astype(np.float64)
    l = x @ w.T
    with np.errstate(all="ignore"):
        s = 1 / (1 + np.exp(-l))
    score = s + bias if mode else l
    ids = np.sort(np.argsort(-score, axis=1, kind="stable")[:, :top_k], axis=1)
    best = np.take_along_axis(l, ids, 1)
    if mode:
        c = np.take_along_axis(s, ids, 1)
        c = c / np.maximum(c.sum(1, keepdims=True), 2.0 ** -14)
    else:
        c = np.exp(best - best.max(1, keepdims=True))
        c = c / c.sum(1, keepdims=True)
    return ids, c * scale, l, np.abs(x) @ np.abs(w).T


def route(be, r, x, top_k, mode, scale=1.0, want_logits=True):
    n = x.shape[0]
    ids = torch.full((n, top_k), -7, dtype=torch.int32, device="cuda")
    coefs, logits = torch.zeros(n, top_k, device="cuda"), torch.zeros(n, r.n_experts, device="cuda")
    space = torch.zeros(be.route_rows_workspace_bytes(r, n), dtype=torch.uint8, device="cuda")
    be.route_rows(r, x, ids, coefs, space, mode=mode, weight_scale=scale, logits=logits if want_logits else None)
    torch.cuda.synchronize()
    return ids.cpu().numpy(), coefs.cpu().numpy(), logits.cpu().numpy()


def check(got, want):
    ids, coefs, logits, terms = want
    np.testing.assert_array_equal(got[0], ids)
    step = 2.0 ** -24 + 2.0 ** -37
    np.testing.assert_array_less(np.abs(got[1] - coefs), np.abs(coefs) * step + 1e-44)
    np.testing.assert_array_less(np.abs(got[2] - logits), np.abs(logits) * step + terms * 2.0 ** -45 + 1e-44)


# (rows, experts, width, top_k): one row and many, either way of the sums, ragged tiles, every count of lanes' experts
SHAPES = [(1, 1, 256, 1), (1, 192, 4096, 8), (3, 7, 256, 7), (16, 16, 512, 16), (17, 65, 768, 2), (64, 128, 1024, 4),
          (65, 129, 1280, 6), (256, 33, 512, 5), (257, 256, 256, 16), (300, 192, 1792, 8), (1000, 40, 512, 3)]


@pytest.mark.parametrize("ty", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("mode", [0, 1])
@pytest.mark.parametrize("rows,experts,width,top_k", SHAPES)
def test_routes(be, rows, experts, width, top_k, mode, ty):
    g = np.random.default_rng(rows + experts)
    w = g.standard_normal((experts, width)).astype(np.float32) / np.float32(np.sqrt(width))
    bias = (0.2 * g.standard_normal(experts)).astype(np.float32)
    r = be.router(w, bias)
    x = torch.from_numpy(g.standard_normal((rows, width)).astype(np.float32)).cuda().to(TYPES[ty])
    check(route(be, r, x, top_k, mode, 2.5), oracle(x, w, bias, top_k, mode, 2.5))
    # rows apart, from an odd element on
    buf = torch.full((rows * (width + 3) + 8,), 50.0, dtype=TYPES[ty], device="cuda")
    view = buf[5:5 + rows * (width + 3)].view(rows, width + 3)[:, :width]
    view.copy_(x)
    a, b = route(be, r, x, top_k, mode, 2.5), route(be, r, view, top_k, mode, 2.5)
    assert all((u == v).all() for u, v in zip(a, b))


@pytest.mark.parametrize("mode", [0, 1])
def test_a_row_s_bits_do_not_depend_on_the_batch(be, mode):
    g = np.random.default_rng(5)
    w, bias = g.standard_normal((192, 2304)).astype(np.float32), g.standard_normal(192).astype(np.float32)
    r = be.router(w, bias)
    x = torch.from_numpy(g.standard_normal((700, 2304)).astype(np.float32)).cuda()
    whole = route(be, r, x, 8, mode)
    for at, n in ((0, 1), (399, 1), (100, 64), (37, 256), (300, 257)):
        part = route(be, r, x[at:at + n], 8, mode)
        assert all((u == v[at:at + n]).all() for u, v in zip(part, whole))


def test_ties_go_to_the_lower_id(be):
    """Experts of the same weights in a row, and selection by bias alone."""
    g = np.random.default_rng(1)
    w = np.repeat(g.standard_normal((4, 512)).astype(np.float32), 48, axis=0)
    w = w[np.arange(192).reshape(4, 48).T.reshape(-1)]   # expert e has the weights of e % 4
    bias = np.zeros(192, np.float32)
    r = be.router(w, bias)
    x = torch.from_numpy(g.standard_normal((70, 512)).astype(np.float32)).cuda()
    for mode in (0, 1):
        ids, coefs, logits = route(be, r, x, 6, mode)
        best = logits[:, :4].argmax(1)
        if mode == 0:
            np.testing.assert_array_equal(ids, best[:, None] + 4 * np.arange(6))
        # the logits reach 40 and more, where 1 / (1 + exp(-l)) is 1 in 64 bits: those of two groups tie too
        # (and where every one is far below 0 the coefficients are shares of the least sum, 2^-14)
        check((ids, coefs, logits), oracle(x, w, bias, 6, mode, 1.0))
    # zero rows: every logit is zero, every score the bias
    bias[[150, 30, 90]] = 1.0
    r = be.router(w, bias)
    zero = torch.zeros(3, 512, device="cuda")
    np.testing.assert_array_equal(route(be, r, zero, 5, 1)[0], np.tile([0, 1, 30, 90, 150], (3, 1)))
    np.testing.assert_array_equal(route(be, r, -zero, 3, 0)[0], np.tile([0, 1, 2], (3, 1)))


def test_scores_that_differ_in_their_last_bits(be):
    """Keys whose upper words agree: one element decides, far below the sum's 32 bits."""
    w = np.zeros((130, 256), np.float32)
    w[:, 0] = 1.0
    w[:, 1] = 2.0 ** -40
    order = np.random.default_rng(2).permutation(130)
    w[:, 1] *= 1 + order
    r = be.router(w)
    x = torch.ones(2, 256, device="cuda")
    want = np.sort(np.argsort(-order)[:9])
    np.testing.assert_array_equal(route(be, r, x, 9, 0)[0], np.tile(want, (2, 1)))
    np.testing.assert_array_equal(route(be, r, -x, 9, 0)[0], np.tile(np.sort(np.argsort(order)[:9]), (2, 1)))


def test_rows_that_are_not_finite_and_far_logits(be):
    g = np.random.default_rng(3)
    w, bias = g.standard_normal((20, 256)).astype(np.float32), g.standard_normal(20).astype(np.float32)
    for rows in (6, 300):
        r = be.router(w, bias)
        x = torch.from_numpy(g.standard_normal((rows, 256)).astype(np.float32)).cuda()
        x[1, 7], x[3, 200] = float("nan"), float("inf")
        x[4] *= 1e4                                  # logits of 10^5: exponentials at 0 and 1
        for mode in (0, 1):
            got = route(be, r, x, 4, mode)
            for t in (1, 3):
                np.testing.assert_array_equal(got[0][t], np.arange(4))
                assert np.isnan(got[1][t]).all()
            fine = [t for t in range(rows) if t not in (1, 3)]
            want = oracle(x[fine], w, bias, 4, mode, 1.0)
            np.testing.assert_array_equal(got[0][fine], want[0])
            np.testing.assert_array_less(np.abs(got[1][fine] - want[1]), want[1] * (2.0 ** -24 + 2.0 ** -37) + 1e-44)
    bias[2] = np.inf                                 # a bias that is not finite: no selection
    assert np.isnan(route(be, be.router(w, bias), x[5:6], 4, 1)[1]).all()
    assert np.isfinite(route(be, be.router(w, bias), x[5:6], 4, 0)[1]).all()


def test_without_logits(be):
    w = np.random.default_rng(4).standard_normal((30, 512)).astype(np.float32)
    r = be.router(w)
    x = torch.randn(9, 512, device="cuda")
    a, b = route(be, r, x, 3, 0), route(be, r, x, 3, 0, want_logits=False)
    assert (a[0] == b[0]).all() and (a[1] == b[1]).all() and not b[2].any()


def test_it_selects_as_the_batch_selection_does(be):
    """Where no two logits are near, the 32-bit batch selection over the same logits chooses the same experts."""
    g = np.random.default_rng(6)
    w, bias = g.standard_normal((64, 512)).astype(np.float32), g.standard_normal(64).astype(np.float32)
    r = be.router(w, bias)
    x = torch.from_numpy(g.standard_normal((50, 512)).astype(np.float32)).cuda()
    for mode in (0, 1):
        ids, coefs, logits = route(be, r, x, 8, mode)
        i2, c2 = torch.zeros(50, 8, dtype=torch.int32, device="cuda"), torch.zeros(50, 8, device="cuda")
        be.route_experts_batch(torch.from_numpy(logits).cuda(), 8, i2, c2, mode=mode, bias=torch.from_numpy(bias).cuda())
        np.testing.assert_array_equal(ids, i2.cpu().numpy())
        # The batch selection is given the logits rounded to 32 bits (U = 2^-24 of each) and rounds their differences:
        # an exponential's argument is off by U (|l| + |m| + |l - m|) <= 4 U max |l|, the sum's terms likewise, and its
        # exponential, sum and quotient round some 24 times.
        np.testing.assert_allclose(coefs, c2.cpu().numpy(), rtol=2.0 ** -24 * (8 * np.abs(logits).max() + 24))
