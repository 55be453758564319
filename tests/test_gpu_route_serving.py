"""Routing as a server calls it: one workspace for every batch up to the largest."""
import numpy as np
import pytest

from test_gpu_route_rows import check, oracle

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


def routed(be, r, x, space, top_k, mode):
    n = x.shape[0]
    ids, coefs = torch.zeros(n, top_k, dtype=torch.int32, device="cuda"), torch.zeros(n, top_k, device="cuda")
    logits = torch.zeros(n, r.n_experts, device="cuda")
    be.route_rows(r, x, ids, coefs, space, mode=mode, logits=logits)
    torch.cuda.synchronize()
    return ids.cpu().numpy(), coefs.cpu().numpy(), logits.cpu().numpy()


@pytest.mark.parametrize("most", [90, 256, 300, 1100])
def test_one_workspace_for_every_batch(be, most):
    rng = np.random.default_rng(most)
    w, bias = rng.standard_normal((40, 512)).astype(np.float32), rng.standard_normal(40).astype(np.float32)
    r = be.router(w, bias)
    space = torch.zeros(be.route_rows_workspace_bytes_up_to(r, most), dtype=torch.uint8, device="cuda")
    x = torch.from_numpy(rng.standard_normal((most, 512)).astype(np.float32)).cuda()
    for n in {most, 1, most // 2, *(k for k in (75, 76, 255, 256, 257) if k <= most)}:
        check(routed(be, r, x[:n], space, 5, 1), oracle(x[:n], w, bias, 5, 1, 1.0))


@pytest.mark.parametrize("mode", [0, 1])
@pytest.mark.parametrize("rows", [1, 300])
def test_experts_masked_by_the_lowest_float(be, rows, mode):
    """A selection bias of the lowest float takes an expert out while enough others are left: a score stays finite, and
    the masked ones tie below all others (mode 1; mode 0 has no bias)."""
    rng = np.random.default_rng(rows)
    w = rng.standard_normal((30, 512)).astype(np.float32)
    bias = (0.1 * rng.standard_normal(30)).astype(np.float32)
    masked = np.arange(30) % 3 == 0
    bias[masked] = np.finfo(np.float32).min
    r = be.router(w, bias)
    x = torch.from_numpy(rng.standard_normal((rows, 512)).astype(np.float32)).cuda()
    space = torch.zeros(be.route_rows_workspace_bytes_up_to(r, rows), dtype=torch.uint8, device="cuda")
    for top_k in (4, 16):
        got = routed(be, r, x, space, top_k, mode)
        check(got, oracle(x, w, bias, top_k, mode, 1.0))
        if mode:
            assert not masked[got[0]].any()
    only = np.where(np.arange(30) == 7, bias, np.finfo(np.float32).min).astype(np.float32)
    r = be.router(w, only)
    got = routed(be, r, x, space, 3, 1)
    np.testing.assert_array_equal(got[0], np.tile([0, 1, 7], (rows, 1)))
    check(got, oracle(x, w, only, 3, 1, 1.0))
