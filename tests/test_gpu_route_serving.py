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
