"""The scale of a block's output in lbh_block_norm_rows.  It multiplies 1 / sqrt(mean + post_eps) first, which is at most 2^537
(post_eps is at least 2^-1074): a scale beyond the float range could make that infinite, and an element that is zero NaN
where its formula is the hidden state.  Such scales are refused, as lbh_gemm_i8_act refuses them."""
import pytest

from test_layer_refusals import ctx, norm   # noqa: F401 (ctx: a fixture)

FLT_MAX = (2.0 - 2.0 ** -23) * 2.0 ** 127


@pytest.mark.parametrize("scale", [1e39, -1e39, FLT_MAX * (1 + 2.0 ** -52), 1.7e308])
def test_scales_beyond_the_float_range_are_refused(ctx, scale):   # noqa: F811
    assert norm(ctx, scale=scale)[0] == "InvalidParameter"
    assert norm(ctx, scale=scale, pw=0)[0] == "InvalidParameter"


@pytest.mark.parametrize("scale", [FLT_MAX, -FLT_MAX, 0.0, 5e-324])
def test_scales_within_it_are_not(ctx, scale):   # noqa: F811
    assert norm(ctx, scale=scale, rows=0)[0] == "Ok"


@pytest.mark.gpu
@pytest.mark.parametrize("n", [60, 515, 4096])
def test_zeros_stay_zeros_under_the_largest_scale(n):
    torch = pytest.importorskip("torch")
    import lbhip
    if not torch.cuda.is_available():
        pytest.fail("no GPU visible")
    be = lbhip.HipBackend(0)
    hidden, one = torch.randn(3, n, device="cuda"), torch.ones(n, device="cuda")
    block, out = torch.zeros(3, n, device="cuda"), torch.zeros(3, n, device="cuda")
    block[1] = -1.0   # normed to -1 and then scaled: the lowest float and beyond
    be.block_norm_rows(block, hidden, out, post_weight=one, post_eps=1e-300, scale=FLT_MAX)
    torch.cuda.synchronize()
    assert torch.equal(out[0], hidden[0]) and torch.equal(out[2], hidden[2])
    assert bool((out[1] <= -FLT_MAX * (1 - 2.0 ** -23)).all())
    be.close()
