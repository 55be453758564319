"""The int8 products with bias and activation in each tile form, where whole tiles lie inside the output (words of 16
bytes, residuals on their way ahead) and at ragged edges beside them: against the 64-bit values, and bit for bit against
the same call over rows at odd addresses, which takes every element by itself.

Tolerances (U = 2^-24): the argument's is test_gpu_i8_act's.  An activation of a float32 output is off by 16 U of its value
and 4 U for each unit of its exponent, as derived there.  Outputs of 16 bits leave out the second part of the
exponent and the reciprocal's step: the sigmoid's argument z has up to four roundings, its product with log2(e) and that
constant one each, 8 U |z| with the exponential's own; the normal distribution's tail has a^2 rounded once, its product with
the constant twice, 4 U a^2 / 2; the rest stays within 16 U of the value."""
import math

import numpy as np
import pytest

from test_gpu_i8_act import ACTS, Case, U, act64, check

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
TILES = range(6, 11)             # the numbers of the tile forms
TOKENS, ROWS, K = 300, 800, 512   # a tile of 256 x 256 (a pair's: of 128) lies inside, with ragged ones on both sides


@pytest.fixture(scope="module")
def be():
    import lbhip
    if not torch.cuda.is_available():
        pytest.fail("no GPU visible")
    b = lbhip.HipBackend(0)
    yield b
    b.close()


@pytest.fixture(scope="module")
def cases(be):
    return {gated: Case(be, TOKENS, ROWS, K, gated, 11 + gated, big=3.0) for gated in (False, True)}


def off_act(x, dx, name, wide):
    v, z = act64(x, name)
    z = z.clamp(max=128.0)   # beyond that the sigmoid is 1 or has gone to 0
    each = 4 * z if wide else 8 * z + (2 * x * x if name == "gelu" else 0)
    slope = 2 * x.abs() + dx if name == "relu2" else 1.13
    return v, slope * dx + v.abs() * U * (16 + each) + x.abs() * 2.0 ** -118


def want(c, act, bias, up_bias, scale, residual, wide):
    v, off = off_act(*c.arg(c.w, bias), act, wide)
    if c.up is not None:
        u, du = c.arg(c.up, up_bias)
        v, off = v * u, off * (u.abs() + du) + v.abs() * du + (v * u).abs() * 2 * U
    scale = float(np.float32(scale))
    y, off = v * scale, off * abs(scale) + (v * scale).abs() * 2 * U
    if residual is not None:
        y = y + residual.double()
        off = off + y.abs() * U
    return y, off * 1.001


def odd(t):
    """The same values from an odd element on."""
    buf = torch.zeros(t.numel() + 1, dtype=t.dtype, device="cuda")
    buf[1:] = t
    return buf[1:]


def rows_in(tokens, cols, pitch, at, ty):
    """(buffer, view of `cols` columns from column `at` on), rows behind the last token."""
    buf = torch.full((tokens + 3, pitch), 7.0, dtype=ty, device="cuda")
    return buf, buf[:tokens, at:at + cols]


def around_is_left_alone(buf, tokens, at, cols):
    rest = buf.clone()
    rest[:tokens, at:at + cols] = 7.0
    return bool((rest == 7.0).all())


@pytest.mark.parametrize("ty", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("kind", ["plain", "residual", "gated"])
@pytest.mark.parametrize("form", TILES)
def test_tiles(be, cases, form, kind, act, ty):
    c = cases[kind == "gated"]
    bias, up_bias = odd(c.bias), odd(c.up_bias) if kind == "gated" else None
    g = torch.Generator(device="cuda").manual_seed(form)
    res = (2 * torch.randn(TOKENS, ROWS, device="cuda", generator=g)).to(ty) if kind == "residual" else None
    outs = []
    try:
        be.set_tuning(be.TUNE_I8_FORM, form)
        for pitch, at in ((ROWS + 16, 0), (ROWS + 1, 1)):   # rows of whole words of 16 bytes; rows of none
            buf, y = rows_in(TOKENS, ROWS, pitch, at, ty)
            r = None
            if res is not None:
                r = rows_in(TOKENS, ROWS, pitch, at, ty)[1]
                r.copy_(res)
            be.gemm_i8_act(c.m, c.q, c.s, y, act, c.space, bias=bias, up_bias=up_bias, residual=r, scale=0.3)
            torch.cuda.synchronize()
            assert around_is_left_alone(buf, TOKENS, at, ROWS)
            outs.append(y)
    finally:
        be.set_tuning(be.TUNE_I8_FORM, 0)
    check(outs[0], *want(c, act, c.bias, up_bias, 0.3, res, ty == torch.float32))
    assert torch.equal(*outs)


@pytest.mark.parametrize("ty", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("form", TILES)
def test_residuals_in_place_inside_tiles(be, cases, form, ty):
    c = cases[False]
    res = torch.randn(TOKENS, ROWS, device="cuda").to(ty)
    y, both = torch.zeros_like(res), res.clone()
    try:
        be.set_tuning(be.TUNE_I8_FORM, form)
        be.gemm_i8_act(c.m, c.q, c.s, y, "gelu_tanh", c.space, bias=c.bias, residual=res, scale=-1.5)
        be.gemm_i8_act(c.m, c.q, c.s, both, "gelu_tanh", c.space, bias=c.bias, residual=both, scale=-1.5)
    finally:
        be.set_tuning(be.TUNE_I8_FORM, 0)
    assert torch.equal(y, both)
    check(y, *want(c, "gelu_tanh", c.bias, None, -1.5, res, ty == torch.float32))


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("act", ACTS)
def test_arguments_far_out_in_the_largest_tile(be, gated, act):
    """Every channel of a column of tiles has one argument, given as its bias: not finite, zero, far out."""
    values = [0.0, -0.0, 0.5, -0.5, 13.1, -13.1, 14.5, -14.5, 87.0, -87.0, 104.5, -104.5, 1e15, -1e15, float("nan"), float("inf")]
    n = 256
    zero, one = torch.zeros(n, 256, dtype=torch.int8, device="cuda"), torch.ones(n, device="cuda")
    m = be.upload_i8_gated(zero, one, zero, one) if gated else be.upload_i8(zero, one)
    bias = torch.tensor(values * (n // len(values)), device="cuda")
    q, s = torch.zeros(256, 256, dtype=torch.int8, device="cuda"), torch.ones(256, device="cuda")
    try:
        be.set_tuning(be.TUNE_I8_FORM, 10)
        for ty in (torch.float32, torch.float16, torch.bfloat16):
            y = torch.zeros(256, n, dtype=ty, device="cuda")
            be.gemm_i8_act(m, q, s, y, act, bias=bias, up_bias=one if gated else None)
            torch.cuda.synchronize()
            assert torch.equal(y[0].expand_as(y).nan_to_num(5.0), y.nan_to_num(5.0))
            assert torch.equal(y[0].view(-1, len(values))[0].expand(n // len(values), -1).nan_to_num(5.0), y[0].view(-1, len(values)).nan_to_num(5.0))
            got = y[0, :len(values)].double()
            assert math.isnan(got[-2].item()) and got[-1].item() == float("inf")
            x = bias[:len(values) - 2].double()
            v, off = off_act(x, torch.zeros_like(x), act, ty == torch.float32)
            half = 0.0 if ty == torch.float32 else torch.finfo(ty).eps / 2
            least = torch.finfo(ty).smallest_normal * (1 if ty == torch.float32 else torch.finfo(ty).eps) + 2.0 ** -126
            bad = (got[:-2] - v).abs() > off * (1 + half) + v.abs() * (half * 1.0001 + 2 * U) + least
            over = v.abs() > torch.finfo(ty).max
            assert not bool((bad & ~over).any()) and bool(torch.isinf(got[:-2][over]).all())
    finally:
        be.set_tuning(be.TUNE_I8_FORM, 0)


@pytest.mark.parametrize("form", [0, *range(1, 12)])
@pytest.mark.parametrize("ty", [torch.float16, torch.bfloat16])
def test_silu_of_a_pair_and_swiglu_in_16_bits(be, cases, form, ty):
    """One formula in two calls: both lie within 2^-16 of it (16 U and 8 U for each unit of an exponent |g| <= 30), far
    less than a step of 16 bits, so their outputs are the same or neighbours."""
    c = cases[True]
    a, b = (torch.zeros(TOKENS, ROWS, dtype=ty, device="cuda") for _ in range(2))
    g = c.arg(c.w, None)[0]
    near = g.abs() <= 30
    assert bool(near.float().mean() > 0.9)
    try:
        be.set_tuning(be.TUNE_I8_FORM, form)
        be.gemm_i8_swiglu(c.m, c.q, c.s, a, c.space)
        be.gemm_i8_act(c.m, c.q, c.s, b, "silu", c.space)
    finally:
        be.set_tuning(be.TUNE_I8_FORM, 0)
    # neighbours of one sign are one apart as integers; what may go to 0 lies below the type's steps
    small = (a.abs() < torch.finfo(ty).smallest_normal) & (b.abs() < torch.finfo(ty).smallest_normal)
    apart = (a.view(torch.int16).int() - b.view(torch.int16).int()).abs()
    assert bool((apart[near & ~small] <= 1).all())


@pytest.mark.parametrize("ty", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("kind", ["plain", "residual", "gated"])
def test_all_forms_give_the_same_bits(be, cases, kind, act, ty):
    c = cases[kind == "gated"]
    res = torch.randn(TOKENS, ROWS, device="cuda").to(ty) if kind == "residual" else None
    outs = []
    try:
        for form in range(12):
            be.set_tuning(be.TUNE_I8_FORM, form)
            y = torch.zeros(TOKENS, ROWS, dtype=ty, device="cuda")
            be.gemm_i8_act(c.m, c.q, c.s, y, act, c.space, bias=c.bias, up_bias=c.up_bias if kind == "gated" else None, residual=res,
                           scale=0.7)
            outs.append(y)
    finally:
        be.set_tuning(be.TUNE_I8_FORM, 0)
    assert [form for form, y in enumerate(outs) if not torch.equal(y, outs[0])] == []
