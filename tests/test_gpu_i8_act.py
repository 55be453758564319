"""int8 products with bias, activation, scale and residual against a plain 64-bit implementation.

The kernel works in float32 (U = 2^-24 a rounding): its argument x = product + bias is off by the product's conversion
and two scales and the addition, dx = 3 U |product| + U |x|; an activation passes dx on with its slope (at most 1.13; of
relu squared 2 |x|) and adds its own roundings: for the sigmoid and the normal distribution some 16 U of its value and
4 U for each unit of its exponent (the argument z of the sigmoid has up to four roundings), and |x| 2^-118 where they
go to 0.  The following products and the residual's addition round once each, and the type once more."""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
U = 2.0 ** -24
ACTS = ["none", "relu", "relu2", "silu", "gelu", "gelu_tanh"]
ROOT = math.sqrt(8.0 / math.pi)


@pytest.fixture(scope="module")
def be():
    import lbhip
    if not torch.cuda.is_available():
        pytest.fail("no GPU visible")
    b = lbhip.HipBackend(0)
    yield b
    b.close()


def act64(x, name):
    """(value, the size of the sigmoid's argument) in 64 bits."""
    zero = torch.zeros_like(x)
    if name == "silu":
        return x * torch.sigmoid(x), x.abs()
    if name == "gelu":
        return x * 0.5 * torch.special.erfc(-x / math.sqrt(2.0)), zero
    if name == "gelu_tanh":
        z = ROOT * (x + 0.044715 * x ** 3)
        return x * torch.sigmoid(z), z.abs()
    return {"none": x, "relu": x.clamp(min=0), "relu2": x.clamp(min=0) ** 2}[name], zero


def off_act(x, dx, name):
    v, z = act64(x, name)
    slope = 2 * x.abs() + dx if name == "relu2" else 1.13
    return v, slope * dx + v.abs() * U * (16 + 4 * z) + x.abs() * 2.0 ** -118


class Case:
    def __init__(self, be, tokens, rows, k, gated, seed, big=1.0):
        g = torch.Generator(device="cuda").manual_seed(seed)

        def mat():
            return (torch.randint(-127, 128, (rows, k), dtype=torch.int8, device="cuda", generator=g),
                    big * (torch.rand(rows, device="cuda", generator=g) + 0.5) / (73 * k ** 0.5))

        self.q = torch.randint(-127, 128, (tokens, k), dtype=torch.int8, device="cuda", generator=g)
        self.s = (torch.rand(tokens, device="cuda", generator=g) + 0.5) / 40
        self.w, self.up = mat(), mat() if gated else None
        self.bias, self.up_bias = (torch.randn(rows, device="cuda", generator=g) for _ in range(2))
        self.m = be.upload_i8_gated(*self.w, *self.up) if gated else be.upload_i8(*self.w)
        self.space = torch.zeros(be.gemm_i8_workspace_bytes(self.m, tokens), dtype=torch.uint8, device="cuda")

    def arg(self, w, bias):
        p = (self.q.double() @ w[0].double().t().contiguous()) * self.s.double()[:, None] * w[1].double()
        x = p if bias is None else p + bias.double()
        return x, 3.001 * U * p.abs() + U * x.abs()

    def want(self, act, bias, up_bias, scale, residual):
        v, off = off_act(*self.arg(self.w, bias), act)
        if self.up is not None:
            u, du = self.arg(self.up, up_bias)
            v, off = v * u, off * (u.abs() + du) + v.abs() * du + (v * u).abs() * 2 * U
        scale = float(np.float32(scale))
        y, off = v * scale, off * abs(scale) + (v * scale).abs() * 2 * U
        if residual is not None:
            y = y + residual.double()
            off = off + y.abs() * U
        return y, off * 1.001


def check(got, want, off):
    half = 0.0 if got.dtype == torch.float32 else torch.finfo(got.dtype).eps / 2
    least = torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps
    bad = (got.double() - want).abs() > off * (1 + half) + want.abs() * half * 1.0001 + least
    assert not bool(bad.any()), f"{int(bad.sum())} of {bad.numel()}"


# odd sizes, one token and many, every kind of form
SHAPES = [(1, 48, 64), (1, 1, 17), (5, 100, 300), (16, 33, 1024), (40, 130, 100), (70, 64, 512), (150, 777, 256), (300, 400, 130)]


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("tokens,rows,k", SHAPES)
def test_activations(be, tokens, rows, k, gated, act):
    c = Case(be, tokens, rows, k, gated, rows + k, big=3.0)
    for i, ty in enumerate((torch.float32, torch.float16, torch.bfloat16)):
        res = None if gated or i == 1 else (2 * torch.randn(tokens, rows, device="cuda")).to(ty)
        bias, up_bias = (c.bias, c.up_bias if gated else None) if i != 2 else (None, None)
        y = torch.full((tokens, rows), 7.0, dtype=ty, device="cuda")
        be.gemm_i8_act(c.m, c.q, c.s, y, act, c.space, bias=bias, up_bias=up_bias, residual=res, scale=0.3)
        check(y, *c.want(act, bias, up_bias, 0.3, res))


@pytest.mark.parametrize("form", range(1, 12))
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("act", ["gelu", "silu"])
def test_every_form_gives_the_same_bits(be, form, gated, act):
    """Inside a tile and at ragged edges, with a bias at an odd address and a residual."""
    c = Case(be, 270, 300, 512, gated, 5)
    bias = torch.zeros(301, device="cuda")[1:]
    bias.copy_(c.bias)
    res = None if gated else torch.randn(270, 300, device="cuda").bfloat16()
    outs = []
    try:
        for f in (0, form):
            be.set_tuning(be.TUNE_I8_FORM, f)
            y = torch.zeros(270, 300, dtype=torch.bfloat16, device="cuda")
            be.gemm_i8_act(c.m, c.q, c.s, y, act, c.space, bias=bias, residual=res)
            outs.append(y)
    finally:
        be.set_tuning(be.TUNE_I8_FORM, 0)
    assert torch.equal(*outs)
    check(outs[1], *c.want(act, c.bias, None, 1.0, res))


@pytest.mark.parametrize("act", ACTS)
def test_arguments_far_out(be, act):
    """Through an identity of scales the arguments are given: large, tiny, zero and not finite."""
    values = [0.0, -0.0, 1e-30, -1e-30, 0.5, -0.5, 3.0, -3.0, 5.9, -5.9, 12.0, -12.0, 13.1, -13.1, 14.5, -14.5, 40.0, -40.0, 87.0, -87.0,
              88.5, -88.5, 103.0, -104.5, 1e4, -1e4, 1e15, -1e15, float("nan"), float("inf"), float("-inf")]
    n = len(values)
    m = be.upload_i8(torch.zeros(n, 16, dtype=torch.int8, device="cuda"), torch.ones(n, device="cuda"))
    bias = torch.tensor(values, device="cuda")
    y = torch.zeros(1, n, device="cuda")
    be.gemm_i8_act(m, torch.zeros(1, 16, dtype=torch.int8, device="cuda"), torch.ones(1, device="cuda"), y, act, bias=bias)
    x = bias.double()
    fine = torch.isfinite(x)
    want, off = off_act(x[fine], torch.zeros_like(x[fine]), act)
    least = 2.0 ** -126   # 32-bit results below the least normal value may be flushed to it
    assert bool(((y[0][fine].double() - want).abs() <= off * 1.001 + want.abs() * 2 * U + least).all())
    assert bool(torch.isnan(y[0, values.index(float("inf")) - 1]))
    assert y[0, n - 2].item() == float("inf")
    if act in ("relu", "relu2"):
        assert y[0, n - 1].item() == 0.0


def test_in_place_strides_and_rows_left_alone(be):
    c = Case(be, 33, 70, 100, False, 9)
    want_y = torch.zeros(33, 70, device="cuda")
    res = torch.randn(33, 70, device="cuda")
    be.gemm_i8_act(c.m, c.q, c.s, want_y, "gelu", c.space, bias=c.bias, residual=res, scale=0.5)
    buf = torch.full((33, 99), 5.0, device="cuda")
    view = buf[:, 7:77]
    view.copy_(res)
    q = torch.full((33, 131), 99, dtype=torch.int8, device="cuda")
    q[:, 3:103] = c.q
    be.gemm_i8_act(c.m, q[:, 3:103], c.s, view, "gelu", c.space, bias=c.bias, residual=view, scale=0.5)
    assert torch.equal(view, want_y)
    assert bool((buf[:, :7] == 5).all()) and bool((buf[:, 77:] == 5).all())


def test_plain_calls_agree_with_the_product_s(be):
    """No activation, no bias, scale 1 is lbh_gemm_i8, and silu of a pair its SwiGLU, bit for bit."""
    for tokens in (1, 20, 200):
        c, p = Case(be, tokens, 160, 256, False, 3), Case(be, tokens, 160, 256, True, 4)
        res = torch.randn(tokens, 160, device="cuda")
        a, b = (torch.zeros(tokens, 160, device="cuda") for _ in range(2))
        be.gemm_i8(c.m, c.q, c.s, a, c.space, residual=res)
        be.gemm_i8_act(c.m, c.q, c.s, b, "none", c.space, residual=res)
        assert torch.equal(a, b)
        be.gemm_i8_swiglu(p.m, p.q, p.s, a, p.space)
        be.gemm_i8_act(p.m, p.q, p.s, b, "silu", p.space)
        assert torch.equal(a, b)
