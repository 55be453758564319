"""int8 products (plain, with the residual, gated) against a plain 64-bit implementation.

The integer sums are exact; what is left are roundings of u = 2^-24: the sum's conversion and the two scales give
(1 + u)^3, the residual's addition one more of the result, and the output's type half a step of its own."""
import numpy as np
import pytest

from lbhip import synth

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
U = 2.0 ** -24


@pytest.fixture(scope="module")
def be():
    import lbhip
    if not torch.cuda.is_available():
        pytest.fail("no GPU visible")
    b = lbhip.HipBackend(0)
    yield b
    b.close()


def make(tokens, rows, k, seed):
    r = np.random.default_rng(seed)
    q = np.clip(np.rint(r.standard_normal((tokens, k)) * 40), -128, 127).astype(np.int8)
    w = np.clip(np.rint(r.standard_normal((rows, k)) * 40), -128, 127).astype(np.int8)
    return q, (r.random(tokens) + 0.5).astype(np.float32) / 40, w, ((r.random(rows) + 0.5) / (40 * k ** 0.5)).astype(np.float32)


def on_gpu(q, pad=0, offset=0):
    """Rows `pad` bytes apart, `offset` bytes into a buffer."""
    t, k = q.shape
    buf = torch.full((t * (k + pad) + offset + 16,), 111, dtype=torch.int8, device="cuda")
    view = buf[offset:offset + t * (k + pad)].view(t, k + pad)[:, :k]
    view.copy_(torch.from_numpy(q))
    return view


def value(q, s, w, ws):
    return (q.astype(np.float64) @ w.astype(np.float64).T) * s.astype(np.float64)[:, None] * ws.astype(np.float64)


def out_step(ty):
    """Half a step of the output's type relative to the value, and of its least subnormal."""
    f = torch.finfo(ty)
    return (0.0 if ty == torch.float32 else f.eps / 2), f.smallest_normal * f.eps / 2


def check(got, want, ty, off):
    """off: the bound on the error of the 32-bit value."""
    half, least = out_step(ty)
    g = got.double().cpu().numpy()
    limit = off * (1 + half) + (np.abs(want) * half + least) * 1.0001
    bad = ~(np.abs(g - want) <= limit)
    assert not bad.any(), (int(bad.sum()), np.argwhere(bad)[:4].tolist(), float(np.nanmax(np.abs(g - want) / limit)))


def plain_off(want):
    return np.abs(want) * 3.001 * U + 2.0 ** -149


# tokens: one, the borders of 16-, 32-, 64-, 128- and 256-token tiles; rows and k of every remainder that matters
PRODUCTS = [(1, 1, 1), (1, 16, 64), (1, 17, 63), (1, 1000, 4096), (2, 5, 15), (3, 255, 129), (7, 33, 1000), (15, 64, 65),
            (16, 100, 128), (17, 31, 16), (31, 257, 130), (32, 512, 192), (33, 48, 640), (63, 129, 256), (64, 1, 8191),
            (65, 130, 127), (100, 511, 512), (127, 256, 1024), (128, 260, 384), (129, 16, 2048), (200, 777, 320),
            (255, 128, 64), (256, 513, 1040), (257, 300, 272), (300, 1025, 768), (513, 260, 96), (1000, 520, 257)]


@pytest.mark.parametrize("tokens,rows,k", PRODUCTS)
@pytest.mark.parametrize("ty", ["f32", "bf16"])
def test_product(be, tokens, rows, k, ty):
    t = TYPES[ty]
    q, s, w, ws = make(tokens, rows, k, seed=tokens * 7 + rows * 3 + k)
    want = value(q, s, w, ws)
    m = be.upload_i8(w, ws)
    assert (m.rows, m.k, m.gated) == (rows, k, False)
    space = torch.zeros(be.gemm_i8_workspace_bytes(m, tokens), dtype=torch.uint8, device="cuda")
    sd = torch.from_numpy(s).cuda()
    first = None
    for pad, offset, ypad in ((0, 0, 0), (-k % 16, 0, 4), (5, 3, 1)):
        buf = torch.full((tokens, rows + ypad), 7.0, dtype=t, device="cuda")
        y = buf[:, :rows]
        be.gemm_i8(m, on_gpu(q, pad, offset), sd, y, space)
        check(y, want, t, plain_off(want))
        assert bool((buf[:, rows:] == 7).all())
        first = y.clone() if first is None else first
        assert torch.equal(first, y)         # the same bits by every path
    res = torch.randn(tokens, rows, generator=torch.Generator().manual_seed(k)).to(t).cuda()
    total = want + res.double().cpu().numpy()
    off = plain_off(want) + (np.abs(total) + plain_off(want)) * U
    y = torch.zeros(tokens, rows, dtype=t, device="cuda")
    be.gemm_i8(m, on_gpu(q), sd, y, space, residual=res)
    check(y, total, t, off)
    be.gemm_i8(m, on_gpu(q), sd, res, space, residual=res)    # in place
    assert torch.equal(res, y)
    m.close()


def test_product_f16_and_columns_of_one_buffer(be):
    q, s, w, ws = make(70, 96, 224, 5)
    want = value(q, s, w, ws)
    m = be.upload_i8(torch.from_numpy(w).cuda(), torch.from_numpy(ws).cuda())
    buf = torch.zeros(70, 192, dtype=torch.float16, device="cuda")
    be.gemm_i8(m, on_gpu(q), torch.from_numpy(s).cuda(), buf[:, 96:], residual=buf[:, :96])
    check(buf[:, 96:], want, torch.float16, plain_off(want) * 1.5)
    assert not bool(buf[:, :96].any())


def gated_off(g, u, h):
    """The bound on the 32-bit value's error: g and u to 3 u; g / (1 + exp(-g)) moves by 1 + |g| of g's error; exp is
    good to two half steps, and the addition, the division and the product round once each.  Where exp(-g) overflows
    (g < -88) the result is -0 and what it should be is below 2^-118 |u|."""
    return np.abs(h) * (3 * (1 + np.abs(g)) + 2 + 3 + 3) * 1.01 * U + 2.0 ** -118 * np.abs(u) + 2.0 ** -148


@pytest.mark.parametrize("tokens,rows,k", PRODUCTS)
@pytest.mark.parametrize("ty", ["f32", "bf16"])
def test_gated(be, tokens, rows, k, ty):
    t = TYPES[ty]
    q, s, w, ws = make(tokens, rows, k, seed=tokens + rows + k)
    _, _, v, vs = make(1, rows, k, seed=k)
    g, u = value(q, s, w, ws), value(q, s, v, vs)
    with np.errstate(over="ignore"):
        want = g / (1 + np.exp(-g)) * u
    m = be.upload_i8_gated(w, ws, v, vs)
    assert (m.rows, m.k, m.gated) == (rows, k, True)
    space = torch.zeros(be.gemm_i8_workspace_bytes(m, tokens), dtype=torch.uint8, device="cuda")
    first = None
    for pad, offset, ypad in ((0, 0, 0), (-k % 16, 0, 4), (7, 1, 3)):
        buf = torch.full((tokens, rows + ypad), 7.0, dtype=t, device="cuda")
        h = buf[:, :rows]
        be.gemm_i8_swiglu(m, on_gpu(q, pad, offset), torch.from_numpy(s).cuda(), h, space)
        check(h, want, t, gated_off(g, u, want))
        assert bool((buf[:, rows:] == 7).all())
        first = h.clone() if first is None else first
        assert torch.equal(first, h)
    for which, (a, b) in enumerate(((w, ws), (v, vs))):
        got = m.read(which)
        assert np.array_equal(got[0], a) and np.array_equal(got[1], b)
    m.close()


@pytest.mark.parametrize("tokens", [1, 20, 70, 300])
def test_gated_far_arguments(be, tokens):
    """Gates from -200 to 200, where exp(-g) overflows and vanishes."""
    rows, k = 64, 32
    q = np.zeros((tokens, k), np.int8)
    q[:, 0], q[:, 1] = 100, np.arange(tokens) % 100 + 1
    w, v = np.zeros((rows, k), np.int8), np.zeros((rows, k), np.int8)
    w[:, 0], v[:, 1] = np.linspace(-127, 127, rows).astype(np.int8), 3
    s, ws, vs = np.full(tokens, 0.5, np.float32), np.full(rows, 4 / 127, np.float32), np.full(rows, 0.25, np.float32)
    g, u = value(q, s, w, ws), value(q, s, v, vs)
    assert g.min() < -199.9 and g.max() > 199.9
    want = g / (1 + np.exp(-g)) * u
    m = be.upload_i8_gated(w, ws, v, vs)
    h = torch.zeros(tokens, rows, device="cuda")
    be.gemm_i8_swiglu(m, on_gpu(q), torch.from_numpy(s).cuda(), h)
    check(h, want, torch.float32, gated_off(g, u, want))


@pytest.mark.parametrize("tokens", [1, 40, 300])
def test_gated_products_beyond_the_range(be, tokens):
    """A gate that overflows to +inf gives inf times the up's sign, one that overflows to -inf is -inf / inf = NaN, as the
    formula says; the other channels stay as they are."""
    rows, k = 32, 16
    q = np.full((tokens, k), 100, np.int8)
    w, v = np.ones((rows, k), np.int8), np.full((rows, k), 2, np.int8)
    w[3], w[5], w[6] = 127, -127, 127
    v[6] = -2
    s, ws, vs = np.full(tokens, 1e30, np.float32), np.full(rows, 1e-33, np.float32), np.full(rows, 1e-33, np.float32)
    ws[[3, 5, 6]] = 1e20
    m = be.upload_i8_gated(w, ws, v, vs)
    h = torch.zeros(tokens, rows, device="cuda")
    be.gemm_i8_swiglu(m, on_gpu(q), torch.from_numpy(s).cuda(), h)
    got = h.cpu().numpy()
    assert (got[:, 3] == np.inf).all() and (got[:, 6] == -np.inf).all() and np.isnan(got[:, 5]).all()
    fine = [c for c in range(rows) if c not in (3, 5, 6)]
    g, u = value(q, s, w, ws)[:, fine], value(q, s, v, vs)[:, fine]
    check(h[:, fine], g / (1 + np.exp(-g)) * u, torch.float32, gated_off(g, u, g / (1 + np.exp(-g)) * u))


@pytest.mark.parametrize("tokens", [1, 40, 300])
def test_gated_far_arguments_times_large_values(be, tokens):
    """Gates below -104, where exp(-g) lies beyond float32 and the gate's factor below 2^-142, next to ups of 1e36:
    the products lie below 1e-5, as 0 does."""
    rows, k = 32, 16
    q = np.zeros((tokens, k), np.int8)
    q[:, 0], q[:, 1] = 100, 100
    w, v = np.zeros((rows, k), np.int8), np.zeros((rows, k), np.int8)
    w[:, 0], v[:, 1] = np.linspace(-127, -104, rows).astype(np.int8), 100
    s, ws, vs = np.ones(tokens, np.float32), np.full(rows, 0.01001, np.float32), np.full(rows, 1e32, np.float32)
    g = value(q, s, w, ws)
    assert g.max() < -104 and g.min() > -128
    m = be.upload_i8_gated(w, ws, v, vs)
    h = torch.zeros(tokens, rows, device="cuda")
    be.gemm_i8_swiglu(m, on_gpu(q), torch.from_numpy(s).cuda(), h)
    assert float(h.abs().max()) < 1e-5


@pytest.mark.parametrize("tokens", [1, 40, 130])
def test_largest_sums(be, tokens):
    """k = 131071 of -128 times -128: 2147467264, the largest sum that int32 has to hold; and its negative."""
    k, rows = 131071, 18
    q, w = np.full((tokens, k), -128, np.int8), np.full((rows, k), -128, np.int8)
    w[1::2] = 127
    s, ws = np.ones(tokens, np.float32), np.ones(rows, np.float32)
    m = be.upload_i8(w, ws)
    y = torch.zeros(tokens, rows, device="cuda")
    space = torch.zeros(be.gemm_i8_workspace_bytes(m, tokens), dtype=torch.uint8, device="cuda")
    be.gemm_i8(m, on_gpu(q, pad=1), torch.from_numpy(s).cuda(), y, space)
    want = np.where(np.arange(rows) % 2 == 0, np.float32(128 * 128 * k), np.float32(-128 * 127 * k))
    assert np.array_equal(y.cpu().numpy(), np.broadcast_to(want, (tokens, rows)))


def test_scales_that_are_not_finite(be):
    import lbhip
    q, s, w, ws = make(40, 50, 100, 1)
    s[3], s[39] = np.nan, 0.0
    m = be.upload_i8(w, ws)
    y = torch.zeros(40, 50, device="cuda")
    be.gemm_i8(m, on_gpu(q, 12), torch.from_numpy(s).cuda(), y,
               torch.zeros(be.gemm_i8_workspace_bytes(m, 40), dtype=torch.uint8, device="cuda"))
    nan = torch.isnan(y).cpu().numpy()
    assert nan[3].all() and nan.sum() == 50 and not bool(y[39].any())
    ws[7] = np.inf
    with pytest.raises(lbhip.QuantError) as e:
        be.upload_i8(w, ws)
    assert (e.value.variant, e.value.row, e.value.field, e.value.bits) == ("NonFiniteScale", 7, 0, 0x7f800000)
    with pytest.raises(lbhip.QuantError) as e:
        be.upload_i8_gated(w, np.ones(50, np.float32), w, ws)
    assert (e.value.row, e.value.field) == (7, 1)


@pytest.mark.parametrize("tokens", [1, 5, 16, 40, 64, 100, 300])
def test_tokens_do_not_depend_on_their_batch(be, tokens):
    q, s, w, ws = make(300, 200, 512, 2)
    m = be.upload_i8(w, ws)
    full, part = torch.zeros(300, 200, device="cuda"), torch.zeros(tokens, 200, device="cuda")
    sd = torch.from_numpy(s).cuda()
    be.gemm_i8(m, on_gpu(q), sd, full)
    be.gemm_i8(m, on_gpu(q)[300 - tokens:], sd[300 - tokens:], part)
    assert torch.equal(full[300 - tokens:], part)


@pytest.mark.parametrize("ty", [synth.Q4_K, synth.Q5_K, synth.IQ2_S, synth.IQ3_S])
def test_from_packed(be, oracle, ty):
    """The int8 form of an uploaded matrix: each decoded row by the row quantizer's rule."""
    rows, k = 37, 768
    a, b = synth.random_matrix(ty, rows, k, 3), synth.random_matrix(ty, rows, k, 4)
    ex = oracle.make_exec(oracle.MODE_DEQUANT_F32)
    da, db = be.upload(ty, rows, k, a), be.upload(ty, rows, k, b)
    got = be.i8_from_packed(da, db)
    for which, raw in enumerate((a, b)):
        om = oracle.make_matrix(ty, rows, k, raw)
        eye = np.eye(k, dtype=np.float32)
        f = np.stack([oracle.gemv(ex, om, eye[i]) for i in range(k)], axis=1).astype(np.float64)
        s = (np.abs(f).max(axis=1) / 127).astype(np.float32)
        want = np.rint(f / np.where(s > 0, s, 1).astype(np.float64)[:, None])
        q, scales = got.read(which)
        assert np.array_equal(scales, s) and np.array_equal(q, np.where((s > 0)[:, None], want, 0).astype(np.int8))
    one = be.i8_from_packed(da)
    assert not one.gated and all(np.array_equal(x, y) for x, y in zip(one.read(), got.read(0)))


def test_from_packed_f32_and_refusals(be):
    import lbhip
    r = np.random.default_rng(2)
    w = r.standard_normal((300, 512)).astype(np.float32)
    w[5] = 0
    q, s = be.i8_from_packed(be.upload(lbhip.F32, 300, 512, w)).read()
    want = (np.abs(w.astype(np.float64)).max(axis=1) / 127).astype(np.float32)
    assert np.array_equal(s, want)
    assert np.array_equal(q, np.rint(w / np.where(want > 0, want, 1).astype(np.float64)[:, None]).astype(np.int8))
    other = be.upload(lbhip.F32, 300, 256, w[:, :256])
    with pytest.raises(lbhip.KernelError) as e:
        be.i8_from_packed(be.upload(lbhip.F32, 300, 512, w), other)
    assert e.value.variant == "DimensionMismatch"
    w[17, 100] = np.nan
    with pytest.raises(lbhip.QuantError) as e:
        be.i8_from_packed(be.upload(lbhip.F32, 300, 512, w))
    assert (e.value.variant, e.value.row) == ("NonFiniteScale", 17)


def test_strided_device_weights_are_copied_in_the_backend_s_stream(be):
    """The copy that makes device weights contiguous runs where the upload reads it, whatever waits on the stream that
    is current."""
    import lbhip
    r = np.random.default_rng(3)
    wide = torch.from_numpy(r.integers(-128, 128, (512, 4096), dtype=np.int8)).cuda()
    scales = torch.from_numpy(r.random((512, 2)).astype(np.float32)).cuda()
    w, s = wide[:, 1000:3000], scales[:, 1]
    torch.cuda.synchronize()
    other = lbhip.HipBackend(0, stream=torch.cuda.Stream())
    torch.cuda._sleep(200_000_000)   # some 0.1 s of work in the current stream
    m = other.upload_i8(w, s)
    got = m.read()
    assert np.array_equal(got[0], w.cpu().numpy()) and np.array_equal(got[1], s.cpu().numpy())
    m.close()
    torch.cuda.synchronize()
    other.close()


@pytest.mark.parametrize("form", range(1, 12))
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("ty", ["f32", "f16", "bf16"])
def test_every_form_gives_the_same_bits(be, form, gated, ty):
    """Each form over ragged and whole tiles of its own size, against the rule's choice and the 64-bit value: with the
    residual (in place and apart), rows at odd addresses, and rows behind the last token left alone."""
    t = TYPES[ty]
    for tokens, rows, k in ((1, 1, 1), (19, 272, 320), (64, 64, 64), (130, 200, 1040), (256, 512, 256), (300, 384, 576)):
        q, s, w, ws = make(tokens, rows, k, seed=form)
        _, _, v, vs = make(1, rows, k, seed=form + 50)
        m = be.upload_i8_gated(w, ws, v, vs) if gated else be.upload_i8(w, ws)
        space = torch.zeros(be.gemm_i8_workspace_bytes(m, tokens), dtype=torch.uint8, device="cuda")
        x, sd = on_gpu(q, -k % 16), torch.from_numpy(s).cuda()
        res = None if gated else torch.randn(tokens, rows, generator=torch.Generator().manual_seed(1)).to(t).cuda()

        def call(form, pad, residual):
            buf = torch.full((tokens + 3, rows + pad), 5.0, dtype=t, device="cuda")
            y = buf[:tokens, :rows]
            be.set_tuning(be.TUNE_I8_FORM, form)
            try:
                if gated:
                    be.gemm_i8_swiglu(m, x, sd, y, space)
                else:
                    if residual == "place":
                        y.copy_(res)
                    be.gemm_i8(m, x, sd, y, space, residual={None: None, "apart": res, "place": y}[residual])
            finally:
                be.set_tuning(be.TUNE_I8_FORM, 0)
            assert bool((buf[tokens:] == 5).all()) and bool((buf[:, rows:] == 5).all())
            return y.clone()

        first = call(0, 0, None)
        for pad in (0, 8, 3):
            assert torch.equal(call(form, pad, None), first), (tokens, rows, k, pad)
        if gated:
            g, u = value(q, s, w, ws), value(q, s, v, vs)
            want = g / (1 + np.exp(-g)) * u
            check(first, want, t, gated_off(g, u, want))
        else:
            check(first, value(q, s, w, ws), t, plain_off(value(q, s, w, ws)))
            added = call(0, 0, "apart")
            for pad in (0, 3):
                assert torch.equal(call(form, pad, "apart"), added) and torch.equal(call(form, pad, "place"), added)
        m.close()


@pytest.mark.parametrize("tokens", [1, 3, 4, 5, 16])
@pytest.mark.parametrize("gated", [False, True])
def test_large_matrices(be, tokens, gated):
    """Matrices from 64 MiB on, which few tokens read past the caches: the same bits as in the smallest tiles."""
    rows, k = (16500, 2060) if gated else (16500, 4112)
    g = torch.Generator(device="cuda").manual_seed(tokens)
    w, v = (torch.randint(-128, 128, (rows, k), dtype=torch.int8, device="cuda", generator=g) for _ in range(2))
    ws = torch.rand(rows, device="cuda", generator=g) / 1e5
    q = torch.randint(-128, 128, (tokens, k), dtype=torch.int8, device="cuda", generator=g)
    s = torch.rand(tokens, device="cuda", generator=g) + 0.5
    m = be.upload_i8_gated(w, ws, v, ws) if gated else be.upload_i8(w, ws)
    assert m.device_bytes > 64 << 20
    space = torch.zeros(be.gemm_i8_workspace_bytes(m, tokens), dtype=torch.uint8, device="cuda")
    outs = []
    for form in (0, 1, 11, 6):
        outs.append(torch.zeros(tokens, rows, device="cuda"))
        be.set_tuning(be.TUNE_I8_FORM, form)
        try:
            (be.gemm_i8_swiglu if gated else be.gemm_i8)(m, q, s, outs[-1], space)
        finally:
            be.set_tuning(be.TUNE_I8_FORM, 0)
    assert all(torch.equal(o, outs[0]) for o in outs)
    c = torch.randint(0, rows, (50,), generator=torch.Generator().manual_seed(1)).numpy()
    q, s, w, v, ws = (t.cpu().numpy() for t in (q, s, w, v, ws))
    g, u = value(q, s, w[c], ws[c]), value(q, s, v[c], ws[c])
    got = outs[0][:, torch.from_numpy(c).cuda()]
    if gated:
        with np.errstate(over="ignore"):
            want = g / (1 + np.exp(-g)) * u
        check(got, want, torch.float32, gated_off(g, u, want))
    else:
        check(got, g, torch.float32, plain_off(g))
    m.close()


@pytest.mark.parametrize("form", [0, 1, 4, 6, 8, 9, 10, 11])
def test_rows_far_apart(be, form):
    """Strides that take the last rows beyond 32 bits: x rows 2^23 bytes apart (2.5 GB), y rows 2^24 elements (10 GB)."""
    tokens, rows, k = 300, 64, 64
    q, s, w, ws = make(tokens, rows, k, seed=77)
    x = torch.empty(tokens * (1 << 23), dtype=torch.int8, device="cuda").view(tokens, 1 << 23)[:, :k]
    x.copy_(torch.from_numpy(q))
    y = torch.empty(tokens * (1 << 24), dtype=torch.bfloat16, device="cuda").view(tokens, 1 << 24)[:, :rows]
    m = be.upload_i8(w, ws)
    be.set_tuning(be.TUNE_I8_FORM, form)
    try:
        be.gemm_i8(m, x, torch.from_numpy(s).cuda(), y)
    finally:
        be.set_tuning(be.TUNE_I8_FORM, 0)
    want = value(q, s, w, ws)
    check(y, want, torch.bfloat16, plain_off(want))


def test_from_packed_f32_in_pieces(be):
    """A matrix of 1 GiB with more rows than one launch takes: exact, and beside the result and its codes only a piece of
    the decoded values is held (the free memory is read all the while)."""
    import threading

    import lbhip
    rows, k = (1 << 20) + 37, 256
    g = torch.Generator(device="cuda").manual_seed(6)
    x = torch.randn(rows, k, device="cuda", generator=g)
    scale = (x.abs().amax(1).double() / 127).float()
    want = torch.empty(rows, k, dtype=torch.int8, device="cuda")
    for at in range(0, rows, 1 << 17):
        part = slice(at, at + (1 << 17))
        want[part] = torch.round(x[part].double() / scale[part].double()[:, None]).to(torch.int8)
    want, scale, host = want.cpu().numpy(), scale.cpu().numpy(), x.cpu().numpy()
    m = be.upload(lbhip.F32, rows, k, host)
    del x, host
    torch.cuda.empty_cache()
    torch.cuda.synchronize()
    before, least, done = torch.cuda.mem_get_info()[0], [1 << 62], threading.Event()

    def watch():
        while not done.is_set():
            least[0] = min(least[0], torch.cuda.mem_get_info()[0])

    thread = threading.Thread(target=watch)
    thread.start()
    try:
        m8 = be.i8_from_packed(m)
    finally:
        done.set()
        thread.join()
    least[0] = min(least[0], torch.cuda.mem_get_info()[0])
    q, s = m8.read()
    assert np.array_equal(s, scale) and np.array_equal(q, want)
    held = before - least[0]
    assert held >= m8.device_bytes
    # the result, the codes, the scales, a piece of 64 MiB, and room for the allocator's own granularity
    assert held <= m8.device_bytes + rows * (k + 4) + (64 << 20) + (64 << 20), held >> 20
    m8.close(), m.close()


@pytest.mark.parametrize("tokens", [1, 20, 70, 200, 300])
def test_gated_down_to_the_least_factor(be, tokens):
    """Gates from -80 to -95 in steps of 0.05 next to ups of 1e36, which bring the factors into sight: good to its roundings
    above -126 ln 2 = -87.34, where the factor is 2^-119.6, and 0 from there on (g itself is off by 2e-5)."""
    rows, k = 300, 16
    q, w, v = np.zeros((tokens, k), np.int8), np.zeros((rows, k), np.int8), np.zeros((rows, k), np.int8)
    q[:, 0], q[:, 1], q[:, 2] = 100, 1, 100
    total = -8000 - 5 * np.arange(rows)
    w[:, 0], w[:, 1], v[:, 2] = -(-total // 100), -(-total % 100), 100
    s, ws, vs = np.ones(tokens, np.float32), np.full(rows, 0.01, np.float32), np.full(rows, 1e32, np.float32)
    g, u = value(q, s, w, ws), value(q, s, v, vs)
    assert g.max() > -80.01 and g.min() < -94.9
    want = g / (1 + np.exp(-g)) * u
    m = be.upload_i8_gated(w, ws, v, vs)
    h = torch.zeros(tokens, rows, device="cuda")
    be.gemm_i8_swiglu(m, on_gpu(q), torch.from_numpy(s).cuda(), h)
    got, border = h.double().cpu().numpy(), -126 * np.log(2)
    seen, gone = g > border + 1e-3, g < border - 1e-3
    limit = np.abs(want) * (3 * (1 + np.abs(g)) + 8) * 1.01 * U
    assert seen.any() and (np.abs(got - want) <= limit)[seen].all()
    assert gone.any() and (got[gone] == 0).all()
    assert (np.abs(want[gone]) < 2.0 ** -119 * u[gone]).all()


@pytest.mark.parametrize("tokens", [1, 3, 4])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("ty", ["f32", "f16", "bf16"])
def test_large_matrices_in_every_type(be, tokens, gated, ty):
    """What few tokens read past the caches, in each output type: with the residual apart and in place, rows of y apart,
    and the bytes around them left alone."""
    t = TYPES[ty]
    rows, k = (16500, 2064) if gated else (16500, 4112)
    g = torch.Generator(device="cuda").manual_seed(tokens)
    w, v = (torch.randint(-128, 128, (rows, k), dtype=torch.int8, device="cuda", generator=g) for _ in range(2))
    ws = (torch.rand(rows, device="cuda", generator=g) + 0.5) / (5000 * k ** 0.5)
    q = torch.randint(-128, 128, (tokens, k), dtype=torch.int8, device="cuda", generator=g)
    s = torch.rand(tokens, device="cuda", generator=g) + 0.5
    m = be.upload_i8_gated(w, ws, v, ws) if gated else be.upload_i8(w, ws)
    assert m.device_bytes > 64 << 20
    res = torch.randn(tokens, rows, device="cuda", generator=g).to(t)

    def call(form, pad, residual):
        buf = torch.full((tokens + 1, rows + pad), 5.0, dtype=t, device="cuda")
        y = buf[:tokens, :rows]
        be.set_tuning(be.TUNE_I8_FORM, form)
        try:
            if gated:
                be.gemm_i8_swiglu(m, q, s, y)
            else:
                if residual == "place":
                    y.copy_(res)
                be.gemm_i8(m, q, s, y, residual={None: None, "apart": res, "place": y}[residual])
        finally:
            be.set_tuning(be.TUNE_I8_FORM, 0)
        assert bool((buf[tokens:] == 5).all()) and bool((buf[:, rows:] == 5).all())
        return y.clone()

    plain = call(6, 0, None)
    added = None if gated else call(6, 0, "apart")
    for form in (0, 1, 11):
        for pad in (0, 4, 3):
            assert torch.equal(call(form, pad, None), plain)
            if not gated:
                assert torch.equal(call(form, pad, "apart"), added) and torch.equal(call(form, pad, "place"), added)
    c = np.random.default_rng(1).integers(0, rows, 60)
    at = torch.from_numpy(c).cuda()
    res, q, s, w, v, ws = (a.cpu() for a in (res[:, at], q, s, w[at], v[at], ws[at]))
    q, s, w, v, ws = (a.numpy() for a in (q, s, w, v, ws))
    a, u = value(q, s, w, ws), value(q, s, v, ws)
    if gated:
        want = a / (1 + np.exp(-a)) * u
        check(plain[:, at], want, t, gated_off(a, u, want))
    else:
        check(plain[:, at], a, t, plain_off(a))
        total = a + res.double().numpy()
        check(added[:, at], total, t, plain_off(a) + (np.abs(total) + plain_off(a)) * U)
    m.close()


@pytest.mark.parametrize("form,cw,tw", [(6, 1, 1), (7, 2, 1), (8, 2, 2), (9, 3, 2), (10, 4, 4)])
@pytest.mark.parametrize("kind", ["plain", "residual", "gated"])
def test_grids_of_many_tiles(be, form, cw, tw, kind):
    """Each tile form over 18 token tiles (two whole panels of eight and a narrow one) and six channel tiles, the last of
    both ragged: 108 tiles, which do not divide evenly among eight XCDs; and over 17 x 5 = 85 whole ones."""
    gated = kind == "gated"
    ch, k = 64 * cw // (2 if gated else 1), 272
    for tokens, rows in ((17 * 64 * tw + 3, 5 * ch + 9), (17 * 64 * tw, 5 * ch)):
        g = torch.Generator(device="cuda").manual_seed(form + tokens)
        w, v = (torch.randint(-128, 128, (rows, k), dtype=torch.int8, device="cuda", generator=g) for _ in range(2))
        q = torch.randint(-128, 128, (tokens, k), dtype=torch.int8, device="cuda", generator=g)
        ws, s = torch.rand(rows, device="cuda", generator=g) / 9e4, torch.rand(tokens, device="cuda", generator=g) + 0.5
        res = torch.randn(tokens, rows, device="cuda", generator=g).bfloat16() if kind == "residual" else None
        m = be.upload_i8_gated(w, ws, v, ws) if gated else be.upload_i8(w, ws)
        outs = []
        for f in (form, 1):
            buf = torch.full((tokens + 2, rows + 8), 5.0, dtype=torch.bfloat16, device="cuda")
            y = buf[:tokens, :rows]
            be.set_tuning(be.TUNE_I8_FORM, f)
            try:
                if gated:
                    be.gemm_i8_swiglu(m, q, s, y)
                else:
                    be.gemm_i8(m, q, s, y, residual=res)
            finally:
                be.set_tuning(be.TUNE_I8_FORM, 0)
            assert bool((buf[tokens:] == 5).all()) and bool((buf[:, rows:] == 5).all())
            outs.append(y.clone())
        assert torch.equal(outs[0], outs[1])
        q, s, w, v, ws = (a.cpu().numpy() for a in (q, s, w, v, ws))
        a = value(q, s, w, ws)
        if gated:
            u = value(q, s, v, ws)
            want = a / (1 + np.exp(-a)) * u
            check(outs[0], want, torch.bfloat16, gated_off(a, u, want))
        else:
            want = a if res is None else a + res.double().cpu().numpy()
            check(outs[0], want, torch.bfloat16, plain_off(a) + (np.abs(want) + plain_off(a)) * U)
        m.close()


@pytest.mark.parametrize("rows,k", [(5, 1), (40, 255), (17, 256), (64, 257), (16, 1000)])
@pytest.mark.parametrize("gated", [False, True])
def test_workspace_sizes(be, rows, k, gated):
    """Rows are padded to 256 bytes; one byte less than the stated size is refused, the size itself is enough."""
    import lbhip
    tokens = 9
    q, s, w, ws = make(tokens, rows, k, 4)
    m = be.upload_i8_gated(w, ws, w, ws) if gated else be.upload_i8(w, ws)
    need = be.gemm_i8_workspace_bytes(m, tokens)
    assert need == tokens * (-(-k // 256) * 256)
    assert m.device_bytes == (2 if gated else 1) * -(-rows // 16) * (16 * (-(-k // 256) * 256) + 64)
    x, sd, y = on_gpu(q, 3, 1), torch.from_numpy(s).cuda(), torch.zeros(tokens, rows, device="cuda")
    call = be.gemm_i8_swiglu if gated else be.gemm_i8
    buf = torch.full((need + 64,), 3, dtype=torch.uint8, device="cuda")
    with pytest.raises(lbhip.KernelError) as e:
        call(m, x, sd, y, buf[:need - 1])
    assert e.value.variant == "ScratchTooSmall"
    call(m, x, sd, y, buf[:need])
    assert bool((buf[need:] == 3).all())
    g = value(q, s, w, ws)
    want = g / (1 + np.exp(-g)) * g if gated else g
    check(y, want, torch.float32, gated_off(g, g, want) if gated else plain_off(g))


def test_the_tallest_matrix(be):
    """2^26 channels, the most there may be, of a gated pair: a launch counts its threads in 32 bits, so 23 tokens do not fit
    one in the streaming form of 16 tokens, which is refused where it is asked for and not chosen otherwise."""
    import lbhip
    rows, k, tokens = 1 << 26, 16, 23
    g = torch.Generator(device="cuda").manual_seed(2)
    w, v = (torch.randint(-128, 128, (rows, k), dtype=torch.int8, device="cuda", generator=g) for _ in range(2))
    ws = (torch.rand(rows, device="cuda", generator=g) + 0.5) / 4e4
    q = torch.randint(-128, 128, (tokens, k), dtype=torch.int8, device="cuda", generator=g)
    s = torch.rand(tokens, device="cuda", generator=g) + 0.5
    m = be.upload_i8_gated(w, ws, v, ws)
    h, tiles = (torch.zeros(tokens, rows, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    be.gemm_i8_swiglu(m, q, s, h)
    try:
        be.set_tuning(be.TUNE_I8_FORM, 1)
        with pytest.raises(lbhip.KernelError):
            be.gemm_i8_swiglu(m, q, s, tiles)
        be.set_tuning(be.TUNE_I8_FORM, 6)
        be.gemm_i8_swiglu(m, q, s, tiles)
    finally:
        be.set_tuning(be.TUNE_I8_FORM, 0)
    assert torch.equal(h, tiles)
    c = torch.cat([torch.randint(0, rows, (500,), generator=torch.Generator().manual_seed(1)), torch.arange(rows - 40, rows)])
    at = c.cuda()
    got = h[:, at]
    q, s, w, v, ws = (a.cpu().numpy() for a in (q, s, w[at], v[at], ws[at]))
    a, u = value(q, s, w, ws), value(q, s, v, ws)
    want = a / (1 + np.exp(-a)) * u
    check(got, want, torch.bfloat16, gated_off(a, u, want))
    m.close()
    del w, v, h, tiles, got
    torch.cuda.empty_cache()
