"""RMS norm rows and their outputs (rows, Q8_K blocks, int8 with scales) against a plain 64-bit implementation.

The kernel computes in 64 bits between its loads and its roundings, as the oracle does; the two differ by some 1e-15
of a value, so the integers and scales have to be equal and the rows are off by their roundings alone."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
EPS = 1e-5


@pytest.fixture(scope="module")
def be():
    import lbhip
    if not torch.cuda.is_available():
        pytest.fail("no GPU visible")
    b = lbhip.HipBackend(0)
    yield b
    b.close()


def strided(t, pad=0, offset=0):
    """t's rows on the GPU, `pad` elements apart and `offset` elements into their buffer; the buffer and the view."""
    rows, n = t.shape
    buf = torch.full((rows * (n + pad) + offset + 8,), 77, dtype=t.dtype, device="cuda")
    view = buf[offset:offset + rows * (n + pad)].view(rows, n + pad)[:, :n]
    view.copy_(t)
    return buf, view


def oracle_norm(hidden, delta, weight, eps):
    """(h as stored, v in 64 bits): the addition in 32 bits, then in the rows' type."""
    h = hidden if delta is None else (hidden.float() + delta.float()).to(hidden.dtype)
    d = h.double().numpy()
    with np.errstate(all="ignore"):
        return h, d * weight.double().numpy() / np.sqrt((d * d).mean(axis=1, keepdims=True) + eps)


def oracle_i8(v):
    with np.errstate(all="ignore"):
        s = (np.abs(v).max(axis=1) / 127.0).astype(np.float32)
        s = np.where(np.isfinite(v).all(axis=1) & np.isfinite(s), s, np.float32("nan"))
        s = np.where(s < np.float32(2.0 ** -126), np.float32(0), s)
        q = np.rint(v / np.where(s > 0, s, 1).astype(np.float64)[:, None])
    return np.where((s > 0)[:, None], q, 0).astype(np.int8), s


def near(got, v, ty):
    """got within the roundings of v: to 32 bits, then to the type, half a step each (and half the least subnormal)."""
    steps = 2.0 ** -24 + (0 if ty == torch.float32 else torch.finfo(ty).eps / 2 * (1 + 2.0 ** -24))
    least = torch.finfo(ty).smallest_normal * torch.finfo(ty).eps / 2
    g = got.double().cpu().numpy()
    np.testing.assert_array_less(np.abs(g - v), np.abs(v) * (steps + 1e-12) + least * 1.01 + 1e-300)


def inputs(rows, n, ty, seed, delta=True):
    g = torch.Generator().manual_seed(seed)
    size = torch.exp(torch.randn(n, generator=g))
    return ((torch.randn(rows, n, generator=g) * size).to(ty), torch.randn(rows, n, generator=g).to(ty) if delta else None,
            1.0 + 0.3 * torch.randn(n, generator=g))


# (rows, n): one row and many, every form (64, 256 and 1024 threads a row, and rows beyond their registers), its borders
SHAPES = [(1, 1), (3, 7), (5, 64), (9, 511), (7, 512), (4, 513), (2, 520), (1, 4096), (33, 2048), (6, 4095), (3, 4097),
          (2, 4104), (2, 7168), (3, 16384), (2, 16385), (1, 50001), (2, 40000)]


@pytest.mark.parametrize("ty", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,n", SHAPES)
def test_norm_rows_and_int8(be, rows, n, ty):
    t = TYPES[ty]
    hidden, delta, weight = inputs(rows, n, t, seed=rows * 100003 + n)
    h, v = oracle_norm(hidden, delta, weight, EPS)
    q_want, s_want = oracle_i8(v)
    # aligned rows, and rows of odd strides from an odd element on
    for pad, offset in ((0, 0), (3, 1)):
        _, hd = strided(hidden, pad, offset)
        _, dd = strided(delta, pad, offset)
        out_buf, out = strided(torch.zeros_like(hidden), pad, offset)
        y_buf, y = strided(torch.zeros_like(hidden), pad, offset)
        q_buf, q = strided(torch.zeros(rows, n, dtype=torch.int8), pad, offset)
        s = torch.full((rows,), -1.0, device="cuda")
        be.rms_norm_i8_rows(hd, weight.cuda(), EPS, q, s, y=y, delta=dd, hidden_out=out)
        torch.cuda.synchronize()
        assert torch.equal(out.cpu(), h)
        np.testing.assert_array_equal(s.cpu().numpy(), s_want)
        np.testing.assert_array_equal(q.cpu().numpy(), q_want)
        near(y, v, t)
        for buf in (out_buf, y_buf, q_buf):   # bytes around the rows are left alone
            rest = buf.clone()
            rest[offset:offset + rows * (n + pad)].view(rows, n + pad)[:, :n] = 77
            assert bool((rest == 77).all())
        assert torch.equal(hd.cpu(), hidden)


@pytest.mark.parametrize("ty", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("y_ty", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n", [96, 1023, 4096])
def test_norm_rows_alone_in_every_type(be, ty, y_ty, n):
    hidden, _, weight = inputs(5, n, TYPES[ty], seed=n, delta=False)
    _, v = oracle_norm(hidden, None, weight, EPS)
    y = torch.zeros(5, n, dtype=TYPES[y_ty], device="cuda")
    be.rms_norm_rows(hidden.cuda(), weight.cuda(), EPS, y)
    near(y, v, TYPES[y_ty])


@pytest.mark.parametrize("ty", ["f32", "bf16"])
@pytest.mark.parametrize("rows,n", [(1, 256), (3, 512), (2, 1024), (5, 4096), (2, 4352), (2, 16384)])
def test_norm_q8_k_is_the_quantizer_s_of_its_rows(be, oracle, rows, n, ty):
    hidden, delta, weight = inputs(rows, n, TYPES[ty], seed=n)
    h, v = oracle_norm(hidden, delta, weight, EPS)
    for pad, offset in ((0, 0), (5, 3)):
        _, hd = strided(hidden, pad, offset)
        out = torch.zeros_like(hidden, device="cuda")
        y = torch.zeros(rows, n, device="cuda")
        enc = torch.full((rows + 1, n // 256 * 292), 9, dtype=torch.uint8, device="cuda")
        be.rms_norm_q8_k_rows(hd, weight.cuda(), EPS, enc[:rows], y=y, delta=delta.cuda(), hidden_out=out)
        torch.cuda.synchronize()
        near(y, v, torch.float32)
        assert torch.equal(out.cpu(), h)
        for r in range(rows):   # bit for bit the blocks of the float32 rows
            np.testing.assert_array_equal(enc[r].cpu().numpy(), oracle.quantize_q8_k(y[r].cpu().numpy()))
        assert bool((enc[rows] == 9).all())
        alone = torch.zeros_like(enc[:rows])   # without the rows
        be.rms_norm_q8_k_rows(hd, weight.cuda(), EPS, alone, delta=delta.cuda())
        assert torch.equal(alone, enc[:rows])


@pytest.mark.parametrize("ty", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,n", [(1, 1), (4, 100), (3, 512), (6, 1536), (2, 13312), (2, 20001)])
def test_quantize_i8_rows(be, rows, n, ty):
    x, _, _ = inputs(rows, n, TYPES[ty], seed=n + 1, delta=False)
    q_want, s_want = oracle_i8(x.double().numpy())
    for pad, offset in ((0, 0), (1, 5)):
        _, xd = strided(x, pad, offset)
        q, s = torch.zeros(rows, n, dtype=torch.int8, device="cuda"), torch.zeros(rows, device="cuda")
        be.quantize_i8_rows(xd, q, s)
        np.testing.assert_array_equal(q.cpu().numpy(), q_want)
        np.testing.assert_array_equal(s.cpu().numpy(), s_want)


@pytest.mark.parametrize("n", [64, 520, 4096, 5000, 17000])
def test_ties_zeros_and_values_that_are_not_finite(be, n):
    rows = 12
    x = torch.randn(rows, n, generator=torch.Generator().manual_seed(n))
    x[0] = 0.0
    x[1] = -0.0
    x[2] = 1e-45                            # a scale that rounds to nothing
    x[3] = 127 * 2.0 ** -127                # a scale of 2^-127, below the least normal value
    x[4] = torch.linspace(-1, 1, n) * 127 * 2.0 ** -126   # the least normal scale
    x[4, 0] = 127 * 2.0 ** -126
    x[5, n // 2] = float("nan")
    x[6, n - 1] = float("inf")
    x[7, 0] = float("-inf")
    x[8] = torch.arange(n) % 255 / 2 - 63.5   # ties: halves of a scale of one
    x[8, 0] = 127.0
    x[9] = 3e38
    x[10] = 5.0                              # equal values, all at the end of the range
    x[11, 1:] = 0.0
    q_want, s_want = oracle_i8(x.double().numpy())
    q, s = torch.full((rows, n), 3, dtype=torch.int8, device="cuda"), torch.zeros(rows, device="cuda")
    be.quantize_i8_rows(x.cuda(), q, s)
    np.testing.assert_array_equal(s.cpu().numpy(), s_want)
    np.testing.assert_array_equal(q.cpu().numpy(), q_want)
    assert s_want[8] == 1.0 and np.isnan(s_want[5:8]).all() and (s_want[:4] == 0).all()
    # the norm of such rows: zeros stay zeros, what is not finite reaches its own row alone
    weight = torch.ones(n)
    _, v = oracle_norm(x, None, weight, EPS)
    q_want, s_want = oracle_i8(v)
    y = torch.zeros(rows, n, device="cuda")
    be.rms_norm_i8_rows(x.cuda(), weight.cuda(), EPS, q, s, y=y)
    np.testing.assert_array_equal(s.cpu().numpy(), s_want)
    np.testing.assert_array_equal(q.cpu().numpy(), q_want)
    fine = np.isfinite(v).all(axis=1)
    assert fine.sum() == rows - 3
    near(y[torch.from_numpy(fine).cuda()], v[fine], torch.float32)
    np.testing.assert_array_equal(np.isnan(y.cpu().numpy()), np.isnan(v))


@pytest.mark.parametrize("ty", ["f32", "f16"])
@pytest.mark.parametrize("scale", [3.0, 5.0, 7.0, 13.0])
@pytest.mark.parametrize("n", [255, 256, 4096, 17000])
def test_quantize_ties_of_scales_that_are_no_power_of_two(be, n, scale, ty):
    """x = scale * (i + 1/2): the quotient is a tie exactly, though 1 / scale is no float of any width."""
    x = ((torch.arange(n) % 253 - 126.5) * scale).to(TYPES[ty]).repeat(3, 1)
    x[:, 0] = 127 * scale
    x[1] = -x[1]
    x[2] = x[2] * 2.0 ** -9
    q_want, s_want = oracle_i8(x.double().numpy())
    assert s_want[0] == scale and s_want[2] == scale / 512 and q_want[0, 127] == 0 and q_want[0, 128] == 2
    for pad, offset in ((0, 0), (3, 1)):
        _, xd = strided(x, pad, offset)
        q, s = torch.zeros(3, n, dtype=torch.int8, device="cuda"), torch.zeros(3, device="cuda")
        be.quantize_i8_rows(xd, q, s)
        np.testing.assert_array_equal(s.cpu().numpy(), s_want)
        np.testing.assert_array_equal(q.cpu().numpy(), q_want)


def test_quantize_values_next_to_ties(be):
    """The float32 neighbours of scale * (i + 1/2) fall to their own sides."""
    for scale in (3.0, 2.0 ** -100 * 1.7, 0.1, 12345.678):
        s32 = np.float32(127 * np.float64(scale))
        s32 = np.float32(np.float64(s32) / 127)
        mid = (np.arange(254) - 126.5) * np.float64(s32)
        x = np.stack([np.float32(mid), np.nextafter(np.float32(mid), np.float32(np.inf)),
                      np.nextafter(np.float32(mid), np.float32(-np.inf))])
        x[:, 0] = np.float32(127 * np.float64(s32))
        q_want, s_want = oracle_i8(x.astype(np.float64))
        q, s = torch.zeros(3, 254, dtype=torch.int8, device="cuda"), torch.zeros(3, device="cuda")
        be.quantize_i8_rows(torch.from_numpy(x).cuda(), q, s)
        np.testing.assert_array_equal(s.cpu().numpy(), s_want)
        np.testing.assert_array_equal(q.cpu().numpy(), q_want)


def test_largest_scale(be):
    """A scale that is the largest float32 is finite; one past it is not."""
    n, top = 127 * 127, np.finfo(np.float32).max
    x = torch.zeros(2, n)
    x[:, 5] = 1.0                              # times 127 after the norm
    x[1, 6] = 1.0                              # and times 127 / sqrt(2)
    weight = torch.ones(n)
    weight[5] = float(top)
    q, s = torch.zeros(2, n, dtype=torch.int8, device="cuda"), torch.zeros(2, device="cuda")
    be.rms_norm_i8_rows(x.cuda(), weight.cuda(), 1e-300, q, s)
    assert s[0].item() == top and q[0, 5].item() == 127 and int(q[0].abs().sum()) == 127
    assert s[1].item() < top and q[1, 5].item() == 127 and q[1, 6].item() == 0
    x = torch.zeros(1, 128 * 128)
    x[0, 5] = 1.0                              # times 128: 128 / 127 of the largest scale
    weight = torch.ones(128 * 128)
    weight[5] = float(top)
    q = torch.ones(1, 128 * 128, dtype=torch.int8, device="cuda")
    be.rms_norm_i8_rows(x.cuda(), weight.cuda(), 1e-300, q, s[:1])
    assert bool(torch.isnan(s[0])) and not bool(q.any())


def test_weight_that_is_not_finite(be):
    x, _, w = inputs(3, 700, torch.float32, 4, delta=False)
    w[9] = float("nan")
    q, s = torch.ones(3, 700, dtype=torch.int8, device="cuda"), torch.zeros(3, device="cuda")
    be.rms_norm_i8_rows(x.cuda(), w.cuda(), EPS, q, s)
    assert bool(torch.isnan(s).all()) and not bool(q.any())


@pytest.mark.parametrize("n", [512, 4352, 16384])
def test_norm_q8_k_of_rows_that_are_zero_or_not_finite(be, n):
    """Each row's blocks are what the row quantizer makes of its float32 values, whatever they are."""
    x, _, w = inputs(6, n, torch.float32, n, delta=False)
    x[0] = 0.0
    x[1, 3] = float("nan")
    x[2, n - 1] = float("inf")
    x[3, 256:512] = 0.0
    x[4, :256] = 5.0
    y = torch.zeros(6, n, device="cuda")
    enc, want = (torch.full((6, n // 256 * 292), 9, dtype=torch.uint8, device="cuda") for _ in range(2))
    be.rms_norm_q8_k_rows(x.cuda(), w.cuda(), EPS, enc, y=y)
    be.quantize_q8_k_rows(y, want, 6, n)
    assert torch.equal(enc, want)
    _, v = oracle_norm(x, None, w, EPS)
    near(y[torch.tensor([0, 3, 4, 5])], v[[0, 3, 4, 5]], torch.float32)


@pytest.mark.parametrize("n", [512, 4096, 4097, 30000])
@pytest.mark.parametrize("into", ["hidden", "delta"])
def test_in_place(be, n, into):
    hidden, delta, weight = inputs(7, n, torch.bfloat16, n)
    h, v = oracle_norm(hidden, delta, weight, EPS)
    hd, dd = hidden.cuda(), delta.cuda()
    y = torch.zeros(7, n, device="cuda")
    be.rms_norm_rows(hd, weight.cuda(), EPS, y, delta=dd, hidden_out=hd if into == "hidden" else dd)
    assert torch.equal((hd if into == "hidden" else dd).cpu(), h)
    assert torch.equal((dd if into == "hidden" else hd).cpu(), delta if into == "hidden" else hidden)
    near(y, v, torch.float32)


def test_columns_of_one_buffer(be):
    """Operands side by side in one buffer, as slices of a fused projection are."""
    hidden, delta, weight = inputs(6, 128, torch.float32, 3)
    buf = torch.zeros(6, 384, device="cuda")
    buf[:, :128], buf[:, 128:256] = hidden.cuda(), delta.cuda()
    be.rms_norm_rows(buf[:, :128], weight.cuda(), EPS, buf[:, 256:], delta=buf[:, 128:256])
    _, v = oracle_norm(hidden, delta, weight, EPS)
    near(buf[:, 256:], v, torch.float32)


def test_many_rows_give_each_row_s_own_bits(be):
    hidden, delta, weight = inputs(2000, 1000, torch.float16, 8)
    outs = []
    for rows in (slice(0, 2000), slice(1234, 1235)):
        h, d = hidden[rows].cuda(), delta[rows].cuda()
        q, s = torch.zeros(h.shape, dtype=torch.int8, device="cuda"), torch.zeros(h.shape[0], device="cuda")
        y = torch.zeros(h.shape, device="cuda")
        be.rms_norm_i8_rows(h, weight.cuda(), EPS, q, s, y=y, delta=d)
        outs.append((q, s, y))
    for a, b in zip(*outs):
        assert torch.equal(a[1234], b[0])


def test_rows_far_apart(be):
    """Rows 2^24 elements apart: the last ones lie beyond 32 bits."""
    hidden, delta, weight = inputs(200, 640, torch.bfloat16, 9)
    h, v = oracle_norm(hidden, delta, weight, EPS)
    x = torch.empty(200 << 24, dtype=torch.bfloat16, device="cuda").view(200, 1 << 24)[:, :640]
    x.copy_(hidden)
    q, s = torch.zeros(200, 640, dtype=torch.int8, device="cuda"), torch.zeros(200, device="cuda")
    y = torch.empty(200 << 23, device="cuda").view(200, 1 << 23)[:, :640]
    be.rms_norm_i8_rows(x, weight.cuda(), EPS, q, s, y=y, delta=delta.cuda(), hidden_out=x)
    assert torch.equal(x.cpu(), h)
    near(y, v, torch.float32)
    q_want, s_want = oracle_i8(v)
    np.testing.assert_array_equal(s.cpu().numpy(), s_want)
    np.testing.assert_array_equal(q.cpu().numpy(), q_want)


def placements(be, hidden, delta, weight, y_ty):
    """hidden_out, y, int8 rows, their scales and (for widths that have them) Q8_K blocks of the same rows, at aligned
    addresses and strides and at odd ones."""
    rows, n = hidden.shape
    w_at = torch.empty(n + 1, device="cuda")
    outs = []
    for pad, offset in ((0, 0), (3, 1), (8, 5)):
        _, hd = strided(hidden, pad, offset)
        _, dd = strided(delta, pad, offset)
        w = w_at[offset & 1:][:n]
        w.copy_(weight)
        _, out = strided(torch.zeros_like(hidden), pad, offset)
        _, y = strided(torch.zeros(rows, n, dtype=y_ty), pad, offset)
        _, q = strided(torch.zeros(rows, n, dtype=torch.int8), pad, offset)
        s = torch.zeros(rows, device="cuda")
        be.rms_norm_i8_rows(hd, w, EPS, q, s, y=y, delta=dd, hidden_out=out)
        got = [out, y, q, s]
        if n % 256 == 0 and n <= 16384:
            enc = torch.zeros(rows, n // 256 * 292, dtype=torch.uint8, device="cuda")
            be.rms_norm_q8_k_rows(hd, w, EPS, enc, delta=dd)
            got.append(enc)
        outs.append([t.clone() for t in got])
    return outs


@pytest.mark.parametrize("ty,y_ty", [("f32", "f32"), ("f16", "bf16"), ("bf16", "f32"), ("f32", "f16")])
@pytest.mark.parametrize("rows,n", [(70, 8), (66, 255), (65, 512), (40, 1024), (31, 4096), (9, 8192), (5, 16384), (3, 33000)])
def test_bits_do_not_depend_on_the_placement(be, rows, n, ty, y_ty):
    hidden, delta, weight = inputs(rows, n, TYPES[ty], seed=n + 5)
    first, *others = placements(be, hidden, delta, weight, TYPES[y_ty])
    for other in others:
        assert all(torch.equal(a, b) for a, b in zip(first, other))


def test_sums_that_depend_on_their_order(be):
    """One value whose square is 1 among four million whose squares are just below half of that one's last bit in 64 bits: those
    that its lane adds to it one by one are lost, so r shows which elements a lane has.  With the elements of words of
    eight that share the large value's lane at zero, another assignment of elements to lanes moves r by 2^-43, which
    takes some 30 of these 16 million values over a rounding border of float32."""
    n, rows = 1 << 22, 4
    g = torch.Generator().manual_seed(1)
    x = 2.0 ** -27 * (1 + 0.35 * torch.rand(rows, n, generator=g))
    x.view(rows, n // 8192, 1024, 8)[:, :, 0] = 0.0
    x[:, 0] = 1.0
    weight = 1.0 + torch.rand(n, generator=g)
    outs = []
    for pad, offset in ((0, 0), (3, 1)):
        _, xd = strided(x, pad, offset)
        _, y = strided(torch.zeros(rows, n), pad, offset)
        be.rms_norm_rows(xd, weight.cuda(), 1e-30, y)
        outs.append(y.clone())
    assert torch.equal(outs[0], outs[1])
    _, v = oracle_norm(x, None, weight, 1e-30)
    near(outs[0], v, torch.float32)
