"""The norms around a block (block output into the stream, gate, scale, next norm) against a plain 64-bit
implementation.

The stream is held to its formula within its roundings (to 32 bits and to the rows' type, half a step each) and what
the activated gate is off by: 2^-38 of the product it enters (the sigmoid is good to 2^-39).  What follows is held to
the formula of the stream as stored: int8 values and scales equal, rows within their roundings."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
PE, EPS, SCALE = 1e-6, 1e-5, 0.37


@pytest.fixture(scope="module")
def be():
    import lbhip
    if not torch.cuda.is_available():
        pytest.fail("no GPU visible")
    b = lbhip.HipBackend(0)
    yield b
    b.close()


def strided(t, pad=0, offset=0):
    rows, n = t.shape
    buf = torch.full((rows * (n + pad) + offset + 8,), 77, dtype=t.dtype, device="cuda")
    view = buf[offset:offset + rows * (n + pad)].view(rows, n + pad)[:, :n]
    view.copy_(t)
    return buf, view


def rms(v, weight, eps):
    with np.errstate(all="ignore"):
        return v * weight.double().numpy() / np.sqrt((v * v).mean(axis=1, keepdims=True) + eps)


def oracle_stream(x, act):
    """(h, |scale * a(gate) * p|) in 64 bits."""
    p = x["block"].double().numpy()
    if x["post"] is not None:
        p = rms(p, x["post"], PE)
    if x["gate"] is not None:
        g = x["gate"].double().numpy()
        with np.errstate(all="ignore"):
            s = 1.0 / (1.0 + np.exp(-g))
        p = p * {"none": g, "sigmoid": s, "silu": g * s}[act]
    return x["hidden"].double().numpy() + SCALE * p, np.abs(SCALE * p)


def oracle_i8(v):
    with np.errstate(all="ignore"):
        s = (np.abs(v).max(axis=1) / 127.0).astype(np.float32)
        s = np.where(np.isfinite(v).all(axis=1) & np.isfinite(s), s, np.float32("nan"))
        s = np.where(s < np.float32(2.0 ** -126), np.float32(0), s)
        q = np.rint(v / np.where(s > 0, s, 1).astype(np.float64)[:, None])
    return np.where((s > 0)[:, None], q, 0).astype(np.int8), s


def near(got, v, ty, more=0.0):
    steps = 2.0 ** -24 + (0 if ty == torch.float32 else torch.finfo(ty).eps / 2 * (1 + 2.0 ** -24))
    least = torch.finfo(ty).smallest_normal * torch.finfo(ty).eps / 2
    g = got.double().cpu().numpy()
    np.testing.assert_array_less(np.abs(g - v), np.abs(v) * (steps + 1e-12) + more * (1 + steps) + least * 1.01 + 1e-300)


def inputs(rows, n, ty, seed, post=True, gate="silu"):
    g = torch.Generator().manual_seed(seed)
    size = torch.exp(torch.randn(n, generator=g))
    return {"block": (3 * torch.randn(rows, n, generator=g)).to(ty), "hidden": (torch.randn(rows, n, generator=g) * size).to(ty),
            "gate": None if gate is None else (2 * torch.randn(1 if gate == "row" else rows, n, generator=g)).to(ty),
            "post": 1.0 + 0.3 * torch.randn(n, generator=g) if post else None, "weight": 1.0 + 0.3 * torch.randn(n, generator=g)}


def call(be, x, act, after, pad=0, offset=0, **outs):
    put = {k: strided(x[k], pad, offset)[1] for k in ("block", "hidden")}
    gate = None
    if x["gate"] is not None:
        gate = strided(x["gate"], pad, offset)[1]
    be.block_norm_rows(put["block"], put["hidden"], after, post_weight=None if x["post"] is None else x["post"].cuda(),
                       post_eps=PE, gate=gate, gate_act=act, scale=SCALE, weight=x["weight"].cuda(), eps=EPS, **outs)


SHAPES = [(1, 1), (3, 7), (2, 8), (5, 64), (9, 511), (7, 512), (4, 513), (2, 1000), (1, 4096), (33, 2048), (6, 4095), (3, 4097),
          (2, 8192), (2, 8199), (3, 16384), (2, 16383)]


@pytest.mark.parametrize("ty", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,n", SHAPES)
def test_stream_rows_and_int8(be, rows, n, ty):
    t = TYPES[ty]
    for i, (post, gate, act) in enumerate(((True, None, "none"), (True, "rows", "silu"), (False, "rows", "sigmoid"),
                                           (True, "row", "none"), (False, None, "none"))):
        x = inputs(rows, n, t, rows * 1009 + n + i, post, gate)
        want, moved = oracle_stream(x, act)
        for pad, offset in ((0, 0), (3, 1)):
            out_buf, out = strided(torch.zeros(rows, n, dtype=t), pad, offset)
            y_buf, y = strided(torch.zeros(rows, n, dtype=t), pad, offset)
            q_buf, q = strided(torch.zeros(rows, n, dtype=torch.int8), pad, offset)
            s = torch.full((rows,), -1.0, device="cuda")
            call(be, x, act, out, pad, offset, y=y, q=q, scales=s)
            torch.cuda.synchronize()
            near(out, want, t, moved * (2.0 ** -38 if act in ("silu", "sigmoid") else 1e-14))
            v = rms(out.double().cpu().numpy(), x["weight"], EPS)
            q_want, s_want = oracle_i8(v)
            np.testing.assert_array_equal(s.cpu().numpy(), s_want)
            np.testing.assert_array_equal(q.cpu().numpy(), q_want)
            near(y, v, t)
            for buf in (out_buf, y_buf, q_buf):   # bytes around the rows are left alone
                rest = buf.clone()
                rest[offset:offset + rows * (n + pad)].view(rows, n + pad)[:, :n] = 77
                assert bool((rest == 77).all())


@pytest.mark.parametrize("y_ty", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n", [96, 1023, 4096])
def test_rows_in_every_type_and_the_stream_alone(be, y_ty, n):
    x = inputs(5, n, torch.bfloat16, n)
    out, alone = (torch.zeros(5, n, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    y = torch.zeros(5, n, dtype=TYPES[y_ty], device="cuda")
    call(be, x, "silu", out, y=y)
    near(y, rms(out.double().cpu().numpy(), x["weight"], EPS), TYPES[y_ty])
    be.block_norm_rows(x["block"].cuda(), x["hidden"].cuda(), alone, post_weight=x["post"].cuda(), post_eps=PE,
                       gate=x["gate"].cuda(), gate_act="silu", scale=SCALE)
    assert torch.equal(alone, out)


@pytest.mark.parametrize("rows,n", [(1, 256), (3, 512), (2, 1024), (5, 4096), (2, 7168), (2, 16384)])
def test_q8_k_is_the_quantizer_s_of_its_rows(be, oracle, rows, n):
    x = inputs(rows, n, torch.float32, n)
    out, y = torch.zeros(rows, n, device="cuda"), torch.zeros(rows, n, device="cuda")
    enc = torch.full((rows + 1, n // 256 * 292), 9, dtype=torch.uint8, device="cuda")
    call(be, x, "sigmoid", out, y=y, encoded=enc[:rows])
    torch.cuda.synchronize()
    near(y, rms(out.double().cpu().numpy(), x["weight"], EPS), torch.float32)
    for r in range(rows):
        np.testing.assert_array_equal(enc[r].cpu().numpy(), oracle.quantize_q8_k(y[r].cpu().numpy()))
    assert bool((enc[rows] == 9).all())
    # beside int8 rows in the same call
    both, q, s = torch.zeros_like(enc[:rows]), torch.zeros(rows, n, dtype=torch.int8, device="cuda"), torch.zeros(rows, device="cuda")
    call(be, x, "sigmoid", out, q=q, scales=s, encoded=both)
    assert torch.equal(both, enc[:rows])
    q_want, s_want = oracle_i8(rms(out.double().cpu().numpy(), x["weight"], EPS))
    np.testing.assert_array_equal(q.cpu().numpy(), q_want)
    np.testing.assert_array_equal(s.cpu().numpy(), s_want)


def test_without_gate_and_norm_it_is_the_residual_s_addition(be):
    """scale 1, no norm behind the block, no gate: bit for bit the stream, rows and int8 rows of rms_norm_i8_rows."""
    for ty in TYPES.values():
        x = inputs(37, 1000, ty, 3, post=False, gate=None)
        w, hid, blk = x["weight"].cuda(), x["hidden"].cuda(), x["block"].cuda()
        got = [torch.zeros_like(hid), torch.zeros(37, 1000, dtype=torch.int8, device="cuda"), torch.zeros(37, device="cuda")]
        want = [torch.zeros_like(t) for t in got]
        be.block_norm_rows(blk, hid, got[0], weight=w, eps=EPS, q=got[1], scales=got[2])
        be.rms_norm_i8_rows(hid, w, EPS, want[1], want[2], delta=blk, hidden_out=want[0])
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("n", [64, 520, 4095, 16384])
@pytest.mark.parametrize("into", ["hidden", "block"])
def test_in_place(be, n, into):
    x = inputs(7, n, torch.bfloat16, n)
    apart = torch.zeros(7, n, dtype=torch.bfloat16, device="cuda")
    y0, y1 = torch.zeros(7, n, device="cuda"), torch.zeros(7, n, device="cuda")
    args = dict(post_weight=x["post"].cuda(), post_eps=PE, gate=x["gate"].cuda(), gate_act="silu", scale=SCALE,
                weight=x["weight"].cuda(), eps=EPS)
    blk, hid = x["block"].cuda(), x["hidden"].cuda()
    be.block_norm_rows(blk, hid, apart, y=y0, **args)
    be.block_norm_rows(blk, hid, hid if into == "hidden" else blk, y=y1, **args)
    assert torch.equal(apart, hid if into == "hidden" else blk) and torch.equal(y0, y1)
    assert torch.equal((blk if into == "hidden" else hid).cpu(), x["block" if into == "hidden" else "hidden"])


@pytest.mark.parametrize("ty", ["f32", "bf16"])
@pytest.mark.parametrize("rows,n", [(70, 8), (300, 255), (65, 512), (40, 1024), (9, 4095), (5, 8200)])
def test_bits_do_not_depend_on_the_placement_or_the_batch(be, rows, n, ty):
    x = inputs(rows, n, TYPES[ty], n + 5)
    outs = []
    for pad, offset in ((0, 0), (3, 1), (8, 5)):
        _, out = strided(torch.zeros(rows, n, dtype=TYPES[ty]), pad, offset)
        _, q = strided(torch.zeros(rows, n, dtype=torch.int8), pad, offset)
        s, y = torch.zeros(rows, device="cuda"), torch.zeros(rows, n, device="cuda")
        call(be, x, "silu", out, pad, offset, y=y, q=q, scales=s)
        outs.append([t.clone() for t in (out, q, s, y)])
    for other in outs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(outs[0], other))
    one = {k: v[rows - 2:rows - 1] if v is not None and v.ndim == 2 else v for k, v in x.items()}
    out, y = torch.zeros(1, n, dtype=TYPES[ty], device="cuda"), torch.zeros(1, n, device="cuda")
    call(be, one, "silu", out, y=y)
    assert torch.equal(out[0], outs[0][0][rows - 2]) and torch.equal(y[0], outs[0][3][rows - 2])


@pytest.mark.parametrize("n", [60, 515, 4096])
def test_values_that_are_zero_large_or_not_finite(be, n):
    """What is not finite stays in its row; zero rows, gates far out, and rows that cancel to nothing."""
    rows = 9
    x = inputs(rows, n, torch.float32, n)
    x["block"][0] = 0.0
    x["block"][1, 3], x["hidden"][2, n - 1], x["gate"][3, 0] = float("nan"), float("inf"), float("nan")
    x["gate"][4, 0], x["gate"][4, 1], x["gate"][4, 2] = 1e30, -1e30, float("inf")
    x["gate"][5, :4] = torch.tensor([-700.0, -708.5, -745.0, 710.0])
    x["hidden"][6], x["block"][6] = 0.0, 0.0
    x["block"][7] = 1e25
    x["gate"][8, 5] = float("-inf")
    for act in ("sigmoid", "silu", "none"):
        out, y = torch.zeros(rows, n, device="cuda"), torch.zeros(rows, n, device="cuda")
        q, s = torch.zeros(rows, n, dtype=torch.int8, device="cuda"), torch.zeros(rows, device="cuda")
        call(be, x, act, out, y=y, q=q, scales=s)
        with np.errstate(all="ignore"):
            want, moved = oracle_stream(x, act)
        got = out.double().cpu().numpy()
        np.testing.assert_array_equal(np.isnan(got), np.isnan(want))
        fine = np.isfinite(want) & (np.abs(want) < 3e38)
        near(out[torch.from_numpy(fine).cuda()], want[fine], torch.float32, moved[fine] * 2.0 ** -38)
        np.testing.assert_array_equal(got[~fine & ~np.isnan(want)], np.float32(want[~fine & ~np.isnan(want)]).astype(np.float64))
        q_want, s_want = oracle_i8(rms(got, x["weight"], EPS))
        np.testing.assert_array_equal(s.cpu().numpy(), s_want)
        np.testing.assert_array_equal(q.cpu().numpy(), q_want)


def test_rows_far_apart(be):
    """Rows 2^24 elements apart: the last ones lie beyond 32 bits."""
    x = inputs(200, 640, torch.bfloat16, 9)
    want, moved = oracle_stream(x, "silu")
    far = torch.empty(200 << 24, dtype=torch.bfloat16, device="cuda").view(200, 1 << 24)[:, :640]
    far.copy_(x["hidden"])
    y = torch.empty(200 << 23, device="cuda").view(200, 1 << 23)[:, :640]
    be.block_norm_rows(x["block"].cuda(), far, far, post_weight=x["post"].cuda(), post_eps=PE, gate=x["gate"].cuda(),
                       gate_act="silu", scale=SCALE, weight=x["weight"].cuda(), eps=EPS, y=y)
    near(far, want, torch.bfloat16, moved * 2.0 ** -38)
    near(y, rms(far.double().cpu().numpy(), x["weight"], EPS), torch.float32)
