"""What the dense-block entry points refuse, without a GPU: every check runs before the first HIP call, so a context
that is only a block of zeros (device 0) and addresses that are never followed suffice.  Each call below is refused,
or has nothing to do."""
import ctypes as C
import math

import pytest

import lbhip

A = 0x10000000   # an address far from every other one used here
F32, F16, BF16 = lbhip.F32, lbhip.F16, lbhip.BF16


class Matrix(C.Structure):
    """The host side of an int8 matrix: device, rows, k, k tiles, channel groups, gated, and no memory."""
    _fields_ = [("device", C.c_int), ("rows", C.c_size_t), ("k", C.c_size_t), ("kt", C.c_size_t),
                ("groups", C.c_size_t), ("gated", C.c_int), ("tiles", C.c_void_p), ("scales", C.c_void_p),
                ("bytes", C.c_size_t)]


@pytest.fixture()
def ctx():
    return C.cast(C.create_string_buffer(4096), C.c_void_p)


def status(fn, *args):
    err = lbhip.LbhError()
    st = fn(*args, C.byref(err))
    assert st == err.status
    return lbhip.STATUS[st], err


def norm(ctx, kind="i8", type=F32, hidden=A, hs=64, delta=0, ds=64, weight=A + (1 << 20), eps=1e-5, rows=4, n=64,
         ho=0, hos=64, y_type=F32, y=0, ys=64, q=A + (2 << 20), qs=64, scales=A + (3 << 20), encoded=A + (4 << 20)):
    L = lbhip.lib()
    head = (ctx, type, hidden, hs, delta, ds, weight, eps, rows, n, ho, hos, y_type, y, ys)
    if kind == "rows":
        return status(L.lbh_rms_norm_rows, *head)
    if kind == "q8_k":
        return status(L.lbh_rms_norm_q8_k_rows, *head, encoded)
    return status(L.lbh_rms_norm_i8_rows, *head, q, qs, scales)


@pytest.mark.parametrize("change,want", [
    (dict(hidden=0), "NullArgument"), (dict(weight=0), "NullArgument"), (dict(q=0), "NullArgument"),
    (dict(scales=0), "NullArgument"), (dict(kind="rows"), "NullArgument"),
    (dict(kind="q8_k", encoded=0, n=256), "NullArgument"),
    (dict(type=12), "UnsupportedType"), (dict(y=A + (5 << 20), y_type=15), "UnsupportedType"),
    (dict(n=0), "ZeroLogicalElements"), (dict(kind="q8_k", n=0), "ZeroLogicalElements"),
    (dict(kind="q8_k", n=255), "LogicalElementsNotDivisible"),
    (dict(kind="q8_k", n=16640, hs=16640), "UnsupportedShape"),
    (dict(eps=0.0), "InvalidParameter"), (dict(eps=-1.0), "InvalidParameter"), (dict(eps=math.inf), "InvalidParameter"),
    (dict(eps=math.nan), "InvalidParameter"),
    (dict(n=(1 << 23) + 1, hs=1 << 24), "UnsupportedShape"), (dict(rows=(1 << 20) + 1), "UnsupportedShape"),
    (dict(hs=1 << 41), "UnsupportedShape"),
    (dict(hs=63), "DimensionMismatch"), (dict(qs=63), "DimensionMismatch"),
    (dict(delta=A + (5 << 20), ds=32), "DimensionMismatch"), (dict(ho=A + (5 << 20), hos=1), "DimensionMismatch"),
    (dict(y=A + (5 << 20), ys=0), "DimensionMismatch"),
    (dict(hidden=A + 2), "InvalidParameter"), (dict(type=BF16, hidden=A + 1), "InvalidParameter"),
    (dict(weight=A + (1 << 20) + 2), "InvalidParameter"), (dict(scales=A + (3 << 20) + 1), "InvalidParameter"),
    # shared bytes: output on input, output on output, hidden_out shifted by one element
    (dict(q=A), "InvalidParameter"), (dict(q=A + 4 * 64 * 4 - 1), "InvalidParameter"),
    (dict(y=A, y_type=F32), "InvalidParameter"), (dict(ho=A + 4), "InvalidParameter"),
    (dict(ho=A, hos=65), "InvalidParameter"),
    (dict(scales=A + (2 << 20) + 8), "InvalidParameter"), (dict(q=A + (1 << 20) + 7), "InvalidParameter"),
    (dict(delta=A + (5 << 20), y=A + (5 << 20)), "InvalidParameter"),
])
def test_norm_refusals(ctx, change, want):
    assert norm(ctx, **change)[0] == want


def test_norm_nothing_to_do(ctx):
    for kind in ("i8", "q8_k"):
        assert norm(ctx, kind=kind, rows=0, n=256)[0] == "Ok"
    assert norm(ctx, kind="rows", y=A + (5 << 20), rows=0)[0] == "Ok"
    assert norm(None)[0] == "NullArgument"


def test_quantize_refusals(ctx):
    fn = lbhip.lib().lbh_quantize_i8_rows
    q, s = A + (2 << 20), A + (3 << 20)
    assert status(fn, None, F32, A, 64, 4, 64, q, 64, s)[0] == "NullArgument"
    assert status(fn, ctx, F32, 0, 64, 4, 64, q, 64, s)[0] == "NullArgument"
    assert status(fn, ctx, 21, A, 64, 4, 64, q, 64, s)[0] == "UnsupportedType"
    assert status(fn, ctx, F16, A, 10, 4, 64, q, 64, s)[0] == "DimensionMismatch"
    assert status(fn, ctx, F16, A, 64, 4, 64, A + 64, 64, s)[0] == "InvalidParameter"
    assert status(fn, ctx, F16, A, 64, 0, 64, q, 64, s)[0] == "Ok"


def product(ctx, gated_call=False, m=True, device=0, rows=48, k=64, gated=0, x=A, xs=64, scales=A + (1 << 20), tokens=4,
            y_type=F32, y=A + (2 << 20), ys=48, residual=0, rs=48, ws=0, wl=0):
    mat = Matrix(device=device, rows=rows, k=k, kt=(k + 127) // 128 * 2, groups=(rows + 15) // 16, gated=gated)
    mp = C.byref(mat) if m else None
    L = lbhip.lib()
    if gated_call:
        return status(L.lbh_gemm_i8_swiglu, ctx, mp, x, xs, scales, tokens, y_type, y, ys, ws, wl)
    return status(L.lbh_gemm_i8, ctx, mp, x, xs, scales, tokens, y_type, y, ys, residual, rs, ws, wl)


@pytest.mark.parametrize("change,want", [
    (dict(m=False), "NullArgument"), (dict(x=0), "NullArgument"), (dict(scales=0), "NullArgument"),
    (dict(y=0), "NullArgument"),
    (dict(gated=1), "InvalidParameter"), (dict(gated_call=True), "InvalidParameter"),
    (dict(device=1), "InvalidParameter"), (dict(y_type=13), "UnsupportedType"),
    (dict(tokens=(1 << 20) + 1), "UnsupportedShape"), (dict(xs=(1 << 23) + 16), "UnsupportedShape"),
    (dict(ys=1 << 41), "UnsupportedShape"),
    (dict(xs=48), "DimensionMismatch"), (dict(ys=47), "DimensionMismatch"),
    (dict(residual=A + (3 << 20), rs=40), "DimensionMismatch"),
    (dict(scales=A + (1 << 20) + 2), "InvalidParameter"), (dict(y=A + (2 << 20) + 2), "InvalidParameter"),
    (dict(y_type=BF16, residual=A + (3 << 20) + 1), "InvalidParameter"),
    (dict(y=A + 128), "InvalidParameter"), (dict(y=A + (1 << 20) - 16), "InvalidParameter"),
    (dict(residual=A + (2 << 20) + 4), "InvalidParameter"),          # y shifted against the residual
    (dict(residual=A + (2 << 20), rs=64), "InvalidParameter"),       # the same start, other rows
    # rows off 16 bytes need the workspace, aligned, large enough and apart from the operands
    (dict(x=A + 8), "NullArgument"), (dict(xs=72), "NullArgument"), (dict(k=60), "NullArgument"),
    (dict(x=A + 8, ws=A + (4 << 20) + 4, wl=1 << 20), "InvalidParameter"),
    (dict(x=A + 8, ws=A + (4 << 20), wl=4 * 128 - 1), "ScratchTooSmall"),
    (dict(x=A + 8, ws=A + 16, wl=4 * 128), "InvalidParameter"),
    (dict(x=A + 8, ws=A + (2 << 20) + 16, wl=4 * 128), "InvalidParameter"),
])
def test_product_refusals(ctx, change, want):
    assert product(ctx, **change)[0] == want


def test_product_nothing_to_do_and_sizes(ctx):
    assert product(ctx, tokens=0)[0] == "Ok"
    assert product(None)[0] == "NullArgument"
    st, err = product(ctx, x=A + 8, ws=A + (4 << 20), wl=100)
    assert (st, err.expected, err.actual) == ("ScratchTooSmall", 4 * 128, 100)
    m = Matrix(rows=48, k=130, kt=4, groups=3)
    L = lbhip.lib()
    assert L.lbh_gemm_i8_workspace_bytes(C.byref(m), 5) == 5 * 256
    assert L.lbh_gemm_i8_workspace_bytes(None, 5) == 0
    assert L.lbh_gemm_i8_workspace_bytes(C.byref(m), (1 << 20) + 1) == 0


def test_matrix_refusals(ctx):
    L, h = lbhip.lib(), C.c_void_p()
    new, pair = L.lbh_i8_matrix_create, L.lbh_i8_matrix_create_gated
    assert status(new, None, 4, 4, A, A, 1, C.byref(h))[0] == "NullArgument"
    assert status(new, ctx, 4, 4, 0, A, 1, C.byref(h))[0] == "NullArgument"
    assert status(new, ctx, 4, 4, A, 0, 1, C.byref(h))[0] == "NullArgument"
    assert status(new, ctx, 4, 0, A, A, 1, C.byref(h))[0] == "ZeroLogicalElements"
    assert status(new, ctx, 0, 4, A, A, 1, C.byref(h))[0] == "DimensionMismatch"
    assert status(new, ctx, 4, 131072, A, A, 1, C.byref(h))[0] == "UnsupportedShape"
    assert status(new, ctx, (1 << 26) + 1, 4, A, A, 1, C.byref(h))[0] == "UnsupportedShape"
    assert status(pair, ctx, 4, 4, A, A, 0, A, 1, C.byref(h))[0] == "NullArgument"
    assert status(pair, ctx, 4, 4, A, A, A, 0, 1, C.byref(h))[0] == "NullArgument"
    assert not h.value
    assert status(new, ctx, 4, 4, A, A + 2, 1, C.byref(h))[0] == "InvalidParameter"
    assert status(pair, ctx, 4, 4, A, A, A, A + 1, 1, C.byref(h))[0] == "InvalidParameter"
    m = Matrix(rows=4, k=8, kt=2, groups=1)
    read = L.lbh_i8_matrix_read
    assert status(read, ctx, None, 0, A, 32, A, 4)[0] == "NullArgument"
    assert status(read, ctx, C.byref(m), 1, A, 32, A, 4)[0] == "InvalidParameter"
    assert status(read, ctx, C.byref(m), 0, A, 31, A, 4)[0] == "OutputLengthMismatch"
    assert status(read, ctx, C.byref(m), 0, A, 32, A, 5)[0] == "OutputLengthMismatch"
    assert status(L.lbh_i8_matrix_from_packed, ctx, None, None, C.byref(h))[0] == "NullArgument"
    assert L.lbh_i8_matrix_destroy(None) == 0


def test_the_form_knob_s_range(ctx):
    fn = lbhip.lib().lbh_ctx_set_tuning
    be = lbhip.HipBackend
    assert [fn(ctx, be.TUNE_I8_FORM, v) for v in (-1, 12)] == [25, 25]
    assert [fn(ctx, be.TUNE_I8_FORM, v) for v in (1, 11, 0)] == [0, 0, 0]


def test_tensors_of_another_device():
    """The Python calls take tensors of their backend's GPU only."""
    torch = pytest.importorskip("torch")

    class Elsewhere:
        def __init__(self, t, device):
            self.t, self.device = t, device

        def get_device(self):
            return self.device

        def __getattr__(self, name):
            return getattr(self.t, name)

    rows, scales = torch.zeros(2, 4), torch.zeros(2)
    assert lbhip._rows(1, Elsewhere(rows, 1), (2, 4)) == (rows.data_ptr(), 4)
    assert lbhip._vector(1, Elsewhere(scales, 1), 2, torch.float32, "scales") == scales.data_ptr()
    assert lbhip._space(1, Elsewhere(rows, 1)) == (rows.data_ptr(), 32)
    for device in (-1, 1):
        with pytest.raises(AssertionError):
            lbhip._rows(0, Elsewhere(rows, device), (2, 4))
        with pytest.raises(AssertionError):
            lbhip._vector(0, Elsewhere(scales, device), 2, torch.float32, "scales")
        with pytest.raises(AssertionError):
            lbhip._space(0, Elsewhere(rows, device))
