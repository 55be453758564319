"""What the entry points around a layer's int8 experts refuse, without a GPU: every check runs before the first HIP
call, so a context that is only a block of zeros (device 0) and addresses that are never followed suffice.  Each call
below is refused, or has nothing to do."""
import ctypes as C
import math

import pytest

import lbhip

A = 0x10000000   # an address far from every other one used here
M = 1 << 20
F32, F16, BF16 = lbhip.F32, lbhip.F16, lbhip.BF16


class Matrix(C.Structure):
    """The host side of an int8 matrix: device, rows, k, k tiles, channel groups, gated, and no memory."""
    _fields_ = [("device", C.c_int), ("rows", C.c_size_t), ("k", C.c_size_t), ("kt", C.c_size_t),
                ("groups", C.c_size_t), ("gated", C.c_int), ("tiles", C.c_void_p), ("scales", C.c_void_p),
                ("bytes", C.c_size_t)]


class Router(C.Structure):
    """The first members of a router: device, experts, width, weights and bias."""
    _fields_ = [("device", C.c_int), ("n_experts", C.c_size_t), ("hidden", C.c_size_t), ("w", C.c_void_p),
                ("bias", C.c_void_p), ("rest", C.c_uint8 * 256)]


class Layer(C.Structure):
    """The host side of a layer's experts, up to the k tiles."""
    _fields_ = [("device", C.c_int), ("n_experts", C.c_size_t), ("n", C.c_size_t), ("ffn", C.c_size_t),
                ("ffn_s", C.c_size_t), ("kt_n", C.c_size_t), ("kt_f", C.c_size_t), ("kt_fs", C.c_size_t),
                ("down_pitch", C.c_size_t), ("rest", C.c_uint8 * 256)]


@pytest.fixture()
def ctx():
    return C.cast(C.create_string_buffer(4096), C.c_void_p)


def status(fn, *args):
    err = lbhip.LbhError()
    st = fn(*args, C.byref(err))
    assert st == err.status
    return lbhip.STATUS[st], err


def norm(ctx, type=F32, block=A, bs=64, pw=A + M, pe=1e-6, gate=0, gs=64, act=0, scale=1.0, hidden=A + 2 * M, hs=64,
         ho=A + 3 * M, hos=64, w=A + 4 * M, eps=1e-5, rows=4, n=64, y_type=F32, y=0, ys=64, q=A + 5 * M, qs=64,
         scales=A + 6 * M, enc=0):
    return status(lbhip.lib().lbh_block_norm_rows, ctx, type, block, bs, pw, pe, gate, gs, act, scale, hidden, hs, ho,
                  hos, w, eps, rows, n, y_type, y, ys, q, qs, scales, enc)


@pytest.mark.parametrize("change,want", [
    (dict(block=0), "NullArgument"), (dict(hidden=0), "NullArgument"), (dict(ho=0), "NullArgument"),
    (dict(q=0), "NullArgument"), (dict(scales=0), "NullArgument"), (dict(w=0), "NullArgument"),
    (dict(q=0, scales=0), "NullArgument"),                                   # a norm without an output
    (dict(type=12), "UnsupportedType"), (dict(y=A + 7 * M, y_type=15), "UnsupportedType"),
    (dict(n=0), "ZeroLogicalElements"), (dict(n=16385, bs=1 << 15, hs=1 << 15, hos=1 << 15, qs=1 << 15), "UnsupportedShape"),
    (dict(rows=M + 1), "UnsupportedShape"), (dict(bs=1 << 41), "UnsupportedShape"), (dict(gate=A + 7 * M, gs=1 << 41), "UnsupportedShape"),
    (dict(enc=A + 7 * M), "LogicalElementsNotDivisible"),
    (dict(scale=math.nan), "InvalidParameter"), (dict(scale=math.inf), "InvalidParameter"),
    (dict(act=1), "InvalidParameter"), (dict(gate=A + 7 * M, act=3), "InvalidParameter"), (dict(gate=A + 7 * M, act=-1), "InvalidParameter"),
    (dict(pe=0.0), "InvalidParameter"), (dict(eps=math.nan), "InvalidParameter"), (dict(eps=math.inf), "InvalidParameter"),
    (dict(bs=63), "DimensionMismatch"), (dict(hs=0), "DimensionMismatch"), (dict(hos=63), "DimensionMismatch"),
    (dict(qs=63), "DimensionMismatch"), (dict(gate=A + 7 * M, gs=63), "DimensionMismatch"), (dict(y=A + 7 * M, ys=1), "DimensionMismatch"),
    (dict(block=A + 2), "InvalidParameter"), (dict(type=BF16, gate=A + 7 * M + 1), "InvalidParameter"),
    (dict(pw=A + M + 2), "InvalidParameter"), (dict(w=A + 4 * M + 1), "InvalidParameter"), (dict(scales=A + 6 * M + 2), "InvalidParameter"),
    # shared bytes: an output on an input or another output, the stream shifted against hidden
    (dict(q=A), "InvalidParameter"), (dict(q=A + 3 * M + 8), "InvalidParameter"), (dict(y=A + 2 * M), "InvalidParameter"),
    (dict(ho=A + 2 * M + 4), "InvalidParameter"), (dict(ho=A + 4), "InvalidParameter"), (dict(ho=A, hos=80), "InvalidParameter"),
    (dict(ho=A + 4 * M), "InvalidParameter"), (dict(scales=A + M), "InvalidParameter"),
    (dict(gate=A + 3 * M, gs=0), "InvalidParameter"), (dict(gate=A + 5 * M), "InvalidParameter"),
])
def test_block_norm_refusals(ctx, change, want):
    assert norm(ctx, **change)[0] == want


def test_block_norm_nothing_to_do(ctx):
    assert norm(ctx, rows=0)[0] == "Ok"
    assert norm(ctx, rows=0, block=0, hidden=0, ho=0)[0] == "Ok"
    assert norm(None)[0] == "NullArgument"


def act(ctx, m=True, device=0, rows=48, k=64, gated=0, x=A, xs=64, scales=A + M, tokens=4, a=3, bias=A + 2 * M, up=0, scale=1.0,
        y_type=F32, y=A + 3 * M, ys=48, residual=0, rs=48, ws=0, wl=0):
    mat = Matrix(device=device, rows=rows, k=k, kt=(k + 255) // 256 * 4, groups=(rows + 15) // 16, gated=gated)
    return status(lbhip.lib().lbh_gemm_i8_act, ctx, C.byref(mat) if m else None, x, xs, scales, tokens, a, bias, up, scale,
                  y_type, y, ys, residual, rs, ws, wl)


@pytest.mark.parametrize("change,want", [
    (dict(m=False), "NullArgument"), (dict(x=0), "NullArgument"), (dict(y=0), "NullArgument"),
    (dict(device=1), "InvalidParameter"), (dict(y_type=13), "UnsupportedType"),
    (dict(a=-1), "InvalidParameter"), (dict(a=6), "InvalidParameter"), (dict(scale=math.nan), "InvalidParameter"),
    (dict(scale=math.inf), "InvalidParameter"), (dict(scale=1e39), "InvalidParameter"),
    (dict(up=A + 4 * M), "InvalidParameter"),                                # not a pair
    (dict(gated=1, residual=A + 4 * M), "InvalidParameter"),                 # a pair
    (dict(bias=A + 2 * M + 2), "InvalidParameter"), (dict(gated=1, up=A + 4 * M + 1), "InvalidParameter"),
    (dict(bias=A + 3 * M + 4), "InvalidParameter"), (dict(gated=1, up=A + 3 * M), "InvalidParameter"),
    (dict(ys=47), "DimensionMismatch"), (dict(xs=63), "DimensionMismatch"), (dict(residual=A + 4 * M, rs=47), "DimensionMismatch"),
    (dict(x=A + 8), "NullArgument"), (dict(x=A + 8, ws=A + 2 * M, wl=4 * 256), "InvalidParameter"),   # the workspace on the bias
    (dict(x=A + 8, ws=A + 5 * M, wl=4 * 256 - 1), "ScratchTooSmall"),
])
def test_product_with_activation_refusals(ctx, change, want):
    assert act(ctx, **change)[0] == want


def test_product_with_activation_nothing_to_do(ctx):
    assert act(ctx, tokens=0)[0] == "Ok"
    assert act(None)[0] == "NullArgument"


def route(ctx, r=True, device=0, experts=48, hidden=512, bias=A, type=F32, x=A + M, xs=512, tokens=4, top_k=4, mode=1,
          scale=1.0, ids=A + 2 * M, coefs=A + 3 * M, logits=0, ws=A + 4 * M, wl=1 << 20):
    rt = Router(device=device, n_experts=experts, hidden=hidden, bias=bias)
    return status(lbhip.lib().lbh_router_route_rows, ctx, C.byref(rt) if r else None, type, x, xs, tokens, top_k, mode, scale,
                  ids, coefs, logits, ws, wl)


@pytest.mark.parametrize("change,want", [
    (dict(r=False), "NullArgument"), (dict(x=0), "NullArgument"), (dict(ids=0), "NullArgument"), (dict(coefs=0), "NullArgument"),
    (dict(ws=0), "NullArgument"), (dict(bias=0), "NullArgument"), (dict(type=12), "UnsupportedType"),
    (dict(device=1), "InvalidParameter"), (dict(mode=2), "InvalidParameter"), (dict(mode=-1), "InvalidParameter"),
    (dict(scale=math.nan), "InvalidParameter"), (dict(top_k=0), "UnsupportedShape"), (dict(top_k=17), "UnsupportedShape"),
    (dict(top_k=5, experts=4), "UnsupportedShape"), (dict(tokens=(1 << 19) + 1), "UnsupportedShape"),
    (dict(xs=1 << 41), "UnsupportedShape"), (dict(xs=511), "DimensionMismatch"), (dict(x=A + M + 2), "InvalidParameter"),
    (dict(ids=A + 2 * M + 1), "InvalidParameter"), (dict(ws=A + 4 * M + 4), "InvalidParameter"),
    (dict(wl=4 * 4 * 48 * 8 - 1), "ScratchTooSmall"), (dict(ids=A + 3 * M), "InvalidParameter"),
    (dict(coefs=A + M + 64), "InvalidParameter"), (dict(logits=A + 4 * M + 8), "InvalidParameter"), (dict(ws=A + M), "InvalidParameter"),
])
def test_route_refusals(ctx, change, want):
    assert route(ctx, **change)[0] == want


def test_route_nothing_to_do_and_sizes(ctx):
    assert route(ctx, tokens=0, x=0, ids=0)[0] == "Ok"
    assert route(None)[0] == "NullArgument"
    f = lbhip.lib().lbh_router_route_rows_workspace_bytes
    r = Router(n_experts=48, hidden=512)
    assert f(C.byref(r), 256) == 4 * 256 * 48 * 8 and f(C.byref(r), 257) == 257 * 48 * 8
    assert f(None, 4) == 0 and f(C.byref(r), (1 << 19) + 1) == 0


def layer(n=64, ffn=48, ffn_s=0, device=0):
    tiles = lambda k: (k + 255) // 256 * 4   # noqa: E731
    return Layer(device=device, n_experts=8, n=n, ffn=ffn, ffn_s=ffn_s, kt_n=tiles(n), kt_f=tiles(ffn),
                 kt_fs=tiles(ffn_s), down_pitch=(n + 15) // 16 * 16)


def moe(ctx, m=True, device=0, x=A, xs=64, scales=A + M, ids=A + 2 * M, coefs=A + 3 * M, tokens=4, top_k=2, y_type=F32,
        y=A + 4 * M, ys=64, residual=0, rs=64, ws=A + 5 * M, wl=8 * M):
    return status(lbhip.lib().lbh_moe_i8_forward, ctx, C.byref(layer(device=device)) if m else None, x, xs, scales, ids,
                  coefs, tokens, top_k, y_type, y, ys, residual, rs, ws, wl)


@pytest.mark.parametrize("change,want", [
    (dict(m=False), "NullArgument"), (dict(x=0), "NullArgument"), (dict(scales=0), "NullArgument"), (dict(ids=0), "NullArgument"),
    (dict(coefs=0), "NullArgument"), (dict(y=0), "NullArgument"), (dict(ws=0), "NullArgument"),
    (dict(device=1), "InvalidParameter"), (dict(y_type=8), "UnsupportedType"),
    (dict(tokens=257), "UnsupportedShape"), (dict(top_k=0), "UnsupportedShape"), (dict(top_k=17), "UnsupportedShape"),
    (dict(tokens=256, top_k=9), "UnsupportedShape"), (dict(xs=(1 << 23) + 1), "UnsupportedShape"), (dict(ys=1 << 41), "UnsupportedShape"),
    (dict(xs=63), "DimensionMismatch"), (dict(ys=63), "DimensionMismatch"), (dict(residual=A + 20 * M, rs=63), "DimensionMismatch"),
    (dict(scales=A + M + 2), "InvalidParameter"), (dict(ids=A + 2 * M + 1), "InvalidParameter"), (dict(coefs=A + 3 * M + 2), "InvalidParameter"),
    (dict(y=A + 4 * M + 2), "InvalidParameter"), (dict(ws=A + 5 * M + 8), "InvalidParameter"),
    (dict(y=A + 16), "InvalidParameter"), (dict(y=A + 2 * M), "InvalidParameter"), (dict(y=A + 3 * M), "InvalidParameter"),
    (dict(ws=A + 4 * M), "InvalidParameter"), (dict(ws=A), "InvalidParameter"), (dict(residual=A + 4 * M + 4), "InvalidParameter"),
    (dict(residual=A + 5 * M + 256), "InvalidParameter"),                    # in the workspace
])
def test_experts_refusals(ctx, change, want):
    assert moe(ctx, **change)[0] == want


def test_experts_nothing_to_do_and_sizes(ctx):
    assert moe(ctx, tokens=0, x=0, y=0, ws=0)[0] == "Ok"
    assert moe(None)[0] == "NullArgument"
    L = lbhip.lib()
    f = L.lbh_moe_i8_workspace_bytes
    need = f(C.byref(layer()), 4, 2)
    assert need > 0 and moe(ctx, wl=need - 1)[0] == "ScratchTooSmall"
    st, err = moe(ctx, wl=5)
    assert (st, err.expected, err.actual) == ("ScratchTooSmall", need, 5)
    assert f(None, 4, 2) == 0 and f(C.byref(layer()), 257, 1) == 0 and f(C.byref(layer()), 256, 9) == 0 and f(C.byref(layer()), 0, 2) == 0
    assert f(C.byref(layer(ffn_s=64)), 4, 2) > need
    assert L.lbh_moe_i8_destroy(None) == 0


def pointers(*mats):
    return (C.c_void_p * len(mats))(*(C.addressof(m) if m is not None else None for m in mats))


def test_layer_creation_refusals(ctx):
    new, h = lbhip.lib().lbh_moe_i8_create, C.c_void_p()

    def mats(n=64, ffn=48, device=0):
        return (Matrix(device=device, rows=ffn, k=n, kt=4, groups=3, gated=1), Matrix(device=device, rows=n, k=ffn, kt=4, groups=4))

    up, down = mats()

    def create(ups, downs, count=None, su=None, sd=None, c=ctx):
        keep = pointers(*ups), pointers(*downs)
        return status(new, c, *keep, len(ups) if count is None else count, C.byref(su) if su else None,
                      C.byref(sd) if sd else None, C.byref(h))[0]

    assert create([up], [down], c=None) == "NullArgument"
    assert create([up], [down], count=0) == "DimensionMismatch"
    assert create([up], [down], count=1025) == "UnsupportedShape"
    assert create([None], [down]) == "NullArgument" and create([up], [None]) == "NullArgument"
    assert create([up, up], [down, None]) == "NullArgument"
    assert create([up], [down], su=up) == "NullArgument" and create([up], [down], sd=down) == "NullArgument"
    assert create([down], [down]) == "InvalidParameter" and create([up], [up]) == "InvalidParameter"
    other = mats(device=1)
    assert create([up, other[0]], [down, down]) == "InvalidParameter"
    assert create([up], [down], su=down, sd=down) == "InvalidParameter"
    wide, tall = mats(n=80), mats(ffn=64)
    assert create([up, wide[0]], [down, wide[1]]) == "DimensionMismatch"
    assert create([up, tall[0]], [down, tall[1]]) == "DimensionMismatch"
    assert create([up], [tall[1]]) == "DimensionMismatch"
    assert create([up], [down], su=wide[0], sd=wide[1]) == "DimensionMismatch"
    assert create([up], [down], su=tall[0], sd=down) == "DimensionMismatch"
    assert not h.value


def test_python_names_are_the_library_s():
    header = (lbhip.PKG_DIR.parent / "include" / "lightbridge_hip.h").read_text()
    for name, value in lbhip.ACTIVATIONS.items():
        assert f"LBH_ACT_{name.upper()} = {value}," in header
    for name, value in lbhip.GATE_ACTS.items():
        assert f"LBH_GATE_{'AS_IS' if name == 'none' else name.upper()} = {value}," in header
