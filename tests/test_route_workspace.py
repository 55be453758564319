"""One workspace for routing calls of any number of rows up to a largest: what lbh_router_route_rows_workspace_bytes_up_to gives
is enough for each of them (every check runs before the first HIP call, so no GPU is needed), and no more than the
largest of their needs."""
import ctypes as C

import pytest

import lbhip
from test_layer_refusals import M, Router, ctx, route   # noqa: F401 (ctx: a fixture)


@pytest.mark.parametrize("experts", [1, 48, 256])
@pytest.mark.parametrize("most", [0, 1, 75, 255, 256, 257, 300, 1023, 1024, 1025, 5000, 1 << 19])
def test_it_is_the_most_that_a_smaller_call_needs(most, experts):
    r = Router(n_experts=experts, hidden=512)
    exact, up_to = lbhip.lib().lbh_router_route_rows_workspace_bytes, lbhip.lib().lbh_router_route_rows_workspace_bytes_up_to
    counts = range(most + 1) if most <= 5000 else [*range(2000), most - 1, most]
    assert up_to(C.byref(r), most) == max(exact(C.byref(r), n) for n in counts)


def test_nothing_for_no_router_and_too_many_rows():
    up_to = lbhip.lib().lbh_router_route_rows_workspace_bytes_up_to
    assert up_to(None, 4) == 0 and up_to(C.byref(Router(n_experts=48, hidden=512)), (1 << 19) + 1) == 0


def test_it_grows_with_the_rows():
    r = Router(n_experts=48, hidden=512)
    up_to = lbhip.lib().lbh_router_route_rows_workspace_bytes_up_to
    sizes = [up_to(C.byref(r), n) for n in range(0, 3000)]
    assert sizes == sorted(sizes)


@pytest.mark.parametrize("tokens", [1, 76, 255, 256, 257, 300])
def test_no_smaller_call_finds_it_too_small(ctx, tokens):   # noqa: F811
    """A refusal for another reason (an output in the workspace) comes behind the check of its size."""
    need = lbhip.lib().lbh_router_route_rows_workspace_bytes_up_to(C.byref(Router(n_experts=48, hidden=512)), 300)
    # x far from everything: rows of 300 * 512 floats
    st, _ = route(ctx, tokens=tokens, x=1 << 40, wl=need, ws=(1 << 41), ids=1 << 42, coefs=1 << 42)
    assert st == "InvalidParameter"   # ids and coefs in one place
