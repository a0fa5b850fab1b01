"""Tokens to experts and back, what needs no GPU: the refusals of the entry points and of the Python operators."""
import ctypes

import pytest
import torch

import void_b200 as void
from void_b200 import _lib

BAD_ARG, ALIGN, SHAPE, WORKSPACE, TOO_LARGE = -1, -2, -3, -6, -8
AT = 4096   # (an address that nothing reads)


def _call(name, order, base, **bad):
    v = dict(base, **bad)
    return getattr(_lib.load(), name)(*[v[k] for k in order])


ROUTE = "scores elem lds rows n_experts top normalize experts weights stream".split()
ROUTE_BASE = dict(scores=AT, elem=0, lds=16, rows=4, n_experts=16, top=2, normalize=1, experts=AT, weights=AT, stream=None)


@pytest.mark.parametrize("bad, status", [
    (dict(scores=None), BAD_ARG), (dict(experts=None), BAD_ARG), (dict(weights=None), BAD_ARG), (dict(elem=3), BAD_ARG), (dict(rows=-1), BAD_ARG),
    (dict(n_experts=0), BAD_ARG), (dict(top=0), BAD_ARG), (dict(top=17), SHAPE), (dict(n_experts=1025), TOO_LARGE), (dict(top=33, n_experts=64), TOO_LARGE),
    (dict(rows=2 ** 31), TOO_LARGE), (dict(lds=-1), SHAPE), (dict(rows=0), 0),
])
def test_route_refuses(bad, status):
    assert _call("void_route", ROUTE, ROUTE_BASE, **bad) == status


GRAD = "scores elem lds rows n_experts top normalize g ldg ds ldd stream".split()
GRAD_BASE = dict(scores=AT, elem=0, lds=16, rows=4, n_experts=16, top=2, normalize=1, g=AT, ldg=2, ds=AT, ldd=16, stream=None)


@pytest.mark.parametrize("bad, status", [
    (dict(g=None), BAD_ARG), (dict(ds=None), BAD_ARG), (dict(ldd=15), SHAPE), (dict(top=17), SHAPE), (dict(n_experts=1025, ldd=1025), TOO_LARGE), (dict(rows=0), 0),
])
def test_route_grad_refuses(bad, status):
    assert _call("void_route_grad", GRAD, GRAD_BASE, **bad) == status


SORT = "experts index_bytes count n_experts offsets position ws ws_bytes stream".split()
SORT_BASE = dict(experts=AT, index_bytes=4, count=100, n_experts=8, offsets=AT, position=AT, ws=None, ws_bytes=0, stream=None)


@pytest.mark.parametrize("bad, status", [
    (dict(experts=None), BAD_ARG), (dict(offsets=None), BAD_ARG), (dict(position=None), BAD_ARG), (dict(index_bytes=2), BAD_ARG), (dict(count=-1), BAD_ARG),
    (dict(n_experts=0), BAD_ARG), (dict(n_experts=1025), TOO_LARGE), (dict(count=2 ** 31), TOO_LARGE), (dict(experts=AT + 2), ALIGN),
    (dict(experts=AT + 4, index_bytes=8), ALIGN),
])
def test_sort_refuses(bad, status):
    assert _call("void_sort_by_expert", SORT, SORT_BASE, **bad) == status


def test_sort_workspace():
    words = _lib.load().void_sort_by_expert_ws_bytes
    assert words(0, 8) == 0 and words(32768, 8) == 0 and words(-1, 8) == 0 and words(1000000, 0) == 0
    assert words(32769, 8) == 9 * 8 * 4
    assert words(2 ** 31 - 1, 1024) == 256 * 1024 * 4


DISPATCH = "x elem ldx tokens cols experts index_bytes top n_experts offsets position out ldo zero ws ws_bytes stream".split()
DISPATCH_BASE = dict(x=AT, elem=0, ldx=16, tokens=4, cols=16, experts=AT, index_bytes=4, top=2, n_experts=8, offsets=AT, position=AT, out=AT, ldo=16, zero=1,
                     ws=None, ws_bytes=0, stream=None)


@pytest.mark.parametrize("bad, status", [
    (dict(x=None), BAD_ARG), (dict(out=None), BAD_ARG), (dict(experts=None), BAD_ARG), (dict(elem=3), BAD_ARG), (dict(tokens=-1), BAD_ARG), (dict(top=0), BAD_ARG),
    (dict(cols=-1), BAD_ARG), (dict(ldx=15), SHAPE), (dict(ldo=15), SHAPE), (dict(tokens=2 ** 30, top=2), TOO_LARGE), (dict(n_experts=1025), TOO_LARGE),
    (dict(cols=68000000, ldx=68000000, ldo=68000000), TOO_LARGE),
])
def test_dispatch_refuses(bad, status):
    assert _call("void_dispatch", DISPATCH, DISPATCH_BASE, **bad) == status


COMBINE = "rows elem ldx tokens cols top position weights weight_elem residual ldr residual_elem out ldo stream".split()
COMBINE_BASE = dict(rows=AT, elem=1, ldx=16, tokens=4, cols=16, top=2, position=AT, weights=AT, weight_elem=0, residual=AT, ldr=16, residual_elem=1, out=AT,
                    ldo=16, stream=None)


@pytest.mark.parametrize("bad, status", [
    (dict(rows=None), BAD_ARG), (dict(out=None), BAD_ARG), (dict(position=None), BAD_ARG), (dict(elem=3), BAD_ARG), (dict(weight_elem=3), BAD_ARG),
    (dict(residual_elem=2), BAD_ARG), (dict(ldx=15), SHAPE), (dict(ldo=15), SHAPE), (dict(ldr=15), SHAPE), (dict(top=0), BAD_ARG),
    (dict(tokens=2 ** 30), TOO_LARGE), (dict(tokens=0), 0), (dict(cols=0), 0),
    (dict(cols=68000000, ldx=68000000, ldr=68000000, ldo=68000000), TOO_LARGE),
])
def test_combine_refuses(bad, status):
    assert _call("void_combine", COMBINE, COMBINE_BASE, **bad) == status


CGRAD = "g ldg rows ldx elem tokens cols top position used weights weight_elem drows ldd dweights stream".split()
CGRAD_BASE = dict(g=AT, ldg=16, rows=AT, ldx=16, elem=1, tokens=4, cols=16, top=2, position=AT, used=AT, weights=AT, weight_elem=0, drows=AT, ldd=16, dweights=AT,
                  stream=None)


@pytest.mark.parametrize("bad, status", [
    (dict(g=None), BAD_ARG), (dict(rows=None), BAD_ARG), (dict(position=None), BAD_ARG), (dict(used=None), BAD_ARG), (dict(elem=3), BAD_ARG),
    (dict(weight_elem=-1), BAD_ARG), (dict(ldg=15), SHAPE), (dict(ldd=15), SHAPE), (dict(ldx=15), SHAPE), (dict(drows=None, dweights=None), 0),
])
def test_combine_grad_refuses(bad, status):
    assert _call("void_combine_grad", CGRAD, CGRAD_BASE, **bad) == status


def test_there_is_no_cpu_path():
    x, ids = torch.zeros(4, 8), torch.zeros(4, 2, dtype=torch.int32)
    for call in (lambda: void.void_route(x, 2), lambda: void.sort_by_expert(ids, 4), lambda: void.void_dispatch(x, ids, 4),
                 lambda: void.void_combine(x, void.ExpertRoutes(torch.zeros(5, dtype=torch.int32), ids, 4))):
        with pytest.raises(_lib.VoidB200Error, match="no CPU path"):
            call()


def test_routes_that_were_written_to_are_refused():
    routes = void.ExpertRoutes(torch.zeros(5, dtype=torch.int32), torch.zeros(4, 2, dtype=torch.int32), 4)
    assert (routes.n_tokens, routes.top_k) == (4, 2) and "n_experts=4" in repr(routes)
    routes.check()
    routes.position[0, 0] = -1
    with pytest.raises(_lib.VoidB200Error, match="written to"):
        routes.check()
    with pytest.raises(TypeError, match="ExpertRoutes"):
        void.void_combine(torch.zeros(8, 8), routes.position)


def test_mirror_is_the_header():
    assert ctypes.sizeof(_lib.Fp8Args) == 184
