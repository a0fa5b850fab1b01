"""Routing, what needs no GPU: refusals of the entry points and operators at their smallest and largest sizes."""
import copy
import pickle

import pytest
import torch

import void_b200 as void
from void_b200 import _lib

from test_routing_cpu import ALIGN, AT, CGRAD, CGRAD_BASE, COMBINE, COMBINE_BASE, DISPATCH, DISPATCH_BASE, GRAD, GRAD_BASE, ROUTE, ROUTE_BASE, SHAPE, SORT, SORT_BASE, _call


def test_dispatch_of_one_token_refuses_rows_that_overlap():
    for bad in (dict(ldo=15), dict(ldo=0), dict(ldo=-16), dict(ldo=15, top=3, index_bytes=8)):
        assert _call("void_dispatch", DISPATCH, DISPATCH_BASE, **dict(bad, tokens=1)) == SHAPE


def test_combine_of_one_token_refuses_rows_that_overlap():
    for bad in (dict(ldx=15), dict(ldx=0), dict(ldx=15, residual=None, top=4)):
        assert _call("void_combine", COMBINE, COMBINE_BASE, **dict(bad, tokens=1)) == SHAPE


def test_gradient_of_one_token_refuses_rows_that_overlap():
    for bad in (dict(ldd=15), dict(ldx=15), dict(ldd=0, dweights=None), dict(ldx=0, drows=None)):
        assert _call("void_combine_grad", CGRAD, CGRAD_BASE, **dict(bad, tokens=1)) == SHAPE


def test_one_row_has_no_pitch():
    """A single token with a single choice: no pitch is ever used, and none refused (without a GPU the calls end later, for that)."""
    for name, order, base, pitches in (("void_dispatch", DISPATCH, DISPATCH_BASE, dict(ldx=0, ldo=0)), ("void_combine", COMBINE, COMBINE_BASE, dict(ldx=0, ldr=0, ldo=0)),
                                       ("void_combine_grad", CGRAD, CGRAD_BASE, dict(ldg=0, ldx=0, ldd=0))):
        if torch.cuda.is_available():
            pytest.skip("the call would read addresses that are none")
        assert _call(name, order, base, **dict(pitches, tokens=1, top=1)) != SHAPE


def test_copies_of_routes_are_routes():
    routes = void.ExpertRoutes(torch.tensor([0, 2, 4]), torch.tensor([[0, 2], [1, 3]], dtype=torch.int32), 2)
    for copied in (copy.copy(routes), copy.deepcopy(routes), pickle.loads(pickle.dumps(routes))):
        copied.check()
        assert torch.equal(copied.offsets, routes.offsets) and torch.equal(copied.position, routes.position) and copied.n_experts == 2
    copied = copy.deepcopy(routes)
    copied.position[0, 0] = -1
    with pytest.raises(_lib.VoidB200Error, match="written to"):
        copied.check()
    routes.check()
    routes.position[0, 0] = -1
    for way in (copy.copy, copy.deepcopy, pickle.dumps):
        with pytest.raises(_lib.VoidB200Error, match="written to"):
            way(routes)


@pytest.mark.parametrize("name, order, base, words, halves", [
    ("void_route", ROUTE, dict(ROUTE_BASE, elem=2), ("experts", "weights"), ("scores",)), ("void_route_grad", GRAD, dict(GRAD_BASE, elem=1), ("g",), ("scores", "ds")),
    ("void_sort_by_expert", SORT, SORT_BASE, ("experts", "offsets", "position"), ()),
    ("void_dispatch", DISPATCH, dict(DISPATCH_BASE, elem=1), ("experts", "offsets", "position"), ("x", "out")),
    ("void_combine", COMBINE, COMBINE_BASE, ("position", "weights"), ("rows", "residual", "out")),
    ("void_combine_grad", CGRAD, CGRAD_BASE, ("position", "used", "weights", "dweights"), ("g", "rows", "drows"))])
def test_addresses_that_hold_no_element_are_refused(name, order, base, words, halves):
    for field in words:
        assert _call(name, order, base, **{field: AT + 2}) == ALIGN, field
    for field in halves:
        assert _call(name, order, base, **{field: AT + 1}) == ALIGN, field
        assert _call(name, order, dict(base, elem=0, residual_elem=0) if "residual" in base else dict(base, elem=0), **{field: AT + 2}) == ALIGN, field
