"""Layer norm, what needs no GPU: the entry points refuse bad arguments before they touch the device, CPU tensors are refused, and
the gradient formula that the GPU tests compare with is the derivative of the forward one."""
import ctypes

import pytest
import torch

import void_b200 as void
from void_b200 import _lib

BAD_ARG, TOO_LARGE = -1, -8


def norm64(x, w, b, eps):
    """The layer norm in the inputs' own (64-bit) precision: y, unit rows, 1 / sqrt(var + eps)."""
    mean = x.mean(-1, keepdim=True)
    c = x - mean
    rstd = 1.0 / torch.sqrt((c * c).mean(-1, keepdim=True) + eps)
    unit = c * rstd
    y = unit if w is None else unit * w
    return (y if b is None else y + b), unit, rstd


def norm_grad64(g, unit, rstd, w):
    gw = g if w is None else g * w
    dx = rstd * (gw - gw.mean(-1, keepdim=True) - unit * (gw * unit).mean(-1, keepdim=True))
    return dx, (g * unit).sum(0), g.sum(0)


def test_gradient_formula_is_the_derivative():
    gen = torch.Generator().manual_seed(5)
    for rows, cols in ((1, 1), (3, 7), (4, 64)):
        x, g = (torch.randn(rows, cols, generator=gen, dtype=torch.float64) for _ in range(2))
        w, b = (torch.randn(cols, generator=gen, dtype=torch.float64) for _ in range(2))
        _, unit, rstd = norm64(x, w, b, 1e-3)
        dx, dw, db = norm_grad64(g, unit, rstd, w)
        h = 1e-6
        for at, grad in ((x, dx), (w, dw), (b, db)):
            step = torch.randn(at.shape, generator=gen, dtype=torch.float64)
            args = [[t + s * h * step if t is at else t for t in (x, w, b)] for s in (1.0, -1.0)]
            diff = ((norm64(*args[0], 1e-3)[0] - norm64(*args[1], 1e-3)[0]) * g).sum() / (2 * h)
            # (error of a central difference: h^2 times a third derivative, about 1e-12 (1e3 for var near eps), and rounding 1e-16 / h)
            assert abs(float(diff - (grad * step).sum())) < 1e-6 * (1.0 + abs(float(diff)))


def test_cpu_tensors_are_refused():
    x = torch.randn(4, 8)
    with pytest.raises(_lib.VoidB200Error, match="no CPU path"):
        void.void_layer_norm(x)
    with pytest.raises(_lib.VoidB200Error, match="no CPU path"):
        void.VOIDLayerNorm(8, device="cpu")(x)


def _fwd(x=16, elem=0, ldx=8, rows=2, cols=8, w=16, b=16, pe=0, eps=1e-5, y=16, ldy=8, stats=None):
    ptr = lambda v: None if v is None else ctypes.c_void_p(v)   # noqa: E731
    return _lib.load().void_layer_norm(ptr(x), elem, ldx, rows, cols, ptr(w), ptr(b), pe, eps, ptr(y), ldy, ptr(stats), None)


@pytest.mark.parametrize("bad, status", [
    (dict(elem=3), BAD_ARG), (dict(elem=-1), BAD_ARG), (dict(elem=0, pe=1), BAD_ARG), (dict(elem=1, pe=2), BAD_ARG),
    (dict(rows=-1), BAD_ARG), (dict(cols=0), BAD_ARG), (dict(cols=-4), BAD_ARG), (dict(ldx=7), BAD_ARG), (dict(ldy=7), BAD_ARG),
    (dict(eps=-1.0), BAD_ARG), (dict(eps=float("nan")), BAD_ARG), (dict(x=None), BAD_ARG), (dict(y=None), BAD_ARG),
    (dict(rows=1 << 31), TOO_LARGE), (dict(cols=(1 << 30) + 8, ldx=1 << 31, ldy=1 << 31), TOO_LARGE),
])
def test_forward_entry_point_refuses(bad, status):
    assert _fwd(**bad) == status


def test_no_tokens_is_no_work():
    assert _fwd(rows=0, x=None, y=None) == 0


def _bwd(g=16, ldg=8, x=16, ldx=8, elem=0, rows=2, cols=8, w=16, pe=0, stats=16, dx=16, lddx=8, dw=16, db=16, ws=16, ws_bytes=1 << 20):
    ptr = lambda v: None if v is None else ctypes.c_void_p(v)   # noqa: E731
    return _lib.load().void_layer_norm_grad(ptr(g), ldg, ptr(x), ldx, elem, rows, cols, ptr(w), pe, ptr(stats), ptr(dx), lddx, ptr(dw),
                                            ptr(db), ptr(ws), ws_bytes, None)


@pytest.mark.parametrize("bad, status", [
    (dict(elem=3), BAD_ARG), (dict(elem=2, pe=1), BAD_ARG), (dict(rows=-1), BAD_ARG), (dict(cols=0), BAD_ARG), (dict(ldg=7), BAD_ARG),
    (dict(ldx=7), BAD_ARG), (dict(lddx=7), BAD_ARG), (dict(g=None), BAD_ARG), (dict(x=None), BAD_ARG), (dict(stats=None), BAD_ARG),
    (dict(rows=1 << 31), TOO_LARGE),
])
def test_backward_entry_point_refuses(bad, status):
    assert _bwd(**bad) == status


def test_backward_with_nothing_wanted_is_no_work():
    assert _bwd(dx=None, dw=None, db=None) == 0
    assert _bwd(rows=0, dw=None, db=None, g=None, x=None, stats=None) == 0


def test_workspace_grows_with_tokens_up_to_the_blocks_of_a_launch():
    ws = _lib.load().void_layer_norm_grad_ws_bytes
    assert ws(0, 8) == 0 and ws(8, 0) == 0 and ws(1, 8) == 64
    assert ws(3, 100) == 3 * 2 * 100 * 4
    assert ws(1 << 30, 100) == ws(1 << 20, 100)
