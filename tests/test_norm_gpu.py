"""Layer norm on the GPU against its formula in 64 bits."""
import pytest
import torch

import void_b200 as void
from test_norm_cpu import norm64, norm_grad64
from void_b200 import _lib

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 1e-44, torch.float16: 2.0 ** -25, torch.bfloat16: 1e-40}   # half the smallest number
# A sum over the features adds at most 16 pieces of 8 per thread in sequence (rows in registers; 70000 features: 9 pieces of 8), then
# ten steps of a tree: fewer than CHAIN roundings, each of at most U times the sum of the absolute values.
CHAIN = 160
TYPES = [(torch.float32, torch.float32), (torch.float16, torch.float16), (torch.float16, torch.float32),
         (torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32)]
SHAPES = [(1, 1), (3, 7), (1, 32), (5, 33), (8, 2048), (700, 64), (300, 1000), (301, 1016), (257, 4096), (2, 16384), (301, 5003), (3, 16383),
          (5, 20001), (3, 70000), (1000, 128), (2500, 24)]


def make(rows, cols, dtype, params, seed=0, shift=0.5):
    gen = torch.Generator(device="cuda").manual_seed(seed + 1000 * rows + cols)

    def r(*shape, scale=1.0, add=0.0, t=dtype):
        return (torch.randn(*shape, generator=gen, device="cuda") * scale + add).to(t)
    return (r(rows, cols, add=shift), r(cols, scale=0.3, add=1.0, t=params), r(cols, scale=0.3, t=params), r(rows, cols))


def unit_error(x, rstd, unit):
    """Bound on the error of a unit row: the mean is off by CHAIN roundings of mean |x|, rstd by half of the variance's CHAIN and the
    mean's square (which is smaller), the product by three more."""
    dmean = (CHAIN + 2) * U * x.abs().mean(-1, keepdim=True)
    return dmean * rstd * (1.0 + unit.abs()) + unit.abs() * (CHAIN + 6) * U


def forward_bound(x, w, b, unit, rstd, y, dtype):
    e = unit_error(x, rstd, unit)
    wa = 1.0 if w is None else w.abs()
    ba = 0.0 if b is None else b.abs()
    raw = e * wa + 3 * U * (unit.abs() * wa + ba)
    return raw + HALF[dtype] * (y.abs() + raw) + TINY[dtype]


def backward_bounds(x, w, g, unit, rstd, dx, dw, db, dtype, params):
    e = unit_error(x, rstd, unit)
    gw = g if w is None else g * w
    rel = (CHAIN + 6) * U
    m1, m2 = gw.abs().mean(-1, keepdim=True), (gw * unit).abs().mean(-1, keepdim=True)
    raw = rstd * (gw.abs() + m1 + unit.abs() * m2) * (3 * rel) + rstd * (e * m2 + unit.abs() * (gw.abs() * e).mean(-1, keepdim=True))
    rows = x.shape[0]
    raw_w = (g.abs() * e).sum(0) + (rows + 16) * U * (g * unit).abs().sum(0)
    raw_b = (rows + 16) * U * g.abs().sum(0)
    return [r + h * (v.abs() + r) + t for r, v, h, t in ((raw, dx, HALF[dtype], TINY[dtype]), (raw_w, dw, HALF[params], TINY[params]),
                                                         (raw_b, db, HALF[params], TINY[params]))]


def within(got, ref, bound):
    off = (got.double() - ref).abs() - bound
    assert bool((off <= 0).all()), (float(off.max()), float(bound.max()))


def check(x, w, b, g, y, grads=None, eps=1e-5):
    xd, wd, bd = (None if t is None else t.detach().double() for t in (x, w, b))
    ref, unit, rstd = norm64(xd, wd, bd, eps)
    within(y, ref, forward_bound(xd, wd, bd, unit, rstd, ref, x.dtype))
    if grads is not None:
        gd = g.double()
        refs = norm_grad64(gd, unit, rstd, wd)
        bounds = backward_bounds(xd, wd, gd, unit, rstd, *refs, x.dtype, x.dtype if w is None else w.dtype)
        for got, r, bound in zip(grads, refs, bounds):
            if got is not None:
                within(got, r, bound)


@pytest.mark.parametrize("dtype, params", TYPES)
@pytest.mark.parametrize("rows, cols", SHAPES)
def test_forward_and_gradients(rows, cols, dtype, params):
    x, w, b, g = make(rows, cols, dtype, params)
    y = void.void_layer_norm(x, w, b)
    assert y.dtype == dtype and y.shape == x.shape
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    y2 = void.void_layer_norm(x, w, b)
    assert torch.equal(y2, y)
    grads = torch.autograd.grad(y2, leaves, g)
    assert [t.dtype for t in grads] == [dtype, params, params]
    check(x, w, b, g, y, grads)


@pytest.mark.parametrize("dtype, params", TYPES)
@pytest.mark.parametrize("rows, cols", [(2700, 1032), (2700, 1031), (1800, 5000), (1801, 5001), (900, 9000), (900, 9002), (900, 9001)])
def test_many_rows(rows, cols, dtype, params):
    # (rows enough for blocks that walk them, on and off 16-byte pieces)
    x, w, b, g = make(rows, cols, dtype, params)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    y = void.void_layer_norm(x, w, b)
    check(x, w, b, g, y, torch.autograd.grad(y, leaves, g))
    wide = torch.full((rows, cols + 3), float("nan"), device="cuda", dtype=dtype)    # what lies between the rows is not read as theirs
    wide[:, :cols] = x.detach()
    check(x, w, b, g, void.void_layer_norm(wide[:, :cols], w, b))


@pytest.mark.parametrize("which", ["neither", "weight", "bias"])
@pytest.mark.parametrize("cols", [100, 104, 20000])
def test_parameters_may_be_left_out(which, cols):
    x, w, b, g = make(9, cols, torch.bfloat16, torch.float32)
    w, b = (w if which == "weight" else None), (b if which == "bias" else None)
    leaves = [t.requires_grad_(True) for t in (x, w, b) if t is not None]
    y = void.void_layer_norm(x, w, b)
    grads = dict(zip([n for n, t in zip("xwb", (x, w, b)) if t is not None], torch.autograd.grad(y, leaves, g)))
    xd, wd, bd = (None if t is None else t.detach().double() for t in (x, w, b))
    ref, unit, rstd = norm64(xd, wd, bd, 1e-5)
    within(y, ref, forward_bound(xd, wd, bd, unit, rstd, ref, x.dtype))
    refs = norm_grad64(g.double(), unit, rstd, wd)
    bounds = backward_bounds(xd, wd, g.double(), unit, rstd, *refs, x.dtype, torch.float32)
    for name, r, bound in zip("xwb", refs, bounds):
        if name in grads:
            within(grads[name], r, bound)


@pytest.mark.parametrize("want", [(0,), (1,), (2,), (1, 2), (0, 2)])
@pytest.mark.parametrize("cols", [96, 9001])
def test_only_the_gradients_that_are_wanted(want, cols):
    x, w, b, g = make(13, cols, torch.float16, torch.float16)
    args = [x, w, b]
    for i in want:
        args[i].requires_grad_(True)
    y = void.void_layer_norm(*args)
    got = torch.autograd.grad(y, [args[i] for i in want], g)
    full = [None] * 3
    for i, t in zip(want, got):
        full[i] = t
    check(x, w, b, g, y, full)


def test_directional_differences():
    x, w, b, g = make(6, 200, torch.float32, torch.float32)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    grads = torch.autograd.grad(void.void_layer_norm(x, w, b), leaves, g)
    gen = torch.Generator(device="cuda").manual_seed(3)
    h = 1e-5
    base = [t.detach().double() for t in (x, w, b)]
    for i in range(3):
        step = torch.randn(base[i].shape, generator=gen, device="cuda", dtype=torch.float64)
        ends = [[t + (s * h * step if j == i else 0.0) for j, t in enumerate(base)] for s in (1.0, -1.0)]
        diff = float(((norm64(*ends[0], 1e-5)[0] - norm64(*ends[1], 1e-5)[0]) * g.double()).sum() / (2 * h))
        size = float((grads[i].double() * step).abs().sum())
        # fp32 gradients: CHAIN roundings of their summands at most; the difference's own error is of order h^2 = 1e-10
        assert abs(float((grads[i].double() * step).sum()) - diff) < 10 * CHAIN * U * size + 1e-6


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_layouts(dtype):
    x, w, b, g = make(24, 160, dtype, dtype)
    wide = torch.zeros(24, 200, device="cuda", dtype=dtype)
    for off in (0, 1, 8):    # rows with a pitch, aligned and not
        v = wide[:, off:off + 160]
        v.copy_(x)
        check(x, w, b, g, void.void_layer_norm(v, w, b))
    t = x.t().contiguous().t()                                    # features far apart
    check(x, w, b, g, void.void_layer_norm(t, w, b))
    check(x[::2], w, b, g, void.void_layer_norm(x[::2], w, b))
    one = x[:1].expand(24, 160)                                   # one row, repeated
    check(one, w, b, g, void.void_layer_norm(one, w, b))
    y3 = void.void_layer_norm(x.view(2, 3, 4, 160), w, b)
    assert y3.shape == (2, 3, 4, 160)
    check(x, w, b, g, y3.view(24, 160))
    check(x[:1], w, b, g, void.void_layer_norm(x[0], w, b).view(1, 160))
    wn = torch.empty(160, 2, device="cuda", dtype=dtype)[:, 0].copy_(w)   # a parameter with a stride, and one off 16 bytes
    bn = torch.empty(161, device="cuda", dtype=dtype)[1:].copy_(b)
    check(x, w, b, g, void.void_layer_norm(x, wn, bn))
    v = wide[:, 1:161].detach().requires_grad_(True)
    gs = torch.empty(160, 24, device="cuda", dtype=dtype).t().copy_(g)
    wp, bp = wn.detach().requires_grad_(True), bn.detach().requires_grad_(True)
    y = void.void_layer_norm(v, wp, bp)
    check(wide[:, 1:161], w, b, g, y, torch.autograd.grad(y, (v, wp, bp), gs))
    ones = torch.ones(24, 160, device="cuda", dtype=dtype)
    leaf = x.clone().requires_grad_(True)
    y = void.void_layer_norm(leaf, w, b)
    check(x, w, b, ones, y, list(torch.autograd.grad(y.sum(), leaf)) + [None, None])   # the gradient of a sum is one value, repeated


def test_one_leaf_twice_and_shared_parameters():
    x, w, b, g = make(10, 64, torch.float32, torch.float32)
    w.requires_grad_(True)
    y = void.void_layer_norm(x, w, w)        # the same tensor as weight and bias
    (dw,) = torch.autograd.grad(y, w, g)
    _, unit, rstd = norm64(x.double(), None, None, 1e-5)
    ref = (g.double() * unit).sum(0) + g.double().sum(0)
    e = (10 + 20) * U * ((g.double() * unit).abs().sum(0) + g.double().abs().sum(0)) + (g.double().abs() * unit_error(x.double(), rstd, unit)).sum(0)
    within(dw, ref, e)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_rows_that_are_not_finite_stay_alone(dtype):
    x, w, b, g = make(40, 96, dtype, dtype)
    clean = void.void_layer_norm(x, w, b)
    bad = x.clone()
    bad[3, 5], bad[17, 0], bad[39, 95] = float("nan"), float("inf"), float("-inf")
    y = void.void_layer_norm(bad.requires_grad_(True), w, b)
    rows = [r for r in range(40) if r not in (3, 17, 39)]
    assert torch.equal(y[rows], clean[rows]) and bool(y[[3, 17, 39]].isnan().all())
    (dx,) = torch.autograd.grad(y, bad, g)
    leaf = x.clone().requires_grad_(True)
    (ref,) = torch.autograd.grad(void.void_layer_norm(leaf, w, b), leaf, g)
    assert torch.equal(dx[rows], ref[rows])


def test_rows_of_one_value_and_large_means():
    x = torch.full((4, 256), 3.0, device="cuda")
    assert torch.equal(void.void_layer_norm(x), torch.zeros_like(x))
    x, w, b, g = make(8, 1024, torch.float32, torch.float32, shift=1e4)     # |mean| is ten thousand times the deviation
    check(x, w, b, g, void.void_layer_norm(x, w, b))
    x, w, b, g = make(8, 1024, torch.float32, torch.float32)
    check(x, w, b, g, void.void_layer_norm(x, w, b, 0.0), eps=0.0)
    check(x, w, b, g, void.void_layer_norm(x, w, b, 2.5), eps=2.5)


def test_no_tokens():
    w, b = torch.ones(16, device="cuda", requires_grad=True), torch.zeros(16, device="cuda", requires_grad=True)
    x = torch.empty(0, 16, device="cuda", requires_grad=True)
    y = void.void_layer_norm(x, w, b)
    dx, dw, db = torch.autograd.grad(y.sum(), (x, w, b))
    assert y.shape == (0, 16) and dx.shape == (0, 16) and not dw.any() and not db.any()


def test_out_and_in_place():
    x, w, b, g = make(33, 128, torch.bfloat16, torch.bfloat16)
    ref = void.void_layer_norm(x, w, b)
    out = torch.empty_like(x)
    assert void.void_layer_norm(x, w, b, out=out) is out and torch.equal(out, ref)
    own = x.clone()
    void.void_layer_norm(own, w, b, out=own)
    assert torch.equal(own, ref)


def test_results_repeat_bit_for_bit():
    x, w, b, g = make(3000, 520, torch.bfloat16, torch.float32)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    first = torch.autograd.grad(void.void_layer_norm(x, w, b), leaves, g)
    for _ in range(3):
        again = torch.autograd.grad(void.void_layer_norm(x, w, b), leaves, g)
        assert all(torch.equal(p, q) for p, q in zip(first, again))


def test_on_another_stream_and_in_a_graph():
    x, w, b, g = make(64, 768, torch.bfloat16, torch.bfloat16)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = void.void_layer_norm(x, w, b)
        grads = torch.autograd.grad(y, leaves, g)
    side.synchronize()
    check(x, w, b, g, y, grads)
    del y, grads                      # (no eager graph of these leaves lives while one is captured)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = void.void_layer_norm(x, w, b)
        grads = torch.autograd.grad(y, leaves, g)
    x2, _, _, g2 = make(64, 768, torch.bfloat16, torch.bfloat16, seed=9)
    with torch.no_grad():
        x.copy_(x2)
        g.copy_(g2)
    graph.replay()
    torch.cuda.synchronize()
    check(x, w, b, g, y, grads)


def test_module_and_training_step():
    layer = void.VOIDLayerNorm(48, dtype=torch.bfloat16)
    x = torch.randn(7, 48, device="cuda").bfloat16().requires_grad_(True)
    y = layer(x)
    y.backward(torch.ones_like(y))
    check(x, layer.weight, layer.bias, torch.ones_like(y), y, (x.grad, layer.weight.grad, layer.bias.grad))
    assert void.VOIDLayerNorm(48, bias=False).bias is None
    state = layer.state_dict()
    assert set(state) == {"weight", "bias"}


def test_refusals():
    x, w, b, g = make(4, 32, torch.bfloat16, torch.bfloat16)
    for call, text in ((lambda: void.void_layer_norm(x.int()), "float32, float16 or bfloat16"),
                       (lambda: void.void_layer_norm(x, w[:31], b), "vectors of 32"),
                       (lambda: void.void_layer_norm(x, w.half()), "float32 or of x's type"),
                       (lambda: void.void_layer_norm(x, w, b.float()), "of one type"),
                       (lambda: void.void_layer_norm(x, w.view(1, 32)), "vectors of 32"),
                       (lambda: void.void_layer_norm(x, w, b, -1.0), "eps"),
                       (lambda: void.void_layer_norm(x[:, :0]), "at least one feature"),
                       (lambda: void.void_layer_norm(x, w, b, out=torch.empty_like(x).t()), "out must be"),
                       (lambda: void.void_layer_norm(x, w, b, out=x.float()), "out must be"),
                       (lambda: void.void_layer_norm(x, w.requires_grad_(True), b, out=torch.empty_like(x)), "out= cannot")):
        with pytest.raises(_lib.VoidB200Error, match=text):
            call()
    x.requires_grad_(True)
    y = void.void_layer_norm(x, w, b)
    with pytest.raises(NotImplementedError, match="second derivative"):
        torch.autograd.grad(y.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="torch.func"):
        torch.func.vmap(lambda t: void.void_layer_norm(t))(x.detach())
    (dx,) = torch.autograd.grad(y, x, g)
    with pytest.raises(RuntimeError, match="second time|freed"):
        torch.autograd.grad(y, x, g)
