"""Tokens to experts and back on a B200, against plain implementations in 64 bits.

Tolerances: u = 2^-24 per fp32 operation along the longest chain that a value goes through, and half a step of the result's type."""
import pytest
import torch

import void_b200 as void
from void_b200 import _lib

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _half_step(v, dtype):
    """Half a step of ``dtype`` at v: relative, and of its smallest number."""
    info = torch.finfo(dtype)
    return v.abs() * (info.eps / 2) + info.smallest_normal * info.eps


def _close(got, want, bound):
    assert got.shape == want.shape
    bad = ~((got.double() - want).abs() <= bound)
    assert not bad.any(), (int(bad.sum()), (got.double() - want).abs().max().item(), bad.nonzero()[0].tolist())


# ------------------------------------------------------------------------------------------ router
def _route(scores, top, normalize):
    """Choices, weights and p over all experts, in 64 bits."""
    s = scores.double().cpu()
    ids = torch.full((s.shape[0], top), -1, dtype=torch.int32)
    w = torch.zeros(s.shape[0], top, dtype=torch.float64)
    p = torch.zeros_like(s)
    for t in range(s.shape[0]):
        order = sorted((e for e in range(s.shape[1]) if s[t, e] > -float("inf")), key=lambda e: (-s[t, e].item(), e))[:top]
        if not order:
            continue
        among = order if normalize else list(range(s.shape[1]))
        x = (s[t, among] - s[t, order[0]]).exp()
        p[t, among] = x / x.sum()
        ids[t, :len(order)] = torch.tensor(order, dtype=torch.int32)
        w[t, :len(order)] = p[t, order]
    return ids.cuda(), w.cuda(), p.cuda()


# A weight is exp (2 ulp, and u of the difference of two scores, at most 40 here) over a sum of E of them (a chain of E / 32 + 5), and a division.
def _weight_bound(w, experts):
    return w.abs() * U * (2 * (4 + 40) + experts / 32 + 5 + 4) + 1e-37


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("normalize", [True, False])
@pytest.mark.parametrize("n, experts, top", [(1, 1, 1), (3, 2, 2), (5, 31, 4), (4, 32, 32), (7, 33, 8), (130, 64, 6), (9, 200, 32), (6, 513, 3), (2, 1024, 8)])
def test_route(n, experts, top, normalize, dtype):
    scores = (torch.randn(n, experts, generator=_gen(n), device="cuda") * 3).to(dtype)
    scores[0, experts // 2] = scores[0, 0]                                       # a tie
    scores[n - 1, ::2] = -float("inf")                                           # masked experts
    if n > 2:
        scores[1] = -float("inf")                                                # nothing left
        scores[2, : experts // 2] = torch.finfo(dtype).min                       # the lowest number is no mask
    ids, w = void.void_route(scores, top, normalize)
    want_ids, want, p = _route(scores, top, normalize)
    assert ids.dtype is torch.int32 and w.dtype is torch.float32 and torch.equal(ids, want_ids)
    _close(w, want, _weight_bound(want, experts))
    # gradient
    scores.requires_grad_(True)
    g = torch.randn(n, top, generator=_gen(n + 1), device="cuda")
    ds, = torch.autograd.grad(void.void_route(scores, top, normalize)[1], scores, g)
    assert ds.dtype is dtype
    gd = g.double() * (want_ids >= 0)
    full = torch.zeros(n, experts, dtype=torch.float64, device="cuda")
    for j in range(top):
        full.scatter_add_(1, want_ids[:, j:j + 1].clamp_min(0).long(), gd[:, j:j + 1])
    mean = (gd * want).sum(1, keepdim=True)
    exact = p * (full - mean)
    size = p * (full.abs() + (gd.abs() * want).sum(1, keepdim=True))
    _close(ds, exact, size * U * (3 * (100 + experts / 32) + 12) + _half_step(exact, dtype) + 1e-37)


def test_route_gradient_against_differences():
    scores = torch.randn(3, 10, generator=_gen(0), device="cuda")
    g = torch.randn(3, 4, generator=_gen(1), device="cuda")
    for normalize in (True, False):
        s = scores.clone().requires_grad_(True)
        ds, = torch.autograd.grad(void.void_route(s, 4, normalize)[1], s, g)

        def value(x):
            return (_route(x, 4, normalize)[1] * g.double()).sum(1)
        for e in range(10):
            # central differences of a smooth function: h^2 of its third derivative (at most a few times |g|)
            step = torch.zeros(3, 10, dtype=torch.float64, device="cuda")
            step[:, e] = 1e-4
            want = (value(scores.double() + step) - value(scores.double() - step)) / 2e-4
            assert (ds[:, e].double() - want).abs().max() < 1e-6


def test_route_of_infinities_and_nan():
    nan, inf = float("nan"), float("inf")
    scores = torch.tensor([[1.0, nan, 2.0, nan], [inf, 0.0, 1.0, -inf], [0.0, -0.0, -1.0, -2.0]], device="cuda")
    ids, w = void.void_route(scores, 3)
    assert ids.tolist() == [[1, 3, 2], [0, 2, 1], [0, 1, 2]]
    assert w[0].isnan().all() and w[1].isnan().all() and w[2].isfinite().all()


def test_route_rows_that_lie_anyhow():
    wide = torch.randn(20, 100, generator=_gen(3), device="cuda")
    for scores in (wide[:, 3:40], wide[::3, 1:38], wide.t()[5:42].t(), wide[:1, :37].expand(8, 37)):
        want = void.void_route(scores.contiguous(), 5)
        got = void.void_route(scores, 5)
        assert torch.equal(want[0], got[0]) and torch.equal(want[1], got[1])
    s = wide[::2, 7:30].detach().clone()
    outer = torch.zeros(10, 60, device="cuda")
    outer[:, 5:28] = s
    leaf = outer.requires_grad_(True)
    ds, = torch.autograd.grad(void.void_route(leaf[:, 5:28], 2)[1].sum(), leaf)
    assert (ds[:, :5] == 0).all() and (ds[:, 28:] == 0).all()


def test_route_gradient_when_the_choices_were_changed():
    scores = torch.randn(6, 12, generator=_gen(4), device="cuda", requires_grad=True)
    g = torch.randn(6, 3, generator=_gen(5), device="cuda")
    want, = torch.autograd.grad(void.void_route(scores, 3)[1], scores, g)
    ids, w = void.void_route(scores, 3)
    ids.fill_(-1)                                                                # dropped by a capacity, say
    got, = torch.autograd.grad(w, scores, g)
    assert torch.equal(want, got)
    w = void.void_route(scores, 3)[1]
    with torch.no_grad():
        scores.add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(w, scores, g)


# ------------------------------------------------------------------------------------------ sort, dispatch, combine
def _sorted(ids, n_experts):
    flat = ids.reshape(-1).tolist()
    runs = [[i for i, e in enumerate(flat) if e == x] for x in range(n_experts)]
    position, offsets = torch.full((len(flat),), -1, dtype=torch.int32), [0]
    for r in runs:
        for k, i in enumerate(r):
            position[i] = offsets[-1] + k
        offsets.append(offsets[-1] + len(r))
    return torch.tensor(offsets, dtype=torch.int32).cuda(), position.view(ids.shape).cuda()


def _ids(n, top, experts, kind, seed, dtype=torch.int32):
    ids = torch.randint(0, experts, (n, top), generator=_gen(seed), device="cuda")
    if kind == "dropped":
        ids = torch.where(torch.rand(n, top, generator=_gen(seed + 1), device="cuda") < 0.4, torch.randint(-9, 0, (n, top), generator=_gen(seed + 2), device="cuda"), ids)
        ids[0] = experts + 5
    elif kind == "one":
        ids[:] = experts - 1
    elif kind == "none":
        ids[:] = -1
    return ids.to(dtype)


SORTS = [(0, 2, 4), (1, 1, 1), (1, 3, 1024), (33, 1, 7), (17, 4, 64), (512, 2, 9), (513, 2, 9), (1365, 3, 33), (4096, 1, 5), (4097, 1, 1000), (5000, 5, 256), (8192, 1, 3), (8193, 1, 12), (16384, 2, 64), (16385, 2, 65), (5000, 8, 256)]


@pytest.mark.parametrize("kind", ["any", "dropped", "one", "none"])
@pytest.mark.parametrize("n, top, experts", SORTS)
def test_sort(n, top, experts, kind):
    if n == 0 and kind == "dropped":
        pytest.skip("no token to drop")
    for dtype in (torch.int32, torch.int64):
        ids = _ids(n, top, experts, kind, n, dtype)
        routes = void.sort_by_expert(ids, experts)
        offsets, position = _sorted(ids, experts)
        assert torch.equal(routes.offsets, offsets) and torch.equal(routes.position, position)


def test_sort_of_many_tiles_and_far_ids():
    ids = torch.randint(0, 300, (150 * 4096 + 77, 1), generator=_gen(8), device="cuda")     # more tiles than SMs
    ids[::7] += 2 ** 33                                                                      # not an expert, though its low half is one
    routes = void.sort_by_expert(ids, 300)
    flat = ids.flatten()
    kept = flat < 300
    order = torch.where(kept, flat, 300).sort(stable=True).indices[: int(kept.sum())]
    position = torch.full((flat.numel(),), -1, dtype=torch.int32, device="cuda")
    position[order] = torch.arange(order.numel(), dtype=torch.int32, device="cuda")
    assert torch.equal(routes.position.flatten(), position)
    counts = torch.bincount(flat[kept], minlength=300).cumsum(0)
    assert torch.equal(routes.offsets[1:].long(), counts) and routes.offsets[0] == 0
    assert torch.equal(void.sort_by_expert(ids.t().contiguous().t(), 300).position, routes.position)


def _layout(t, how):
    """t as it is, with a pitch, starting on an odd element, or transposed in memory."""
    if how == "plain" or t.shape[0] == 0:
        return t
    if how == "pitch":
        return torch.empty(t.shape[0], t.shape[1] + 8, dtype=t.dtype, device=t.device)[:, :t.shape[1]].copy_(t)
    if how == "odd":
        return torch.empty(t.shape[0], t.shape[1] + 3, dtype=t.dtype, device=t.device)[:, 1:t.shape[1] + 1].copy_(t)
    return t.t().contiguous().t()


ROWS = [(1, 1, 1, 1), (5, 8, 2, 3), (7, 33, 3, 4), (16, 2048, 2, 8), (300, 130, 4, 17), (9, 4099, 5, 2), (40, 4104, 9, 300), (600, 64, 6, 31), (3, 9000, 1, 2), (2, 40, 40, 64)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("how", ["plain", "pitch", "odd", "transposed"])
@pytest.mark.parametrize("n, d, top, experts", ROWS)
def test_dispatch_and_combine(n, d, top, experts, how, dtype):
    ids = _ids(n, top, experts, "any" if n == 1 else "dropped", d)
    x = _layout(torch.randn(n, d, generator=_gen(1), device="cuda").to(dtype), how).requires_grad_(True)
    rows, routes = void.void_dispatch(x, ids, experts)
    offsets, position = _sorted(ids, experts)
    assert torch.equal(routes.offsets, offsets) and torch.equal(routes.position, position)
    kept = position.flatten() >= 0
    at, token = position.flatten()[kept].long(), torch.arange(n * top, device="cuda")[kept] // top
    want = torch.zeros(n * top, d, dtype=dtype, device="cuda")
    want[at] = x.detach()[token]
    assert torch.equal(rows, want)
    g = _layout(torch.randn(n * top, d, generator=_gen(2), device="cuda").to(dtype), how)
    dx, = torch.autograd.grad(rows, x, g)
    exact = torch.zeros(n, d, dtype=torch.float64, device="cuda").index_add_(0, token, g.double()[at])
    size = torch.zeros(n, d, dtype=torch.float64, device="cuda").index_add_(0, token, g.double().abs()[at])
    _close(dx, exact, size * U * (top + 1) + _half_step(exact, dtype))

    ys = torch.randn(n * top, d, generator=_gen(3), device="cuda").to(dtype)
    ys[offsets[-1]:] = float("nan")                                  # rows that are no token's
    ys = _layout(ys, how).requires_grad_(True)
    gy = _layout(torch.randn(n, d, generator=_gen(5), device="cuda").to(dtype), how)
    for weight_type, residual_type in ((None, None), (torch.float32, dtype), (dtype, torch.float32)):
        w = r = None
        weights = torch.ones(n, top, dtype=torch.float64, device="cuda")
        if weight_type is not None:
            w = torch.randn(n, top, generator=_gen(4), device="cuda").to(weight_type)
            weights = w.double()
            w[position < 0] = float("inf")                           # of dropped choices
            w.requires_grad_(True)
        exact = torch.zeros(n, d, dtype=torch.float64, device="cuda")
        if residual_type is not None:
            r = _layout(torch.randn(n, d, generator=_gen(6), device="cuda").to(residual_type), how).requires_grad_(True)
            exact += r.detach().double()
        part = weights.flatten()[kept][:, None] * ys.detach().double()[at]
        size = exact.abs().index_add(0, token, part.abs())
        exact = exact.index_add(0, token, part)
        y = void.void_combine(ys, routes, w, r)
        assert y.dtype is dtype
        _close(y.detach(), exact, size * U * (top + 2) + _half_step(exact, dtype))
        leaves = [t for t in (ys, w, r) if t is not None]
        grads = dict(zip([i for i, t in enumerate((ys, w, r)) if t is not None], torch.autograd.grad(y, leaves, gy)))
        dy = torch.zeros(n * top, d, dtype=torch.float64, device="cuda")
        dy[at] = weights.flatten()[kept][:, None] * gy.double()[token]
        _close(grads[0], dy, dy.abs() * U + _half_step(dy, dtype))
        if w is not None:
            dw = torch.zeros(n * top, dtype=torch.float64, device="cuda")
            size = torch.zeros_like(dw)
            product = ys.detach().double()[at] * gy.double()[token]
            dw[kept], size[kept] = product.sum(1), product.abs().sum(1)
            # a thread's chain of d / 256 (and the rest of a 16-byte piece), its warp's and its block's
            _close(grads[1], dw.view(n, top), (size * U * (d / 256 + 8 + 5 + 8 + 2)).view(n, top) + _half_step(dw.view(n, top), weight_type))
        if r is not None:
            assert torch.equal(grads[2], gy.to(residual_type))


def test_nothing_but_what_is_wanted():
    ids = _ids(10, 2, 4, "dropped", 1)
    routes = void.sort_by_expert(ids, 4)
    ys = torch.randn(20, 24, generator=_gen(1), device="cuda")
    w, r, g = torch.rand(10, 2, generator=_gen(2), device="cuda"), torch.randn(10, 24, device="cuda"), torch.randn(10, 24, generator=_gen(3), device="cuda")
    want = None
    for wanted in ((1, 1, 1), (1, 0, 0), (0, 1, 0), (0, 0, 1)):
        leaves = [t.clone().requires_grad_(bool(k)) for t, k in zip((ys, w, r), wanted)]
        y = void.void_combine(leaves[0], routes, leaves[1], leaves[2])
        grads = iter(torch.autograd.grad(y, [t for t in leaves if t.requires_grad], g))
        got = [next(grads) if k else None for k in wanted]
        want = want or got
        for a, b in zip(got, want):
            assert a is None or torch.equal(a, b)


def test_combine_against_differences():
    ids = torch.tensor([[0, 1], [1, -1], [2, 0]], device="cuda")
    routes = void.sort_by_expert(ids, 3)
    ys = torch.randn(6, 5, generator=_gen(1), device="cuda").requires_grad_(True)
    w = torch.rand(3, 2, generator=_gen(2), device="cuda").requires_grad_(True)
    g = torch.randn(3, 5, generator=_gen(3), device="cuda")
    dys, dw = torch.autograd.grad(void.void_combine(ys, routes, w), (ys, w), g)
    place = routes.position.tolist()

    def value(y, v):
        return sum(v[t, j] * (g[t].double() * y[place[t][j]]).sum() for t in range(3) for j in range(2) if place[t][j] >= 0)
    y64, w64 = ys.detach().double(), w.detach().double()
    for i in range(6):
        for c in range(5):   # (linear in either: differences are exact but for rounding)
            step = torch.zeros_like(y64)
            step[i, c] = 0.5
            assert abs(dys[i, c].item() - float(value(y64 + step, w64) - value(y64 - step, w64))) < 1e-6
    for t in range(3):
        for j in range(2):
            step = torch.zeros_like(w64)
            step[t, j] = 0.5
            assert abs(dw[t, j].item() - float(value(y64, w64 + step) - value(y64, w64 - step))) < 1e-6


def test_single_columns_and_gradients_that_are_repeated():
    ids = torch.tensor([[0, 2], [1, -1], [2, 2], [0, 1]], device="cuda")
    for d in (1, 5):
        x = torch.randn(4, d, generator=_gen(1), device="cuda").requires_grad_(True)
        w = torch.rand(4, 2, generator=_gen(2), device="cuda").requires_grad_(True)
        rows, routes = void.void_dispatch(x, ids, 3)
        dx, = torch.autograd.grad(rows.sum(), x, retain_graph=True)           # (the gradient of a sum has no strides)
        assert torch.equal(dx, (ids >= 0).sum(1, keepdim=True).float().expand(4, d))
        ys = rows.detach().requires_grad_(True)
        dys, dw = torch.autograd.grad(void.void_combine(ys, routes, w).sum(), (ys, w))
        place = routes.position.long()
        chosen = torch.where((place >= 0)[:, :, None], ys.detach()[place.clamp_min(0)].double(), 0.0)
        _close(dw, chosen.sum(2), chosen.abs().sum(2) * U * d)               # (a sum of d numbers, in whatever order: at most d roundings)
        assert torch.equal(dys[place[0, 1]], w.detach()[0, 1].expand(d))
    column = torch.randn(1, 1, device="cuda").expand(4, 1)
    assert torch.equal(void.void_dispatch(column, ids, 3)[0], void.void_dispatch(column.contiguous(), ids, 3)[0])
    scores = torch.randn(4, 1, device="cuda").requires_grad_(True)
    ds, = torch.autograd.grad(void.void_route(scores, 1)[1].sum(), scores)
    assert (ds == 0).all()
    assert torch.equal(void.void_combine(column[:1].expand(8, 1), void.sort_by_expert(ids, 3), residual=column), (1 + (ids >= 0).sum(1, keepdim=True)) * column)


def test_no_tokens_and_no_features():
    for n, d in ((0, 8), (3, 0), (0, 0)):
        x = torch.randn(n, d, device="cuda", requires_grad=True)
        w = torch.rand(n, 2, device="cuda", requires_grad=True)
        rows, routes = void.void_dispatch(x, torch.zeros(n, 2, dtype=torch.int64, device="cuda"), 4)
        assert rows.shape == (2 * n, d) and routes.offsets.tolist() == [0] + [2 * n] * 4
        y = void.void_combine(rows, routes, w, x)
        dx, dw = torch.autograd.grad(y.sum(), (x, w))
        assert dx.shape == (n, d) and (dw == 0).all()
    ids, w = void.void_route(torch.randn(0, 5, device="cuda", requires_grad=True), 2)
    assert ids.shape == w.shape == (0, 2)


def test_many_choices_of_few_tokens():
    for n, top, experts in ((1, 1024, 1000), (1, 1500, 7), (3, 700, 64)):
        ids = torch.randint(-1, experts, (n, top), generator=_gen(n), device="cuda")
        x = torch.randn(n, 40, generator=_gen(2), device="cuda")
        rows, routes = void.void_dispatch(x, ids, experts)
        offsets, position = _sorted(torch.where(ids < 0, -1, ids), experts)
        assert torch.equal(routes.offsets, offsets) and torch.equal(routes.position, position)
        y = void.void_combine(rows, routes)
        exact = x.double() * (ids >= 0).sum(1, keepdim=True)
        _close(y, exact, exact.abs() * U * (top + 1))


def test_given_results():
    ids = _ids(40, 3, 6, "dropped", 2)
    x = torch.randn(40, 48, generator=_gen(1), device="cuda")
    want, routes = void.void_dispatch(x, ids, 6)
    used = int(routes.offsets[-1])
    outer = torch.full((120, 60), 7.0, device="cuda")
    out = outer[:, 4:52]
    version = out._version
    got, _ = void.void_dispatch(x, ids, 6, out=out)
    assert got is out and out._version > version
    assert torch.equal(out[:used], want[:used]) and (out[used:] == 7).all() and (outer[:, :4] == 7).all() and (outer[:, 52:] == 7).all()
    # sharing memory with x: read from a copy
    both = torch.randn(120, 48, generator=_gen(2), device="cuda")
    inside = both[:40]
    want = void.void_dispatch(inside.clone(), ids, 6)[0]
    kept = both.clone()
    assert torch.equal(void.void_dispatch(inside, ids, 6, out=both)[0][:used], want[:used]) and torch.equal(both[used:], kept[used:])
    # combine: into the residual, and into the rows themselves
    ys, w, r = torch.randn(120, 48, generator=_gen(3), device="cuda"), torch.rand(40, 3, generator=_gen(4), device="cuda"), torch.randn(40, 48, generator=_gen(5), device="cuda")
    want = void.void_combine(ys, routes, w, r)
    stream = r.clone()
    assert void.void_combine(ys, routes, w, stream, out=stream) is stream and torch.equal(stream, want)
    rows = ys.clone()
    assert torch.equal(void.void_combine(rows, routes, w, r, out=rows[40:80]), want)
    shifted = torch.empty(41 * 48, device="cuda")
    shifted[:1920] = r.flatten()
    assert torch.equal(void.void_combine(ys, routes, w, shifted[:1920].view(40, 48), out=shifted[48:].view(40, 48)), want)


def test_refusals():
    x, ids = torch.randn(8, 16, device="cuda"), torch.zeros(8, 2, dtype=torch.int32, device="cuda")
    rows, routes = void.void_dispatch(x, ids, 4)
    bad = [
        (lambda: void.void_route(x.double(), 2), "float32, float16"), (lambda: void.void_route(x, 17), "top_k"), (lambda: void.void_route(x, 0), "top_k"),
        (lambda: void.void_route(x[0], 1), "matrix"), (lambda: void.void_route(torch.zeros(2, 1025, device="cuda"), 1), "1024"),
        (lambda: void.sort_by_expert(ids.float(), 4), "int32 or int64"), (lambda: void.sort_by_expert(ids[0], 4), "top_k"),
        (lambda: void.sort_by_expert(ids, 0), "1024"), (lambda: void.sort_by_expert(ids, 1025), "1024"),
        (lambda: void.void_dispatch(x[:7], ids, 4), "each of the 7 tokens"), (lambda: void.void_dispatch(x.double(), ids, 4), "float32"),
        (lambda: void.void_dispatch(x, ids, 4, out=rows.half()), "out must be"), (lambda: void.void_dispatch(x, ids, 4, out=rows[:8]), "out must be"),
        (lambda: void.void_dispatch(x, ids, 4, out=rows.clone().requires_grad_()), "differentiated"),
        (lambda: void.void_combine(rows[:15], routes), "each of the 8 x 2"), (lambda: void.void_combine(rows, routes, torch.ones(8, 3, device="cuda")), "weights"),
        (lambda: void.void_combine(rows, routes, residual=x[:7]), "residual"), (lambda: void.void_combine(rows.int(), routes), "float32"),
        (lambda: void.void_combine(rows, routes, out=x.half()), "out must be"), (lambda: void.void_combine(rows, routes, out=x.t()), "out must be"),
    ]
    for call, text in bad:
        with pytest.raises(_lib.VoidB200Error, match=text):
            call()
    leaf = x.clone().requires_grad_(True)
    for y in (void.void_dispatch(leaf, ids, 4)[0], void.void_route(leaf, 2)[1],
              void.void_combine(void.void_dispatch(leaf, ids, 4)[0], routes, torch.ones(8, 2, device="cuda"))):
        with pytest.raises(NotImplementedError, match="second derivative"):
            torch.autograd.grad(y.sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError, match="torch.func"):
        torch.func.grad(lambda t: void.void_route(t, 2)[1].sum())(x)
    import torch.autograd.forward_ad as fwd
    with fwd.dual_level(), pytest.raises(NotImplementedError, match="tangent"):
        void.void_dispatch(fwd.make_dual(x, x), ids, 4)
    routes.position[0, 0] = -1
    with pytest.raises(_lib.VoidB200Error, match="written to"):
        void.void_combine(rows, routes)


# ------------------------------------------------------------------------------------------ as they are used
def test_tokens_written_just_before():
    """Tokens are asked for while their choices are still being sorted: what writes them must be through by then."""
    given = [torch.randn(3000, 512, generator=_gen(s), device="cuda") for s in (1, 2)]
    ids = torch.randint(0, 32, (3000, 2), generator=_gen(3), device="cuda")
    want = [void.void_dispatch(x, ids, 32)[0] for x in given]
    x = given[0].clone()
    got = []
    for i in range(60):
        x.copy_(given[i % 2])
        got.append(void.void_dispatch(x, ids, 32)[0] if i % 3 else void.void_dispatch(x.mul_(1), ids.add_(0), 32)[0])
    for i, rows in enumerate(got):
        assert torch.equal(rows, want[i % 2]), i


def test_captured_and_replayed_with_other_tokens():
    x, scores = torch.randn(24, 64, generator=_gen(1), device="cuda"), torch.randn(24, 8, generator=_gen(2), device="cuda")

    def layer():
        ids, w = void.void_route(scores, 2)
        rows, routes = void.void_dispatch(x, ids, 8)
        return rows, void.void_combine(rows * 2, routes, w, residual=x)
    layer()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        layer()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        rows, y = layer()
    for seed in (3, 4):
        x.copy_(torch.randn(24, 64, generator=_gen(seed), device="cuda"))
        scores.copy_(torch.randn(24, 8, generator=_gen(seed + 10), device="cuda"))
        scores[5] = -float("inf")
        graph.replay()
        got = rows.clone(), y.clone()
        want = layer()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_streams_and_two_layers_at_once():
    x = torch.randn(700, 512, generator=_gen(1), device="cuda")
    ids = torch.randint(0, 16, (700, 4), generator=_gen(2), device="cuda")
    want = void.void_dispatch(x, ids, 16)
    back = void.void_combine(want[0], want[1])
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(4)]
    for _ in range(5):
        results = []
        for s in streams:
            with torch.cuda.stream(s):
                rows, routes = void.void_dispatch(x, ids, 16)
                results.append((rows, routes, void.void_combine(rows, routes)))
        torch.cuda.synchronize()
        for rows, routes, y in results:
            assert torch.equal(rows, want[0]) and torch.equal(routes.position, want[1].position) and torch.equal(y, back)


def test_a_layer_of_sparse_experts_in_training():
    """Router, dispatch, SparseExperts and combine with a residual: the output and every gradient against the formula in 64 bits."""
    import numpy as np
    import scipy.sparse as sp
    n, d, experts, top = 50, 96, 4, 2
    weights = [void.csr_to_void(sp.random(d, d, density=0.3, format="csr", dtype=np.float32, random_state=e)).to("cuda") for e in range(experts)]
    layer = void.SparseExperts(void.stack_experts(weights), bias=True, activation="silu")
    x = torch.randn(n, d, generator=_gen(1), device="cuda").requires_grad_(True)
    gate = (torch.randn(d, experts, generator=_gen(2), device="cuda") * 0.1).requires_grad_(True)
    ids, w = void.void_route(x @ gate, top)
    rows, routes = void.void_dispatch(x, ids, experts)
    y = void.void_combine(layer(rows, routes.offsets), routes, w, residual=x)
    g = torch.randn(n, d, generator=_gen(3), device="cuda")
    dx, dgate, dv = torch.autograd.grad(y, (x, gate, layer.values), g)
    x64, gate64 = x.detach().double().requires_grad_(True), gate.detach().double().requires_grad_(True)
    dense = []
    for e in range(experts):
        a = torch.zeros(d, d, dtype=torch.float64, device="cuda")
        t = weights[e]
        for v, r, c in zip(t.values.double(), t.block_rows.tolist(), t.block_cols.tolist()):
            a[r * 32:r * 32 + 32, c * 32:c * 32 + 32] = v
        dense.append(a.requires_grad_(True))
    s = x64 @ gate64
    p = torch.softmax(s.gather(1, ids.long()), 1)
    out = x64
    for j in range(top):
        for e in range(experts):
            z = x64 @ dense[e].t()
            out = out + torch.where(ids[:, j:j + 1] == e, p[:, j:j + 1] * z * torch.sigmoid(z), 0.0)
    want = torch.autograd.grad(out, (x64, gate64, *dense), g.double())
    # TF32 products (10 bits) of about 30 terms, forward and back: 2^-11 each way of values of size 1, a few of them one after the other
    def near(a, b):
        return ((a.double() - b).abs().max() / b.abs().max()).item() < 8 * 2.0 ** -11
    assert near(y, out) and near(dx, want[0]) and near(dgate, want[1])
    at = 0
    for e in range(experts):
        t = weights[e]
        for k, (r, c) in enumerate(zip(t.block_rows.tolist(), t.block_cols.tolist())):
            assert (dv[at + k].double() - want[2 + e][r * 32:r * 32 + 32, c * 32:c * 32 + 32]).abs().max() < 8 * 2.0 ** -11 * want[2 + e].abs().max()
        at += t.n_blocks


def test_a_captured_backward_pass():
    x = torch.randn(64, 128, generator=_gen(1), device="cuda")
    ids = torch.randint(0, 8, (64, 2), generator=_gen(2), device="cuda")
    leaf = x.clone().requires_grad_(True)
    w = torch.rand(64, 2, generator=_gen(3), device="cuda").requires_grad_(True)

    def step():
        rows, routes = void.void_dispatch(leaf, ids, 8)
        return torch.autograd.grad(void.void_combine(rows, routes, w).square().sum(), (leaf, w))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    with torch.no_grad():
        leaf.copy_(torch.randn(64, 128, generator=_gen(9), device="cuda"))
    ids.copy_(torch.randint(0, 8, (64, 2), generator=_gen(10), device="cuda"))
    graph.replay()
    for a, b in zip(got, step()):
        assert torch.equal(a, b)


def test_a_backward_pass_is_not_captured_beside_an_eager_graph_of_its_leaves():
    leaf = torch.randn(8, 16, device="cuda", requires_grad=True)
    ids = torch.zeros(8, 1, dtype=torch.int32, device="cuda")
    eager = void.void_dispatch(leaf, ids, 2)[0]
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="cannot be captured"):
        with torch.cuda.graph(graph):
            void.void_dispatch(leaf, ids, 2)[0].sum().backward()
    del eager
