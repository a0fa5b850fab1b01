"""Linear layers with bias, activation and residual on the GPU, forward and backward, against their formulas in 64 bits."""
import pytest
import torch

import void_b200 as void
from test_linear_cpu import ACTS, HALF, U, act64, layer64, layer_grads64, rounded, within
from test_norm_cpu import norm64
from test_norm_gpu import forward_bound
from void_b200 import _lib

pytestmark = pytest.mark.gpu
TYPES = [torch.float16, torch.bfloat16, torch.float32]


def weight(m, k, density, dtype, seed=0):
    """A VOID weight with about ``density`` of its tiles at random places (some tile rows may be empty), zero outside the matrix."""
    gen = torch.Generator().manual_seed(seed + 7 * m + k)
    nbr, nbc = (m + 31) // 32, (k + 31) // 32
    mask = torch.rand(nbr, nbc, generator=gen) < density
    values = torch.randn(int(mask.sum()), 32, 32, generator=gen) * (max(density, 0.05) * k) ** -0.5
    a = void.void_from_block_mask(mask.numpy(), values.cuda(), shape=(m, k))
    if m % 32:
        a.values[a.block_rows == m // 32, m % 32:, :] = 0
    if k % 32:
        a.values[a.block_cols == k // 32, :, k % 32:] = 0
    return a.to_dtype(dtype)


def rand(*shape, dtype=torch.float32, seed=0, scale=1.0):
    gen = torch.Generator(device="cuda").manual_seed(seed + 31 * shape[0] + shape[-1])
    return (torch.randn(*shape, generator=gen, device="cuda") * scale).to(dtype)


def check_layer(y, a, x, bias, r, act):
    xd, ad, bd, rd = (None if t is None else t.double() for t in (x, a.to_dense(), bias, r))
    _, ref, _, e = layer64(xd, ad, bd, rd, act, x.dtype)
    within(y, ref, rounded(e, ref, y.dtype))


SHAPES = [(1, 64, 32), (3, 70, 45), (8, 256, 512), (16, 1000, 96), (17, 333, 100), (33, 96, 200), (130, 515, 333), (257, 1024, 640), (300, 128, 64),
          (513, 2048, 1000)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("n, k, m", SHAPES)
def test_inference(n, k, m, act, dtype):
    a, x = weight(m, k, 0.3, dtype), rand(n, k, dtype=dtype)
    bias, r = rand(m, seed=1), rand(n, m, dtype=dtype, seed=2)
    check_layer(void.void_linear(a, x, bias, void.get_activation_code(act), residual=r), a, x, bias, r, act)
    check_layer(void.void_linear(a, x, None, void.get_activation_code(act), residual=r.float()), a, x, None, r, act)


@pytest.mark.parametrize("dtype", TYPES)
def test_residual_layouts(dtype):
    a, x, r = weight(100, 200, 0.4, dtype), rand(40, 200, dtype=dtype), rand(40, 100, dtype=dtype, seed=3)
    base = void.void_linear(a, x, residual=r)
    check_layer(base, a, x, None, r, "none")
    wide = torch.zeros(40, 150, device="cuda", dtype=dtype)
    for off in (0, 1, 8):
        wide[:, off:off + 100] = r
        assert torch.equal(void.void_linear(a, x, residual=wide[:, off:off + 100]), base)
    assert torch.equal(void.void_linear(a, x, residual=r.t().contiguous().t()), base)
    one = r[:1].expand(40, 100)
    assert torch.equal(void.void_linear(a, x, residual=one), void.void_linear(a, x, residual=one.contiguous()))
    # a residual of another 16-bit type is added without a rounding of its own
    other = torch.float16 if dtype == torch.bfloat16 else torch.bfloat16
    check_layer(void.void_linear(a, x, residual=r.to(other)), a, x, None, r.to(other), "none")
    # in place: the residual stream takes the result
    stream = r.clone()
    assert void.void_linear(a, x, residual=stream, out=stream) is stream and torch.equal(stream, base)
    # memory that the result shares in another way is read before it is written
    buf = torch.zeros(41, 100, device="cuda", dtype=dtype)
    buf[1:] = r
    void.void_linear(a, x, residual=buf[1:], out=buf[:40])
    assert torch.equal(buf[:40], base)


@pytest.mark.parametrize("n", [1, 5, 128, 300])
def test_a_weight_without_tiles(n):
    a, x, r, bias = weight(64, 96, 0.0, torch.bfloat16), rand(n, 96, dtype=torch.bfloat16), rand(n, 64, dtype=torch.bfloat16), rand(64)
    assert a.n_blocks == 0
    check_layer(void.void_linear(a, x, bias, 3, residual=r), a, x, bias, r, "silu")


@pytest.mark.parametrize("n", [3, 100, 700])
@pytest.mark.parametrize("bias_type", [torch.float16, torch.bfloat16])
def test_biases_in_their_own_type(n, bias_type):
    a, x, r = weight(333, 515, 0.3, torch.bfloat16), rand(n, 515, dtype=torch.bfloat16), rand(n, 333, dtype=torch.bfloat16, seed=2)
    back = weight(515, 333, 0.3, torch.bfloat16, seed=5)
    bias, bias2 = rand(333, seed=1, dtype=bias_type), rand(515, seed=1, dtype=bias_type)
    check_layer(void.void_linear(a, x, bias, 2), a, x, bias, None, "gelu")
    check_layer(void.void_linear(a, x, bias, 2, residual=r), a, x, bias, r, "gelu")
    check_layer(void.void_linear(a, x, torch.stack([bias, bias], 1)[:, 0], 2), a, x, bias, None, "gelu")
    odd = torch.empty(334, device="cuda", dtype=bias_type)[1:].copy_(bias)
    check_layer(void.void_linear(a, x, odd, 2), a, x, bias, None, "gelu")
    ref, e = feed_forward64(x, None, a, bias.double(), back, bias2.double(), "gelu", torch.bfloat16)
    within(void.fused_sparse_mlp(x, a, back, "gelu", bias, bias2, residual=x), ref, e)


def test_no_tokens():
    a = weight(64, 96, 0.5, torch.float16)
    x, r = torch.empty(0, 96, device="cuda", dtype=torch.float16), torch.empty(0, 64, device="cuda", dtype=torch.float16)
    assert void.void_linear(a, x, residual=r).shape == (0, 64)
    layer = void.SparseLinear(96, 64, a, activation="gelu")
    y = layer(x.requires_grad_(True), residual=r)
    grads = torch.autograd.grad(y, (x, layer.sparse_weight.values, layer.bias), torch.empty_like(y))
    assert grads[0].shape == (0, 96) and not grads[1].any() and not grads[2].any()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("n, density, residual_type", [(1024, 0.45, None), (2048, 0.1, torch.float32), (1111, 0.3, None)])
def test_large_products_by_every_kernel(n, density, residual_type, dtype):
    # (the first calls take the row kernel, on a transposed copy of x; from the fourth on a store for groups of tile rows is there)
    a, x = weight(4096, 4096, density, dtype), rand(n, 4096, dtype=dtype)
    bias, r = rand(4096, seed=1), rand(n, 4096, dtype=residual_type or dtype, seed=2)
    xd, ad = x.double(), a.to_dense().double()
    _, ref, _, e = layer64(xd, ad, bias.double(), r.double(), "gelu", dtype)
    e = rounded(e, ref, dtype)
    for _ in range(6):
        within(void.void_linear(a, x, bias, 2, residual=r), ref, e)
        torch.cuda.synchronize()


def test_residual_of_infinities_and_nan_stays_in_place():
    a, x, r = weight(100, 200, 0.4, torch.bfloat16), rand(40, 200, dtype=torch.bfloat16), rand(40, 100, dtype=torch.bfloat16)
    base = void.void_linear(a, x, residual=r)
    bad = r.clone()
    bad[3, 7], bad[39, 99] = float("nan"), float("-inf")
    y = void.void_linear(a, x, residual=bad)
    assert bool(y[3, 7].isnan()) and float(y[39, 99]) == float("-inf")
    y[3, 7], y[39, 99] = base[3, 7], base[39, 99]
    assert torch.equal(y, base)


@pytest.mark.parametrize("out_dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n, k, m", [(4, 320, 96), (70, 515, 333), (300, 1024, 256)])
def test_int8(n, k, m, out_dtype):
    q = void.quantize_void_tensor(weight(m, k, 0.4, torch.float32))
    gen = torch.Generator(device="cuda").manual_seed(n)
    x = torch.randint(-128, 128, (n, k), generator=gen, device="cuda", dtype=torch.int8)
    scale, bias, r = rand(n).abs() + 0.1, rand(m, seed=1), rand(n, m, dtype=out_dtype, seed=2)
    y = void.void_linear(q, x, bias, 1, x_scale=scale, out_dtype=out_dtype, residual=r)
    nbr = (m + 31) // 32
    row = q.block_rows.long().cpu()
    mean = torch.zeros(nbr, dtype=torch.float64).scatter_reduce(0, row, q.scales.double().cpu(), "mean", include_self=False).cuda()
    dense = torch.zeros(nbr, (k + 31) // 32, 32, 32, device="cuda", dtype=torch.float64)
    dense[q.block_rows.long(), q.block_cols.long()] = q.values.double()
    dense = dense.permute(0, 2, 1, 3).reshape(nbr * 32, -1)[:m, :k]
    part = (x.double() @ dense.t()) * mean.repeat_interleave(32)[:m] * scale.double()[:, None]
    ref = (part + bias.double()).clamp_min(0) + r.double()
    # exact sums, one rounding to fp32; the mean scale (a sum of up to K / 32 terms), two products and two sums in fp32
    e = (k / 32 + 8) * U * part.abs() + 4 * U * (bias.double().abs() + ref.abs() + r.double().abs())
    within(y, ref, rounded(e, ref, out_dtype))


# ------------------------------------------------------------------------------------------ training
def train(layer, x, r, g):
    leaves = [x.requires_grad_(True), layer.sparse_weight.values, layer.bias] + ([r.requires_grad_(True)] if r is not None else [])
    y = layer(x, residual=r) if r is not None else layer(x)
    return y, torch.autograd.grad(y, leaves, g)


def tiles_of(dense, a):
    m, k = a.shape
    padded = torch.zeros((m + 31) // 32 * 32, (k + 31) // 32 * 32, dtype=dense.dtype, device=dense.device)
    padded[:m, :k] = dense
    return padded.view(padded.shape[0] // 32, 32, padded.shape[1] // 32, 32)[a.block_rows.long(), :, a.block_cols.long()]


def check_training(layer, a, x, r, g, y, grads, act):
    dtype = x.dtype
    xd, ad, bd, gd = x.detach().double(), a.to_dense().double(), layer.bias.detach().double(), g.double()
    rd = None if r is None else r.detach().double()
    z, ref, ez, e = layer64(xd, ad, bd, rd, act, dtype)
    within(y, ref, rounded(e, ref, dtype))
    (dx, edx), (da, eda), (db, edb) = layer_grads64(gd, z, ez, xd, ad, act, dtype, layer.bias.dtype)
    within(grads[0], dx, edx)
    within(grads[1], tiles_of(da, a), tiles_of(eda, a))
    within(grads[2], db, edb)
    if r is not None:
        assert torch.equal(grads[3], g.to(r.dtype))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("n, k, m", [(1, 64, 32), (3, 70, 45), (33, 96, 200), (130, 515, 333), (257, 1024, 640)])
def test_training(n, k, m, act, dtype):
    a, x = weight(m, k, 0.3, dtype), rand(n, k, dtype=dtype)
    r, g = rand(n, m, dtype=dtype, seed=2), rand(n, m, dtype=dtype, seed=3)
    layer = void.SparseLinear(k, m, a, activation=act)
    with torch.no_grad():
        layer.bias.copy_(rand(m, seed=1))
    y, grads = train(layer, x, r, g)
    check_training(layer, a, x, r, g, y, grads, act)


def test_training_with_fp32_bias_and_residual_and_without_a_bias():
    a, x, g = weight(200, 300, 0.3, torch.bfloat16), rand(50, 300, dtype=torch.bfloat16), rand(50, 200, dtype=torch.bfloat16)
    r = rand(50, 200, seed=5)
    layer = void.SparseLinear(300, 200, a, dtype=torch.float32, activation="silu")
    assert layer.bias.dtype == torch.float32
    y, grads = train(layer, x, r, g)
    check_training(layer, a, x, r, g, y, grads, "silu")
    assert grads[2].dtype == torch.float32 and grads[3].dtype == torch.float32
    bare = void.SparseLinear(300, 200, a, bias=False, activation="silu")
    y2 = bare(x)
    grads2 = torch.autograd.grad(y2, (x, bare.sparse_weight.values), g)
    assert torch.equal(grads2[0], grads[0]) and torch.equal(grads2[1], grads[1])       # (the bias was zero)


@pytest.mark.parametrize("want", [(0,), (1,), (2,), (3,), (2, 3)])
def test_only_the_gradients_that_are_wanted(want):
    a, g = weight(64, 96, 0.5, torch.float16), rand(20, 64, dtype=torch.float16)
    layer = void.SparseLinear(96, 64, a, activation="gelu")
    x, r = rand(20, 96, dtype=torch.float16), rand(20, 64, dtype=torch.float16)
    full = train(layer, x, r, g)[1]
    for t in (x, layer.sparse_weight.values, layer.bias, r):
        t.requires_grad_(False)
    args = [x, layer.sparse_weight.values, layer.bias, r]
    for i in want:
        args[i].requires_grad_(True)
    got = torch.autograd.grad(layer(x, residual=r), [args[i] for i in want], g)
    assert all(torch.equal(p, full[i]) for p, i in zip(got, want))


def test_gradient_of_a_sum_and_odd_gradients():
    a, x = weight(45, 70, 0.5, torch.bfloat16), rand(9, 70, dtype=torch.bfloat16)
    layer = void.SparseLinear(70, 45, a, activation="relu")
    y = layer(x.requires_grad_(True))
    ones = torch.ones_like(y)
    got = torch.autograd.grad(y.sum(), (x, layer.sparse_weight.values, layer.bias))
    check_training(layer, a, x, None, ones, y, got, "relu")
    g = rand(45, 9, dtype=torch.bfloat16).t()                       # columns far apart
    y = layer(x)
    check_training(layer, a, x, None, g, y, torch.autograd.grad(y, (x, layer.sparse_weight.values, layer.bias), g), "relu")


def test_x_as_residual_gets_both_gradients():
    a, x, g = weight(96, 96, 0.5, torch.bfloat16), rand(30, 96, dtype=torch.bfloat16), rand(30, 96, dtype=torch.bfloat16)
    layer = void.SparseLinear(96, 96, a, activation="gelu")
    (alone,) = torch.autograd.grad(layer(x.requires_grad_(True)), x, g)
    (both,) = torch.autograd.grad(layer(x, residual=x), x, g)
    within(both, alone.double() + g.double(), HALF[torch.bfloat16] * (alone.double() + g.double()).abs())


def test_directional_differences():
    a = weight(64, 96, 0.5, torch.float16)
    x, g = rand(12, 96, dtype=torch.float16), rand(12, 64, dtype=torch.float16)
    layer = void.SparseLinear(96, 64, a, activation="gelu")
    _, grads = train(layer, x, None, g)
    xd, ad, gd = x.detach().double(), a.to_dense().double(), g.double()
    h = 1e-5
    step = rand(12, 96, seed=9).double()
    diff = float(((act64((xd + h * step) @ ad.t(), "gelu") - act64((xd - h * step) @ ad.t(), "gelu")) * gd).sum() / (2 * h))
    # z and dz are kept in fp16 and so is the result: three roundings, at most 2^-11 of each summand in the sum they go through
    z = xd @ ad.t()
    size = float((((gd.abs() * (1 + z.abs())) @ ad.abs()) * step.abs()).sum())
    assert abs(float((grads[0].double() * step).sum()) - diff) < 4 * HALF[torch.float16] * size


def test_batches_of_sequences():
    a, x = weight(64, 96, 0.5, torch.bfloat16), rand(24, 96, dtype=torch.bfloat16)
    r, g = rand(24, 64, dtype=torch.bfloat16, seed=2), rand(24, 64, dtype=torch.bfloat16, seed=3)
    layer = void.SparseLinear(96, 64, a, activation="silu")
    flat, grads = train(layer, x, r, g)
    x3, r3 = x.detach().view(2, 3, 4, 96).requires_grad_(True), r.detach().view(2, 3, 4, 64).requires_grad_(True)
    y3 = layer(x3, residual=r3)
    grads3 = torch.autograd.grad(y3, (x3, layer.sparse_weight.values, layer.bias, r3), g.view(2, 3, 4, 64))
    assert torch.equal(y3.view(24, 64), flat) and all(torch.equal(p.reshape(q.shape), q) for p, q in zip(grads3, grads))
    with pytest.raises(AssertionError, match="residual"):
        layer(x3, residual=r3[0])


def test_refusals():
    a, x, r = weight(64, 96, 0.5, torch.bfloat16), rand(6, 96, dtype=torch.bfloat16), rand(6, 64, dtype=torch.bfloat16)
    layer = void.SparseLinear(96, 64, a, activation="gelu")
    with pytest.raises(AssertionError, match="residual"):
        void.void_linear(a, x, residual=r[:5])
    with pytest.raises(_lib.VoidB200Error, match="residual must be"):
        layer(x, residual=r[:, :63])
    with pytest.raises(_lib.VoidB200Error, match="unsupported"):
        void.void_linear(a, x, residual=r.double())
    with pytest.raises(_lib.VoidB200Error, match="no CPU path"):
        void.void_linear(a, x, residual=r.cpu())
    y = layer(x.requires_grad_(True))
    with pytest.raises(NotImplementedError, match="second derivative"):
        torch.autograd.grad(y.sum(), x, create_graph=True)
    torch.autograd.grad(y.sum(), x)
    with pytest.raises(RuntimeError, match="second time|freed"):
        torch.autograd.grad(y.sum(), x)


# ------------------------------------------------------------------------------------------ the layers together
def feed_forward64(x, norm, w1, b1, w2, b2, act, dtype):
    """x + W2 act(W1 norm(x) + b1) + b2 with its bound: every stage's result is rounded to ``dtype``."""
    xd = x.double()
    h, e = xd, None
    if norm is not None:
        w, b = (None if t is None else t.detach().double() for t in norm)
        h, unit, rstd = norm64(xd, w, b, 1e-5)
        e = forward_bound(xd, w, b, unit, rstd, h, dtype)
    _, hidden, _, e = layer64(h, w1.to_dense().double(), b1, None, act, dtype, e)
    _, y, _, e = layer64(hidden, w2.to_dense().double(), b2, xd, "none", dtype, rounded(e, hidden, dtype))
    return y, rounded(e, y, dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n, k, m", [(1, 64, 160), (8, 256, 512), (70, 333, 1000), (2048, 1024, 4096)])
def test_feed_forward_inference(n, k, m, dtype):
    w1, w2, x = weight(m, k, 0.3, dtype), weight(k, m, 0.3, dtype), rand(n, k, dtype=dtype)
    b1, b2, norm = rand(m, seed=1), rand(k, seed=2), (rand(k, dtype=dtype, scale=0.2) + 1, rand(k, dtype=dtype, seed=3))
    for _ in range(2):    # (packed on the first call)
        y = void.fused_sparse_mlp(x, w1, w2, "gelu", b1, b2, residual=x, norm=norm)
        ref, e = feed_forward64(x, norm, w1, b1.double(), w2, b2.double(), "gelu", dtype)
        within(y, ref, e)
    y = void.fused_sparse_mlp(x, w1, w2, "silu", residual=x)
    ref, e = feed_forward64(x, None, w1, None, w2, None, "silu", dtype)
    within(y, ref, e)
    if n == 8:
        y3 = void.fused_sparse_mlp(x.view(2, 4, k), w1, w2, "silu", residual=x.view(2, 4, k))
        assert y3.shape == (2, 4, k) and torch.equal(y3.view(8, k), y)


def test_feed_forward_module_matches_its_parts_and_trains():
    dtype = torch.bfloat16
    w1, w2 = weight(640, 200, 0.3, dtype), weight(200, 640, 0.3, dtype)
    block = void.SparseFeedForward(w1, w2)
    x, g = rand(90, 200, dtype=dtype), rand(90, 200, dtype=dtype, seed=4)
    y = block(x.requires_grad_(True))
    ref, e = feed_forward64(x.detach(), (block.norm.weight, block.norm.bias), w1, None, w2, None, "gelu", dtype)
    within(y, ref, e)
    y.backward(g)
    assert all(p.grad is not None and bool(p.grad.isfinite().all()) for p in block.parameters()) and x.grad is not None
    # the same parts one after the other
    x2 = x.detach().clone().requires_grad_(True)
    y2 = block.down(block.up(block.norm(x2)), residual=x2)
    assert torch.equal(y2, y)
    grads = torch.autograd.grad(y2, [x2] + list(block.parameters()), g)
    assert all(torch.equal(p, q) for p, q in zip(grads, [x.grad] + [p.grad for p in block.parameters()]))
    # inference over packed weights: the same numbers up to its own roundings
    z = void.fused_sparse_mlp(x.detach(), w1, w2, "gelu", block.up.bias.detach(), block.down.bias.detach(), residual=x.detach(),
                              norm=(block.norm.weight.detach(), block.norm.bias.detach()))
    within(z, ref, e)
    assert void.SparseFeedForward(w1, w2, norm=False).norm is None


def test_training_step_in_a_graph_and_on_another_stream():
    dtype = torch.bfloat16
    block = void.SparseFeedForward(weight(320, 96, 0.4, dtype), weight(96, 320, 0.4, dtype), "silu")
    x, g = rand(64, 96, dtype=dtype).requires_grad_(True), rand(64, 96, dtype=dtype, seed=4)
    leaves = [x] + list(block.parameters())

    def step():
        y = block(x)
        return [y.detach()] + list(torch.autograd.grad(y, leaves, g))
    expected = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        on_side = step()
    side.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(on_side, expected))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    with torch.no_grad():
        x.copy_(rand(64, 96, dtype=dtype, seed=77))
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(outs, step()))


def test_inference_in_a_graph():
    dtype = torch.float16
    w1, w2, x = weight(320, 96, 0.4, dtype), weight(96, 320, 0.4, dtype), rand(8, 96, dtype=dtype)
    norm = (rand(96, dtype=dtype) + 1, rand(96, dtype=dtype, seed=1))
    call = lambda: void.fused_sparse_mlp(x, w1, w2, "gelu", residual=x, norm=norm)   # noqa: E731
    call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = call()
    x.copy_(rand(8, 96, dtype=dtype, seed=50))
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, call())
