"""Linear layers, layers of experts and layer norm where an operand is at an edge: biases in 16 bits on a transposed copy, sums that
a bias cancels, results that share memory with an operand, rows longer than a block's registers."""
import pytest
import torch

import void_b200 as void
from test_experts_gpu import experts_of, offsets_of
from test_linear_cpu import U, rounded, within
from test_linear_gpu import feed_forward64, rand, weight
from test_norm_cpu import norm64, norm_grad64
from test_norm_gpu import backward_bounds, make
from void_b200 import _lib

pytestmark = pytest.mark.gpu


# (large enough that one transposed copy of x pays for both layers: nothing else transposes)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("groups", [True, False])
def test_mlp_with_biases_of_16_bits_on_a_transposed_copy(groups, dtype):
    w1, w2, x = weight(8192, 1024, 0.3, dtype), weight(1024, 8192, 0.3, dtype), rand(2048, 1024, dtype=dtype)
    b1, b2 = rand(8192, seed=1, dtype=dtype), rand(1024, seed=2, dtype=dtype)
    for w in (w1, w2):
        void.allow_group_stores(w, groups)
    ref, e = feed_forward64(x, None, w1, b1.double(), w2, b2.double(), "gelu", dtype)
    for _ in range(5):       # (the first calls pack, the later ones may find stores for groups of tile rows)
        within(void.fused_sparse_mlp(x, w1, w2, "gelu", b1, b2, residual=x), ref, e)
        torch.cuda.synchronize()
    odd = rand(2048, 1032, dtype=dtype)[:, 1:1025]       # a residual that lies in no 16-byte pieces
    within(void.fused_sparse_mlp(x, w1, w2, "gelu", b1, b2, residual=odd), ref - x.double() + odd.double(), e + e)


TYPES = [torch.float16, torch.bfloat16, torch.float32]


def relu_layers(dense, bias, dtype):
    """A linear layer and a layer of two experts with these weights, in training with ReLU; and how they are called on n tokens."""
    a = void.dense_to_void(dense.to(dtype), threshold=-1.0)
    layer = void.SparseLinear(dense.shape[1], dense.shape[0], a, dtype=torch.float32, activation="relu")
    experts = void.SparseExperts(void.stack_experts([a, a]), activation="relu", dtype=torch.float32)
    with torch.no_grad():
        layer.bias.copy_(bias)
        experts.bias.copy_(bias)
    return [(layer, layer.sparse_weight.values, lambda x: layer(x)),
            (experts, experts.values, lambda x: experts(x, offsets_of([x.shape[0] - x.shape[0] // 3, x.shape[0] // 3])))]



@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m", [64, 45])
def test_infinite_gradients_stop_where_relu_has_no_slope(m, dtype):
    dense, bias = weight(m, 96, 1.0, torch.float32).to_dense(), rand(m, seed=1)
    x, g = rand(40, 96, dtype=dtype), rand(40, m, dtype=dtype, seed=3)
    bias[7] = -1e4 if dtype != torch.float16 else -1e3
    bad = g.clone()
    g[:, 7] = 0.0
    bad[:, 7] = float("inf")
    bad[3, 7] = float("nan")
    for layer, values, call in relu_layers(dense, bias, dtype):
        got = [torch.autograd.grad(call(x.requires_grad_(True)), (x, values, layer.bias), t) for t in (g, bad)]
        assert all(torch.equal(p, q) for p, q in zip(*got))


def tile_rows(layer):
    return layer.block_rows if isinstance(layer, void.SparseExperts) else layer.sparse_weight.block_rows


# z = size - size = 0, in one output of many or in all of them: zero, without a slope.
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("size", [1.0, 2.0 ** -10, 2.0 ** -30])
@pytest.mark.parametrize("n", [1, 8, 40, 300])
@pytest.mark.parametrize("alone", [True, False])
def test_a_sum_that_its_bias_cancels_is_zero_and_has_no_slope(alone, n, size, dtype):
    m, k = 64, 96
    size = max(size, 2.0 ** -24) if dtype == torch.float16 else size
    dense, bias = weight(m, k, 1.0, torch.float32).to_dense(), rand(m, seed=1)
    rows = torch.tensor([5] if alone else list(range(m)), device="cuda")
    dense[rows] = 0.0
    dense[rows, 0] = size
    bias[rows] = -size
    x, g = rand(n, k, dtype=dtype), rand(n, m, dtype=dtype, seed=3)
    x[:, 0] = 1.0
    for layer, values, call in relu_layers(dense, bias, dtype):
        y = call(x.requires_grad_(True))
        dx, dv, db = torch.autograd.grad(y, (x, values, layer.bias), g)
        assert not y[:, rows].any() and not db[..., rows].any()
        assert not (dv[tile_rows(layer) % 2 == 0][:, 5].any() if alone else dv.any() or dx.any())


# Sums around half of fp16's smallest number: the result is the sum rounded, the slope asks for its sign.
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [1, 8, 40, 300])
def test_results_in_training_are_those_of_the_sums(n, dtype):
    dense, bias = torch.zeros(32, 64, device="cuda"), torch.zeros(32, device="cuda")
    dense[:8, 0] = 2.0 ** -13 * torch.tensor([0.5, -0.5, 1.0, -1.0, 1.5, -1.5, 0.25, -0.25], device="cuda")
    dense[8, 0], bias[9] = 1.0, 2.0 ** -26
    x = torch.zeros(n, 64, dtype=dtype, device="cuda")
    x[:, 0] = 2.0 ** -12
    z = dense[:, 0].double() * 2.0 ** -12 + bias.double()
    for layer, _, call in relu_layers(dense, bias, dtype):
        y = call(x.requires_grad_(True))
        db, = torch.autograd.grad(y, (layer.bias,), torch.ones_like(y))
        assert torch.equal(y, z.clamp_min(0).to(dtype).expand(n, 32))
        assert torch.equal(db.reshape(-1, 32).sum(0), n * (z > 0).float())


# Every sum of a token is all but cancelled by its bias: what is left, some 2^-24 of the sum, has to give the slope.
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("n, scale", [(1, 1.0), (40, 1.0), (300, 1.0), (40, 100.0)])
def test_slopes_of_a_token_whose_sums_are_all_cancelled(n, scale, dtype):
    m, k = 256, 3200
    dense, x = weight(m, k, 1.0, torch.float32).to_dense().to(dtype).float(), rand(n, k, dtype=dtype)
    x[0] *= scale
    sums = x[0].double() @ dense.double().t()
    nudge = (torch.arange(m, device="cuda") % 7 - 3).double() * 2.0 ** -23
    bias = -(sums * (1.0 + nudge)).float()
    g = torch.zeros(n, m, dtype=dtype, device="cuda")
    g[0] = 1.0
    for layer, _, call in relu_layers(dense, bias, dtype):
        y = call(x.requires_grad_(True))
        db, = torch.autograd.grad(y, (layer.bias,), g)
        assert torch.equal(db.reshape(-1, m).sum(0), (sums + bias.double() > 0).float())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_slopes_are_the_same_every_time_where_most_sums_are_cancelled(dtype):
    m, k, n = 300, 1600, 333
    dense, x = weight(m, k, 1.0, torch.float32).to_dense().to(dtype).float(), rand(1, k, dtype=dtype).expand(n, k).contiguous()
    bias = -(x[0].double() @ dense.double().t()).float()
    for layer, values, call in relu_layers(dense, bias, dtype):
        grads = []
        for _ in range(3):
            y = call(x.requires_grad_(True))
            grads.append(torch.autograd.grad(y, (x, values, layer.bias), torch.ones_like(y)))
        assert all(torch.equal(p, q) for other in grads[1:] for p, q in zip(grads[0], other))
        assert bool((grads[0][2] >= 0).all()) and bool((y >= 0).all()) and float(y.detach().max()) < 1e-3


# dx may take the place of g or of x, through the C ABI, in rows of every length.
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("place", ["g", "x"])
@pytest.mark.parametrize("rows, cols", [(5, 100), (700, 1024), (9, 8200), (40, 8201), (33, 20000), (700, 16392)])
def test_norm_gradient_in_the_place_of_an_operand(rows, cols, place, dtype):
    x, w, b, g = make(rows, cols, dtype, torch.float32)
    lib, elem, stream = _lib.load(), _lib.ELEM_CODE[dtype], torch.cuda.current_stream().cuda_stream
    y, stats = torch.empty_like(x), torch.empty(2, rows, device="cuda")
    assert lib.void_layer_norm(x.data_ptr(), elem, cols, rows, cols, w.data_ptr(), b.data_ptr(), _lib.ELEM_CODE[torch.float32], 1e-5, y.data_ptr(), cols,
                               stats.data_ptr(), stream) == 0
    xd, wd, gd = x.double(), w.double(), g.double()
    _, unit, rstd = norm64(xd, wd, b.double(), 1e-5)
    refs = norm_grad64(gd, unit, rstd, wd)
    bounds = backward_bounds(xd, wd, gd, unit, rstd, *refs, dtype, torch.float32)
    dx = g if place == "g" else x
    dw, db = torch.empty_like(w), torch.empty_like(w)
    ws = torch.empty(lib.void_layer_norm_grad_ws_bytes(rows, cols), dtype=torch.uint8, device="cuda")
    assert lib.void_layer_norm_grad(g.data_ptr(), cols, x.data_ptr(), cols, elem, rows, cols, w.data_ptr(), _lib.ELEM_CODE[torch.float32], stats.data_ptr(),
                                    dx.data_ptr(), cols, dw.data_ptr(), db.data_ptr(), ws.data_ptr(), ws.numel(), stream) == 0
    for got, ref, bound in zip((dx, dw, db), refs, bounds):
        within(got, ref, bound)


def test_norm_into_memory_that_an_operand_shares():
    x, w, b, _ = make(300, 1000, torch.bfloat16, torch.bfloat16)
    want = void.void_layer_norm(x, w, b)
    buf = torch.empty(303, 1000, dtype=torch.bfloat16, device="cuda")
    for first, to in ((0, 3), (3, 0), (0, 0), (1, 2)):        # rows further on, further back, the very same
        buf[first:first + 300] = x
        out = buf[to:to + 300]
        assert void.void_layer_norm(buf[first:first + 300], w, b, out=out) is out and torch.equal(out, want)
    wide = torch.empty(300, 1008, dtype=torch.bfloat16, device="cuda")
    wide[:, :1000] = x                                       # the same beginning, another pitch
    out = wide.flatten()[:300000].view(300, 1000)
    assert torch.equal(void.void_layer_norm(wide[:, :1000], w, b, out=out), want)
    buf[0], buf[1] = w, b                                    # parameters where the first rows of the result will be
    assert torch.equal(void.void_layer_norm(x, buf[0], buf[1], out=buf[:300]), want)


def test_experts_into_memory_that_an_operand_shares_is_refused():
    weights, e = experts_of(2, 64, 64, 0.5, torch.float16)
    offsets, x = offsets_of([4, 6]), rand(10, 64, dtype=torch.float16)
    want = void.void_expert_linear(e, x, offsets)
    buf = torch.empty(22, 64, dtype=torch.float16, device="cuda")
    for first, to in ((0, 1), (9, 0), (5, 5)):
        with pytest.raises(_lib.VoidB200Error, match="must not be x, nor"):
            void.void_expert_linear(e, buf[first:first + 10], offsets, out=buf[to:to + 10])
    pair = torch.empty(10, 128, dtype=torch.float16, device="cuda")
    with pytest.raises(_lib.VoidB200Error, match="must not be x, nor"):
        void.void_expert_linear(e, pair[:, :64], offsets, out=pair[:, 56:120])
    pair[:, 64:] = x                                         # side by side, behind one another: nothing in common
    assert torch.equal(void.void_expert_linear(e, pair[:, 64:], offsets, out=pair[:, :64]), want) and torch.equal(pair[:, 64:], x)
    buf[12:] = x
    assert torch.equal(void.void_expert_linear(e, buf[12:], offsets, out=buf[:10]), want)
    with pytest.raises(_lib.VoidB200Error, match="bias or the offsets"):
        void.void_expert_linear(e, x, offsets, buf[:2], out=buf[:10])
    with pytest.raises(_lib.VoidB200Error, match="row-major"):
        void.void_expert_linear(e, x.float(), offsets, out=torch.empty(2, 10, 64, device="cuda"))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [3, 40, 300])
def test_a_layer_into_its_own_tokens(n, dtype):
    a, x = weight(200, 200, 0.5, dtype), rand(n, 200, dtype=dtype)
    want = void.void_linear(a, x, residual=x)
    stream = x.clone()
    assert torch.equal(void.void_linear(a, stream, out=stream, residual=stream), want)
    buf = torch.empty(n + 1, 200, dtype=dtype, device="cuda")
    buf[1:] = x
    assert torch.equal(void.void_linear(a, buf[1:], out=buf[:n], residual=x), want)


def test_a_result_that_was_given_counts_as_written():
    dtype = torch.bfloat16
    a, e = weight(64, 64, 0.5, dtype), experts_of(2, 64, 64, 0.5, dtype)[1]
    x, r = rand(10, 64, dtype=dtype), rand(10, 64, dtype=dtype, seed=1)
    for write in (lambda out: void.void_expert_linear(e, x, offsets_of([4, 6]), out=out), lambda out: void.void_linear(a, x, out=out, residual=out),
                  lambda out: void.void_layer_norm(x, out=out), lambda out: void.void_spmv(a, x[0], out=out[0])):
        factor, out = torch.ones(10, 64, dtype=dtype, device="cuda", requires_grad=True), r.clone()
        y = factor * out
        write(out)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.sum().backward()
    with torch.inference_mode():
        out = torch.empty_like(r)
        void.void_expert_linear(e, x, offsets_of([4, 6]), out=out)
        void.void_linear(a, x, out=out, residual=r)


# A layer's product counts once towards the third one, behind which a store for groups of tile rows is built.
def test_a_linear_layer_is_counted_once_before_a_group_store_is_built():
    a, x = weight(4096, 4096, 0.45, torch.bfloat16), rand(2048, 4096, dtype=torch.bfloat16)
    void.void_linear(a, x)
    torch.cuda.synchronize()
    held = torch.cuda.memory_allocated()
    void.void_linear(a, x)
    assert torch.cuda.memory_allocated() - held < a.values.numel()
    void.void_linear(a, x)
    assert torch.cuda.memory_allocated() - held > 2 * a.values.numel()


# The bias's gradient is a sum of its own type, whatever the tokens' is.
@pytest.mark.parametrize("act", ["relu", "silu", "none"])
def test_bias_gradients_in_their_own_type(act):
    a, x = weight(64, 96, 0.5, torch.bfloat16), rand(257, 96, dtype=torch.bfloat16)
    experts = void.SparseExperts(void.stack_experts([a, a]), activation=act, dtype=torch.float16)
    layers = [(experts, lambda: experts(x, offsets_of([257, 0])))]
    if act != "none":
        layer = void.SparseLinear(96, 64, a, dtype=torch.float16, activation=act)
        layers.append((layer, lambda: layer(x)))
    for layer, call in layers:
        with torch.no_grad():
            layer.bias.fill_(50.0)       # (slopes of one)
        y = call()
        db, = torch.autograd.grad(y, (layer.bias,), torch.ones_like(y))
        assert db.dtype == torch.float16 and torch.equal(db.reshape(-1, 64)[0].float(), torch.full((64,), 257.0, device="cuda"))


@pytest.mark.parametrize("density", [0.1, 0.5])
def test_int8_layers_with_a_residual_by_every_kernel(density):
    # (rows, rows on a transposed copy, groups of tile rows on that copy; a residual that lies anyhow leaves the groups)
    n, k, m = 1100, 4096, 4096
    q = void.quantize_void_tensor(weight(m, k, density, torch.float32))
    gen = torch.Generator(device="cuda").manual_seed(n)
    x = torch.randint(-128, 128, (n, k), generator=gen, device="cuda", dtype=torch.int8)
    scale, bias, around = rand(n).abs() + 0.1, rand(m, seed=1), rand(n, m + 3, dtype=torch.bfloat16, seed=2)
    row = q.block_rows.long().cpu()
    mean = torch.zeros(128, dtype=torch.float64).scatter_reduce(0, row, q.scales.double().cpu(), "mean", include_self=False).cuda()
    dense = torch.zeros(128, 128, 32, 32, device="cuda", dtype=torch.float64)
    dense[q.block_rows.long(), q.block_cols.long()] = q.values.double()
    part = (x.double() @ dense.permute(0, 2, 1, 3).reshape(m, k).t()) * mean.repeat_interleave(32) * scale.double()[:, None]
    z = part + bias.double()
    for r in (around[:, :m].contiguous(), around[:, 1:m + 1]):
        ref = z.clamp_min(0) + r.double()
        # exact sums, one rounding to fp32; the mean scale (a sum of up to K / 32 terms), two products and two sums in fp32
        e = (k / 32 + 8) * U * part.abs() + 4 * U * (bias.double().abs() + ref.abs() + r.double().abs())
        for _ in range(5):
            within(void.void_linear(q, x, bias, 1, x_scale=scale, out_dtype=torch.bfloat16, residual=r), ref, rounded(e, ref, torch.bfloat16))
            torch.cuda.synchronize()


@pytest.mark.parametrize("dtype", TYPES)
def test_weights_taken_from_a_layer_follow_its_training(dtype):
    a, x = weight(64, 96, 0.5, dtype), rand(40, 96, dtype=dtype)
    experts, layer = void.SparseExperts(void.stack_experts([a, a]), bias=False), void.SparseLinear(96, 64, a, bias=False)
    kept, matrix, offsets = experts.get_experts(), layer.sparse_weight.get_void_tensor(), offsets_of([25, 15])
    for _ in range(3):
        want, want2 = void.void_expert_linear(kept, x, offsets), void.void_linear(matrix, x)
        assert not kept.values.requires_grad and not matrix.values.requires_grad
        with torch.no_grad():                                # a step of an optimiser
            experts.values.mul_(2.0)
            layer.sparse_weight.values.mul_(2.0)
        assert torch.equal(void.void_expert_linear(kept, x, offsets), 2 * want) and torch.equal(void.void_linear(matrix, x), 2 * want2)


@pytest.mark.parametrize("dtype", TYPES)
def test_relu_in_training_captured_and_replayed_with_other_tokens(dtype):
    dense, bias = weight(200, 96, 1.0, torch.float32).to_dense(), rand(200, seed=1)
    bias[::3] = 0.0
    x, g = rand(150, 96, dtype=dtype), rand(150, 200, dtype=dtype, seed=3)
    x.requires_grad_(True)
    for layer, values, call in relu_layers(dense, bias, dtype):
        def step():
            y = call(x)
            return [y.detach(), *torch.autograd.grad(y, (x, values, layer.bias), g)]
        if isinstance(layer, void.SparseExperts):            # (the offsets are made outside: a capture copies nothing from the host)
            offsets = offsets_of([100, 50])
            call = lambda t, f=layer, o=offsets: f(t, o)     # noqa: E731
        step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = step()
        for seed in (50, 51):
            with torch.no_grad():
                x.copy_(rand(150, 96, dtype=dtype, seed=seed))
                x[7] = 0.0
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(p, q) for p, q in zip(outs, step()))
