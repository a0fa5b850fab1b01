"""Layer norm, linear layers and layers of experts where a call is unusual: captured while something else lives, two graphs on one
weight, waits that run out, results and residuals that lie anyhow."""
import ctypes

import pytest
import torch

import void_b200 as void
from test_experts_gpu import check_forward, experts_of, offsets_of
from test_linear_cpu import layer64, rounded, within
from test_linear_gpu import rand, weight
from test_norm_gpu import check, make
from void_b200 import _lib

pytestmark = pytest.mark.gpu


def _steps():
    dtype = torch.bfloat16
    x = rand(40, 96, dtype=dtype).requires_grad_(True)
    linear = void.SparseLinear(96, 64, weight(64, 96, 0.5, dtype), activation="gelu")
    layer = void.SparseExperts(experts_of(2, 64, 96, 0.5, dtype)[1], activation="silu")
    norm = void.VOIDLayerNorm(96, dtype=dtype)
    offsets = offsets_of([25, 15])
    return [(x, linear, lambda: linear(x)), (x, layer, lambda: layer(x, offsets)), (x, norm, lambda: norm(x))]


@pytest.mark.parametrize("which", range(3))
def test_backward_captured_while_an_eager_graph_of_the_leaves_lives(which):
    x, module, forward = _steps()[which]
    leaves = [x] + [p for p in module.parameters() if p.requires_grad]
    alive = forward()                                   # recorded on the default stream, and not given up
    want = torch.autograd.grad(alive, leaves, torch.ones_like(alive), retain_graph=True)
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="recorded on the default stream lives"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            y = forward()
            torch.autograd.grad(y, leaves, torch.ones_like(y))
    torch.cuda.synchronize()
    y = None
    again = torch.autograd.grad(alive, leaves, torch.ones_like(alive))   # the eager graph is as it was
    assert all(torch.equal(p, q) for p, q in zip(want, again))
    del alive, again
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = forward()
        got = torch.autograd.grad(y, leaves, torch.ones_like(y))
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(want, got))


# Results and residuals with pitches and beginnings of any number of elements: written and read by eight lanes together.  The buffers
# around them stay what they were.
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n, k, m", [(33, 96, 45), (129, 64, 33), (300, 160, 98), (1000, 96, 1001), (40, 96, 31)])
@pytest.mark.parametrize("pad, first", [(0, 0), (1, 0), (2, 2), (5, 3)])
def test_results_and_residuals_that_lie_anyhow(pad, first, n, k, m, dtype):
    a, x, bias = weight(m, k, 0.4, dtype), rand(n, k, dtype=dtype), rand(m, seed=1)
    around, behind = rand(n, m + pad + first, dtype=dtype, seed=2), rand(n, m + 3, dtype=dtype, seed=3)
    was, out, residual = around.clone(), around[:, first:first + m], behind[:, 1:1 + m]
    dense = a.to_dense().double()
    for r, act, code in ((None, "none", 0), (residual, "gelu", 2), (residual.float(), "silu", 3)):
        void.void_linear(a, x, bias, code, out, residual=r)
        _, ref, _, err = layer64(x.double(), dense, bias.double(), None if r is None else r.double(), act, dtype)
        within(out, ref, rounded(err, ref, dtype))
        assert torch.equal(around[:, :first], was[:, :first]) and torch.equal(around[:, first + m:], was[:, first + m:])
    mine = out.clone()                                  # in place: the residual stream is the result
    void.void_linear(a, x, bias, 1, out, residual=out)
    _, ref, _, err = layer64(x.double(), dense, bias.double(), mine.double(), "relu", dtype)
    within(out, ref, rounded(err, ref, dtype))
    assert torch.equal(around[:, :first], was[:, :first]) and torch.equal(around[:, first + m:], was[:, first + m:])
    void.check_device_status()


@pytest.mark.parametrize("each", [3, 7, 60, 200])     # every chunk length, and so every kernel
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_experts_into_a_result_that_lies_anyhow(each, dtype):
    counts = [each, 0, 2 * each - 1, 1]
    weights, e = experts_of(4, 45, 96, 0.5, dtype)
    tokens = sum(counts) + 3
    x, bias, around = rand(tokens, 96, dtype=dtype), rand(4, 45, dtype=dtype, seed=1), rand(tokens, 50, dtype=dtype, seed=2)
    was, out = around.clone(), around[:, 3:48]
    void.void_expert_linear(e, x, offsets_of(counts, 1), bias, 2, out=out)
    check_forward(out, weights, x, counts, 1, bias, "gelu", untouched=was[:, 3:48])
    assert torch.equal(around[:, :3], was[:, :3]) and torch.equal(around[:, 48:], was[:, 48:])
    void.check_device_status()


@pytest.mark.parametrize("each", [3, 7, 60, 200])
def test_infinities_of_other_tokens_stay_with_them(each):
    counts = [each, 2, 2 * each - 1, 0, 1]
    weights, e = experts_of(5, 72, 96, 0.5, torch.float16)
    tokens, offsets = sum(counts) + 5, offsets_of(counts, 2)
    x, bias = rand(tokens, 96, dtype=torch.float16), rand(5, 72, seed=1)
    clean = void.void_expert_linear(e, x, offsets, bias, 3)
    bad, rows = x.clone(), torch.ones(tokens, dtype=torch.bool, device="cuda")
    for at, value in ((0, "nan"), (1, "inf"), (2 + each, "nan"), (tokens - 4, "-inf"), (tokens - 1, "nan"), (4 + each, "inf")):
        bad[at], rows[at] = float(value), False
    y = void.void_expert_linear(e, bad, offsets, bias, 3)
    assert torch.equal(y[rows], clean[rows])
    assert not y[[0, 1, tokens - 1]].any() and not y[2 + each].isfinite().any()


def test_a_result_of_experts_that_is_its_input_is_refused():
    e, x = experts_of(2, 64, 64, 0.5, torch.float16)[1], rand(10, 64, dtype=torch.float16)
    with pytest.raises(_lib.VoidB200Error, match="must not be x"):
        void.void_expert_linear(e, x, offsets_of([4, 6]), out=x)


# (rows enough for the blocks that stay, whose threads take sixteen elements one by one up to 6144, and 32 beyond)
@pytest.mark.parametrize("dtype, params", [(torch.float32, torch.float32), (torch.bfloat16, torch.float32), (torch.float16, torch.float16)])
@pytest.mark.parametrize("rows, cols", [(1800, 4097), (1900, 5003), (1777, 6143), (1800, 6145), (2300, 4095), (2000, 8191)])
def test_norm_of_many_rows_that_lie_in_no_pieces(rows, cols, dtype, params):
    x, w, b, g = make(rows, cols, dtype, params)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    y = void.void_layer_norm(x, w, b)
    check(x, w, b, g, y, torch.autograd.grad(y, leaves, g))


# The slope of ReLU is one where z is positive, however near to zero: with gradients of ones the bias's is the number of such tokens.
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("n, k, m, density", [(700, 8192, 2048, 0.3), (300, 5003, 3001, 0.5), (2000, 1024, 1000, 1.0)])
def test_slopes_next_to_the_border_of_relu(n, k, m, density, dtype):
    a, x = weight(m, k, density, dtype), rand(n, k, dtype=dtype).requires_grad_(True)
    layer = void.SparseLinear(k, m, a, dtype=torch.float32, activation="relu")
    with torch.no_grad():
        layer.bias.copy_(rand(m, seed=1, scale=0.1))
    y = layer(x)
    counts, = torch.autograd.grad(y, (layer.bias,), torch.ones_like(y))
    z = x.detach().double() @ a.to_dense().double().t() + layer.bias.detach().double()
    assert torch.equal(counts, (z > 0).sum(0).float())
    weights, e = experts_of(3, m, k, density, dtype)
    runs, bias = [n // 2, 0, n // 3], rand(3, m, seed=2, scale=0.1)
    experts = void.SparseExperts(e, activation="relu", dtype=torch.float32)
    with torch.no_grad():
        experts.bias.copy_(bias)
    y = experts(x, offsets_of(runs, 5))
    counts, = torch.autograd.grad(y, (experts.bias,), torch.ones_like(y))
    at = 5
    for i, c in enumerate(runs):
        z = x.detach()[at:at + c].double() @ weights[i].to_dense().double().t() + bias[i].double()
        assert torch.equal(counts[i], (z > 0).sum(0).float())
        at += c


# z = a + 2^-25 - a: what fp16 rounds to nothing, or the sum loses beside a; and its negative.
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("n", [3, 40, 300])
def test_slopes_of_sums_that_their_bias_takes_to_nothing(n, dtype):
    a = weight(64, 32, 1.0, dtype)
    a.values.zero_()
    sizes = [0.25, 0.25, 1.0, 1.0, 64.0, 64.0]
    for i, size in enumerate(sizes):                      # rows of the first tile
        a.values[0, i, 0], a.values[0, i, 1] = size, 2.0 ** -13 * (1 if i % 2 == 0 else -1)
    a.values[0, 31, 0] = 4.0
    x = torch.zeros(n, 32, dtype=dtype, device="cuda")
    x[:, 0], x[:, 1] = 1.0, 2.0 ** -12
    bias = torch.zeros(64, device="cuda")
    bias[:len(sizes)] = -torch.tensor(sizes, device="cuda")
    want = torch.zeros(64, device="cuda")
    want[[0, 2, 4, 31]] = float(n)
    layer = void.SparseLinear(32, 64, a, dtype=torch.float32, activation="relu")
    experts = void.SparseExperts(void.stack_experts([a, a]), activation="relu", dtype=torch.float32)
    with torch.no_grad():
        layer.bias.copy_(bias)
        experts.bias.copy_(bias)
    y = layer(x.requires_grad_(True))
    assert torch.equal(torch.autograd.grad(y, (layer.bias,), torch.ones_like(y))[0], want)
    y = experts(x, offsets_of([n, 0]))
    counts, = torch.autograd.grad(y, (experts.bias,), torch.ones_like(y))
    assert torch.equal(counts[0], want) and not counts[1].any()


DROP_FIRST_GROUP = 1 << 16


@pytest.mark.parametrize("chunk", [8, 32, 64, 128])
def test_a_wait_of_the_experts_kernels_runs_out_with_a_status(chunk):
    weights, e = experts_of(3, 64, 256, 0.5, torch.bfloat16)
    counts = [9, 0, 70]
    x, offsets = rand(79, 256, dtype=torch.bfloat16), offsets_of(counts)
    want = void.void_expert_linear(e, x, offsets)
    torch.cuda.synchronize()
    void.check_device_status()
    p, lib = next(iter(e.tensor._packed_fp_cache.values())), _lib.load()
    plan = torch.zeros(lib.void_expert_plan_words(3, 79, chunk), dtype=torch.int32, device="cuda")
    stream, status = torch.cuda.current_stream().cuda_stream, _lib.status_word(x.device)
    assert lib.void_expert_plan(offsets.data_ptr(), 4, 3, 79, chunk, plan.data_ptr(), status.data_ptr(), stream) == 0
    got = torch.zeros_like(want)
    a = _lib.SpmmArgs()
    a.tiles, a.tile_cols, a.row_ptr, a.nbr, a.nnz, a.M, a.K, a.N = p.tiles.data_ptr(), p.tile_cols.data_ptr(), p.row_ptr.data_ptr(), 2, p.nnz, 64, 256, 79
    a.nbc, a.b, a.ldb, a.b_scale, a.out, a.ldc, a.out_dtype, a.transposed = 8, x.data_ptr(), 512, 1.0, got.data_ptr(), 64, _lib.OUT_DTYPE_CODE[x.dtype], 1
    a.status = status.data_ptr()
    experts = _lib.Experts(plan=plan.data_ptr(), n_experts=3, chunk=chunk, zero_rest=1)

    def launch(hooks):
        a.test_hooks = hooks
        assert lib.void_expert_linear(ctypes.byref(a), None, ctypes.byref(experts), _lib.KIND_BF16, stream) == 0
        torch.cuda.synchronize()
    launch(DROP_FIRST_GROUP | 5)                        # no CTA gets its first tiles; its waits are limited to 5 ms
    with pytest.raises(void.VoidB200Error, match="wait gave up"):
        void.check_device_status()
    launch(0)
    void.check_device_status()
    check_forward(got, weights, x, counts, 0, None, "none")


def test_two_graphs_of_one_weight_replayed_side_by_side():
    dtype = torch.bfloat16
    weights, e = experts_of(4, 200, 160, 0.4, dtype)
    a = weight(160, 200, 0.4, dtype)
    norm = (rand(160, seed=1), rand(160, seed=2))
    runs = [([30, 0, 200, 11], rand(241, 160, dtype=dtype, seed=3)), ([1, 2, 0, 4], rand(7, 160, dtype=dtype, seed=4))]
    offsets = [offsets_of(c) for c, _ in runs]

    def call(i):
        x = runs[i][1]
        h = void.void_layer_norm(x, *norm)
        return void.void_linear(a, void.void_expert_linear(e, h, offsets[i], None, 3), None, 0, residual=x)
    want = [call(0), call(1)]
    torch.cuda.synchronize()
    graphs, outs, streams = [], [], [torch.cuda.Stream(), torch.cuda.Stream()]
    for i in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[i]):
            outs.append(call(i))
    for _ in range(20):
        for i in (0, 1):
            with torch.cuda.stream(streams[i]):
                graphs[i].replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1])
    void.check_device_status()
