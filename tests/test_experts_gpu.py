"""Layers of experts on the GPU, forward and backward, against their formulas in 64 bits."""
import pytest
import torch

import void_b200 as void
from test_linear_cpu import ACTS, layer64, layer_grads64, rounded, within
from test_linear_gpu import rand, tiles_of, weight
from void_b200 import _lib

pytestmark = pytest.mark.gpu
TYPES = [torch.float16, torch.bfloat16, torch.float32]


def experts_of(n, m, k, density, dtype, seed=0):
    weights = [weight(m, k, density, dtype, seed=seed + 100 * e) for e in range(n)]
    return weights, void.stack_experts(weights)


def offsets_of(counts, first=0, dtype=torch.int32):
    return torch.tensor([first] + counts, dtype=torch.int64).cumsum(0).to(dtype).cuda()


def check_forward(y, weights, x, counts, first, bias, act, untouched=None):
    """Every run against its expert; rows in no run are zeros, or what they were."""
    at = first
    rest = torch.ones(x.shape[0], dtype=torch.bool)
    for e, c in enumerate(counts):
        if c:
            run = slice(at, at + c)
            _, ref, _, err = layer64(x[run].double(), weights[e].to_dense().double(), None if bias is None else bias[e].double(), None, act, x.dtype)
            within(y[run], ref, rounded(err, ref, x.dtype))
            rest[run] = False
        at += c
    rest = rest.cuda()
    expected = torch.zeros_like(y) if untouched is None else untouched
    assert torch.equal(y[rest], expected[rest])


# experts, features in and out, tokens per expert, tokens before the first and behind the last run.  The kernels: chunks of 8, 32, 64 and
# 128 tokens (at most 4, 8, 96 tokens per expert on average, and more); experts that get none, one, all; more experts than a warp
# and than a block of the plan has threads.
CASES = [
    (1, 64, 32, [1], 0, 0), (1, 96, 200, [300], 0, 0), (3, 70, 45, [0, 5, 2], 0, 0), (4, 256, 512, [9, 0, 0, 1], 0, 3), (4, 333, 100, [0, 60, 1, 0], 2, 1),
    (2, 515, 333, [31, 33], 0, 0), (8, 1024, 640, [0, 700, 1, 129, 128, 127, 0, 3], 0, 0), (5, 128, 64, [128, 256, 0, 1, 130], 7, 60),
    (3, 96, 64, [0, 0, 0], 0, 10), (40, 64, 64, [3, 0, 9, 1] * 10, 0, 0), (70, 64, 33, [100 * (e % 7 == 3) + e % 3 for e in range(70)], 1, 5),
    (1500, 32, 32, [e % 4 for e in range(1500)], 0, 2), (2, 2048, 1000, [1000, 1300], 0, 17),
    (6, 130, 96, [40, 0, 1, 0, 3, 0], 0, 1), (2, 640, 300, [190, 1], 0, 0), (3, 1500, 90, [20, 2, 0], 1, 0),
    (32, 64, 64, [e % 5 for e in range(31)] + [40], 3, 2), (33, 64, 64, [9] + [e % 3 for e in range(32)], 0, 1), (32, 64, 40, [0] * 31 + [300], 0, 0), (2, 1500, 70, [4, 2], 0, 0),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("case", CASES, ids=lambda c: "%d-%d-%d" % c[:3])
def test_inference(case, act, dtype):
    n, k, m, counts, before, behind = case
    if n > 100 and (act != "gelu" or dtype != torch.bfloat16):
        pytest.skip("one act and type for the many experts")
    weights, e = experts_of(n, m, k, 0.3 if n <= 100 else 1.0, dtype)
    tokens = before + sum(counts) + behind
    x, bias = rand(tokens, k, dtype=dtype), rand(n, m, seed=1)
    code = void.get_activation_code(act)
    y = void.void_expert_linear(e, x, offsets_of(counts, before), bias, code)
    assert y.shape == (tokens, m) and y.dtype == dtype
    check_forward(y, weights, x, counts, before, bias, act)
    # with int64 offsets and without biases; into a matrix of one's own, whose other rows stay
    y2 = void.void_expert_linear(e, x, offsets_of(counts, before, torch.int64), None, code)
    check_forward(y2, weights, x, counts, before, None, act)
    mine = rand(tokens, m + 5, dtype=dtype, seed=8)[:, :m]
    was = mine.clone()
    assert void.void_expert_linear(e, x, offsets_of(counts, before), bias, code, out=mine) is mine
    check_forward(mine, weights, x, counts, before, bias, act, untouched=was)
    void.check_device_status()


@pytest.mark.parametrize("rows, chunk, offsets", [
    (100, 8, [0, 10, 10, 47, 100]), (100, 128, [3, 3, 3, 4, 90]), (1000, 32, [0] + [7 * e for e in range(1, 60)]), (5000, 16, list(range(0, 3001))),
    (50, 8, [0, 20, 10, 60, 55]), (50, 8, [-5, 20, 1 << 20, 30, 50]), (0, 8, [0, 0, 0]),
])
def test_plan(rows, chunk, offsets):
    n = len(offsets) - 1
    given = torch.tensor(offsets, dtype=torch.int32, device="cuda")
    plan = torch.full((_lib.load().void_expert_plan_words(n, rows, chunk),), -7, dtype=torch.int32, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    _lib.check(_lib.load().void_expert_plan(_lib.ptr(given), 4, n, rows, chunk, _lib.ptr(plan), _lib.ptr(status), _lib.stream_ptr()))
    words = plan.tolist()
    bounds, low = [], 0
    for o in offsets:
        low = max(low, min(max(o, 0), rows))
        bounds.append(low)
    chunks, ptr = [], [0]
    for e in range(n):
        chunks += [[e, a, min(a + chunk, bounds[e + 1]), 0] for a in range(bounds[e], bounds[e + 1], chunk)]
        ptr.append(len(chunks))
    assert words[0] == len(chunks) and words[4:5 + n] == bounds and words[5 + n:6 + 2 * n] == ptr
    table = (4 + 2 * (n + 1) + 3) // 4 * 4
    assert [words[table + 4 * i:table + 4 * i + 4] for i in range(len(chunks))] == chunks
    assert int(status) == (0 if bounds == offsets else 3)


@pytest.mark.parametrize("counts", [[30, 40, 50, 60], [3, 4, 5, 6], [300, 0, 200, 1]])
def test_offsets_that_are_not_in_order_are_taken_as_empty_runs_and_reported(counts):
    weights, e = experts_of(4, 64, 96, 0.4, torch.bfloat16)
    x = rand(sum(counts), 96, dtype=torch.bfloat16)
    good = offsets_of(counts).tolist()
    bad = torch.tensor([-3, good[2], good[1], good[3], good[4] + 1000], device="cuda")
    y = void.void_expert_linear(e, x, bad)
    check_forward(y, weights, x, [good[2], 0, good[3] - good[2], good[4] - good[3]], 0, None, "none")
    with pytest.raises(_lib.VoidB200Error, match="offsets"):
        void.check_device_status()
    void.check_device_status()


@pytest.mark.parametrize("counts", [[5, 9, 3], [200, 100, 30]])
def test_tokens_that_are_not_finite_stay_alone(counts):
    weights, e = experts_of(3, 64, 96, 0.5, torch.float16)
    tokens = sum(counts) + 20
    x, offsets = rand(tokens, 96, dtype=torch.float16), offsets_of(counts)
    clean = void.void_expert_linear(e, x, offsets)
    bad = x.clone()
    last = sum(counts)
    rows = [0, counts[0], last - 1]
    bad[rows] = float("nan")
    bad[last:] = float("inf")
    y = void.void_expert_linear(e, bad, offsets)
    keep = torch.ones(tokens, dtype=torch.bool, device="cuda")
    keep[rows] = False
    assert torch.equal(y[keep], clean[keep]) and not y[last:].any()


def test_layouts():
    weights, e = experts_of(3, 45, 70, 0.5, torch.bfloat16)
    counts = [70, 0, 90]
    x, offsets = rand(160, 70, dtype=torch.bfloat16), offsets_of(counts)
    base = void.void_expert_linear(e, x, offsets)
    wide = torch.zeros(160, 90, device="cuda", dtype=torch.bfloat16)
    for off in (0, 1, 8):
        wide[:, off:off + 70] = x
        assert torch.equal(void.void_expert_linear(e, wide[:, off:off + 70], offsets), base)
    assert torch.equal(void.void_expert_linear(e, x.t().contiguous().t(), offsets), base)
    assert torch.equal(void.void_expert_linear(e, x, torch.stack([offsets, offsets], 1)[:, 0]), base)
    # weights of another type: the product in fp32 operands
    y = void.void_expert_linear(e.to_dtype(torch.float32), x, offsets)
    check_forward(y, weights, x, counts, 0, None, "none")
    mine = rand(160, 45, dtype=torch.bfloat16, seed=3)
    void.void_expert_linear(e.to_dtype(torch.float32), x, offsets, out=mine)
    assert torch.equal(mine, y)
    assert void.void_expert_linear(e, x[:0], torch.zeros(4, dtype=torch.int32, device="cuda")).shape == (0, 45)


@pytest.mark.parametrize("counts", [[3, 4, 0], [70, 1, 200]])
def test_biases_in_their_own_type(counts):
    weights, e = experts_of(3, 45, 70, 0.5, torch.bfloat16)
    x, offsets = rand(sum(counts), 70, dtype=torch.bfloat16), offsets_of(counts)
    for t in (torch.float16, torch.bfloat16):
        bias = rand(3, 45, seed=1, dtype=t)
        check_forward(void.void_expert_linear(e, x, offsets, bias, 3), weights, x, counts, 0, bias, "silu")
        check_forward(void.void_expert_linear(e, x, offsets, bias.t().contiguous().t(), 3), weights, x, counts, 0, bias, "silu")


def test_weights_without_tiles():
    weights, e = experts_of(2, 64, 96, 0.0, torch.bfloat16)
    for counts in ([3, 4], [100, 80]):
        x, bias = rand(sum(counts), 96, dtype=torch.bfloat16), rand(2, 64)
        check_forward(void.void_expert_linear(e, x, offsets_of(counts), bias, 2), weights, x, counts, 0, bias, "gelu")


def test_edited_weights_are_packed_again():
    weights, e = experts_of(2, 64, 96, 0.5, torch.bfloat16)
    x, offsets = rand(200, 96, dtype=torch.bfloat16), offsets_of([120, 80])
    check_forward(void.void_expert_linear(e, x, offsets), weights, x, [120, 80], 0, None, "none")
    e.values.mul_(2)
    for w in weights:
        w.values.mul_(2)
    check_forward(void.void_expert_linear(e, x, offsets), weights, x, [120, 80], 0, None, "none")


# ------------------------------------------------------------------------------------------ training
def check_training(layer, weights, x, counts, first, g, y, grads, act):
    dtype = x.dtype
    bias = None if layer.bias is None else layer.bias.detach()
    check_forward(y, weights, x.detach(), counts, first, bias, act)
    at, tile = first, 0
    rest = torch.ones(x.shape[0], dtype=torch.bool)
    for e, c in enumerate(counts):
        w = weights[e]
        run = slice(at, at + c)
        mine = grads[1][tile:tile + w.n_blocks]
        if c:
            xd, ad, gd = x[run].detach().double(), w.to_dense().double(), g[run].double()
            z, _, ez, _ = layer64(xd, ad, None if bias is None else bias[e].double(), None, act, dtype)
            (dx, edx), (da, eda), (db, edb) = layer_grads64(gd, z, ez, xd, ad, act, dtype, dtype if bias is None else bias.dtype)
            within(grads[0][run], dx, edx)
            within(mine, tiles_of(da, w), tiles_of(eda, w))
            if bias is not None:
                within(grads[2][e], db, edb)
        else:
            assert not mine.any() and (bias is None or not grads[2][e].any())
        rest[run] = False
        at, tile = at + c, tile + w.n_blocks
    assert not grads[0][rest.cuda()].any()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("case", [c for c in CASES if c[0] <= 100 and c[1] < 2000], ids=lambda c: "%d-%d-%d" % c[:3])
def test_training(case, act, dtype):
    n, k, m, counts, before, behind = case
    weights, e = experts_of(n, m, k, 0.3, dtype)
    tokens = before + sum(counts) + behind
    x, g = rand(tokens, k, dtype=dtype).requires_grad_(True), rand(tokens, m, dtype=dtype, seed=3)
    layer = void.SparseExperts(e, activation=act)
    with torch.no_grad():
        layer.bias.copy_(rand(n, m, seed=1))
    y = layer(x, offsets_of(counts, before))
    grads = torch.autograd.grad(y, (x, layer.values, layer.bias), g)
    check_training(layer, weights, x, counts, before, g, y, grads, act)
    void.check_device_status()


def test_training_with_fp32_biases_and_without():
    weights, e = experts_of(3, 64, 96, 0.4, torch.bfloat16)
    counts = [130, 0, 70]
    x, g, offsets = rand(200, 96, dtype=torch.bfloat16).requires_grad_(True), rand(200, 64, dtype=torch.bfloat16), offsets_of(counts)
    layer = void.SparseExperts(e, activation="silu", dtype=torch.float32)
    y = layer(x, offsets)
    grads = torch.autograd.grad(y, (x, layer.values, layer.bias), g)
    assert grads[2].dtype == torch.float32
    check_training(layer, weights, x, counts, 0, g, y, grads, "silu")
    bare = void.SparseExperts(e, bias=False, activation="silu")
    again = torch.autograd.grad(bare(x, offsets), (x, bare.values), g)
    assert torch.equal(again[0], grads[0]) and torch.equal(again[1], grads[1])      # (the biases were zero)


@pytest.mark.parametrize("counts", [[70, 100, 30], [3, 7, 5]])
@pytest.mark.parametrize("act", ["none", "gelu"])
def test_gradients_of_a_run_take_nothing_from_its_neighbours(counts, act):
    weights, e = experts_of(3, 64, 96, 0.5, torch.bfloat16)
    tokens = sum(counts) + 40
    x, g = rand(tokens, 96, dtype=torch.bfloat16), rand(tokens, 64, dtype=torch.bfloat16, seed=3)
    layer, offsets = void.SparseExperts(e, activation=act), offsets_of(counts)

    def grads(xs, gs):
        xs = xs.clone().requires_grad_(True)
        return torch.autograd.grad(layer(xs, offsets), (xs, layer.values, layer.bias), gs)
    clean = grads(x, g)
    bad_x, bad_g = x.clone(), g.clone()
    middle = slice(counts[0], counts[0] + counts[1])
    bad_x[middle], bad_g[middle] = float("inf"), float("nan")
    bad_x[sum(counts):], bad_g[sum(counts):] = float("nan"), float("inf")
    dirty = grads(bad_x, bad_g)
    t = [0]
    for w in weights:
        t.append(t[-1] + w.n_blocks)
    for i, run in ((0, slice(0, counts[0])), (2, slice(counts[0] + counts[1], sum(counts)))):
        assert torch.equal(dirty[0][run], clean[0][run])
        assert torch.equal(dirty[1][t[i]:t[i + 1]], clean[1][t[i]:t[i + 1]])
        assert torch.equal(dirty[2][i], clean[2][i])
    assert not dirty[0][sum(counts):].any()


@pytest.mark.parametrize("want", [(0,), (1,), (2,), (0, 2)])
@pytest.mark.parametrize("act", ["none", "relu"])
def test_only_the_gradients_that_are_wanted(want, act):
    _, e = experts_of(2, 64, 96, 0.5, torch.float16)
    x, g, offsets = rand(150, 96, dtype=torch.float16).requires_grad_(True), rand(150, 64, dtype=torch.float16), offsets_of([100, 50])
    layer = void.SparseExperts(e, activation=act)
    args = [x, layer.values, layer.bias]
    full = torch.autograd.grad(layer(x, offsets), args, g)
    for t in args:
        t.requires_grad_(False)
    for i in want:
        args[i].requires_grad_(True)
    got = torch.autograd.grad(layer(x, offsets), [args[i] for i in want], g)
    assert all(torch.equal(p, full[i]) for p, i in zip(got, want))


def test_one_expert_is_a_linear_layer():
    w = weight(333, 515, 0.3, torch.bfloat16)
    x, g = rand(300, 515, dtype=torch.bfloat16).requires_grad_(True), rand(300, 333, dtype=torch.bfloat16)
    layer, experts = void.SparseLinear(515, 333, w, activation="gelu"), void.SparseExperts(void.stack_experts([w]), activation="gelu")
    y, z = layer(x), experts(x, offsets_of([300]))
    a = torch.autograd.grad(y, (x, layer.sparse_weight.values, layer.bias), g)
    b = torch.autograd.grad(z, (x, experts.values, experts.bias), g)
    # the same sums in the same order up to how many meet in one instruction: within the bounds of both
    check_training(experts, [w], x, [300], 0, g, z, b, "gelu")
    check_training(experts, [w], x, [300], 0, g, y, (a[0], a[1], a[2][None]), "gelu")


def test_graph_replayed_with_other_tokens_and_offsets_and_another_stream():
    dtype = torch.bfloat16
    weights, e = experts_of(4, 64, 96, 0.5, dtype)
    layer = void.SparseExperts(e, activation="silu")
    x, g, offsets = rand(260, 96, dtype=dtype).requires_grad_(True), rand(260, 64, dtype=dtype, seed=3), offsets_of([100, 0, 60, 90])
    leaves = (x, layer.values, layer.bias)

    def step():
        y = layer(x, offsets)
        return [y.detach()] + list(torch.autograd.grad(y, leaves, g))

    def serve():
        return void.void_expert_linear(e, x.detach(), offsets, None, 3)
    expected, served = step(), serve()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        on_side = step() + [serve()]
    side.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(on_side, expected + [served]))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step() + [serve()]
    counts = [0, 170, 5, 40]
    with torch.no_grad():
        x.copy_(rand(260, 96, dtype=dtype, seed=77))
        offsets.copy_(offsets_of(counts))
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(outs, step() + [serve()]))
    check_training(layer, weights, x, counts, 0, g, outs[0], outs[1:4], "silu")


def test_module_and_the_layers_of_a_block_together():
    dtype = torch.bfloat16
    ups, up = experts_of(4, 320, 96, 0.4, dtype)
    downs, down = experts_of(4, 96, 320, 0.4, dtype, seed=7)
    norm, first, second = void.VOIDLayerNorm(96, dtype=dtype), void.SparseExperts(up, activation="gelu"), void.SparseExperts(down)
    counts = [64, 3, 0, 90]
    x, offsets = rand(157, 96, dtype=dtype).requires_grad_(True), offsets_of(counts)
    y = x + second(first(norm(x), offsets), offsets)
    y.backward(torch.ones_like(y))
    params = [p for m in (norm, first, second) for p in m.parameters()]
    assert all(p.grad is not None and bool(p.grad.isfinite().all()) for p in params + [x])
    # inference over the same weights: the norm, both layers, stage by stage within their own bounds
    h = void.void_layer_norm(x.detach(), norm.weight.detach(), norm.bias.detach())
    mid = void.void_expert_linear(first.get_experts(), h, offsets, first.bias.detach(), 2)
    check_forward(mid, ups, h, counts, 0, first.bias.detach(), "gelu")
    out = void.void_expert_linear(second.get_experts(), mid, offsets, second.bias.detach())
    check_forward(out, downs, mid, counts, 0, second.bias.detach(), "none")
    assert set(first.state_dict()) == {"values", "bias", "block_rows", "block_cols"}


def test_refusals():
    _, e = experts_of(2, 64, 96, 0.5, torch.bfloat16)
    x, offsets = rand(10, 96, dtype=torch.bfloat16), offsets_of([4, 6])
    layer = void.SparseExperts(e)
    for call, text in ((lambda: void.void_expert_linear(e, x, offsets[:2]), "vector of 3"),
                       (lambda: void.void_expert_linear(e, x, offsets.float()), "int32 or int64"),
                       (lambda: void.void_expert_linear(e, x, offsets.cpu()), "no CPU path"),
                       (lambda: void.void_expert_linear(e, x.int(), offsets), "float32, float16 or bfloat16"),
                       (lambda: void.void_expert_linear(e, x, offsets, out=x.float()[:, :64]), "x's type"),
                       (lambda: void.void_expert_linear(e, x, offsets, out=torch.empty(10, 65, device="cuda", dtype=x.dtype)), "out must be"),
                       (lambda: layer(x, offsets[:2]), "vector of 3")):
        with pytest.raises(_lib.VoidB200Error, match=text):
            call()
    with pytest.raises(AssertionError, match="bias"):
        void.void_expert_linear(e, x, offsets, torch.zeros(2, 63, device="cuda"))
    with pytest.raises(AssertionError, match="Dimension"):
        layer(x[:, :95], offsets)
    y = layer(x.requires_grad_(True), offsets)
    with pytest.raises(NotImplementedError, match="second derivative"):
        torch.autograd.grad(y.sum(), x, create_graph=True)
    torch.autograd.grad(y.sum(), x)
    with pytest.raises(RuntimeError, match="second time|freed"):
        torch.autograd.grad(y.sum(), x)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n, k, m, density, counts, before, behind", [
    (4, 1024, 2000, 0.3, [700, 0, 1500, 331], 0, 0), (4, 1024, 2000, 0.3, [700, 0, 1500, 331], 5, 300), (3, 2048, 4096, 0.45, [900, 1, 400], 0, 77),
    (8, 515, 1104, 0.5, [600, 601, 0, 0, 1, 700, 129, 1000], 3, 1),
])
def test_groups_of_tile_rows(n, k, m, density, counts, before, behind, dtype):
    # (the first calls take the row kernel; from the fourth on a store for groups of each expert's tile rows is there)
    weights, e = experts_of(n, m, k, density, dtype)
    tokens = before + sum(counts) + behind
    x, bias, offsets = rand(tokens, k, dtype=dtype), rand(n, m, seed=1), offsets_of(counts, before)
    first = void.void_expert_linear(e, x, offsets, bias, 3)
    check_forward(first, weights, x, counts, before, bias, "silu")
    for _ in range(5):
        y = void.void_expert_linear(e, x, offsets, bias, 3)
        torch.cuda.synchronize()
    check_forward(y, weights, x, counts, before, bias, "silu")
    packed = next(iter(e.tensor._packed_fp_cache.values()))
    allowed, stores, done = _lib.native().packed_grouped(packed.native, None)
    assert allowed and (dtype == torch.float32 or (stores == 1 and done == 1))
    other = list(reversed(counts))
    y = void.void_expert_linear(e, x, offsets_of(other, before), bias.bfloat16(), 1)
    check_forward(y, weights, x, other, before, bias.bfloat16(), "relu")
    mine = rand(tokens, m, dtype=dtype, seed=8)
    was = mine.clone()
    void.void_expert_linear(e, x, offsets, None, 0, out=mine)
    check_forward(mine, weights, x, counts, before, None, "none", untouched=was)
    void.allow_group_stores(e.tensor, False)
    assert torch.equal(void.void_expert_linear(e, x, offsets, bias, 3), first)
    void.check_device_status()
