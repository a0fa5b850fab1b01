"""Linear layers, layers of experts and layer norm where an operand is at an edge: biases in 16 bits on a transposed copy, sums that
a bias cancels, results that share memory with an operand, rows longer than a block's registers."""
import pytest
import torch

import void_b200 as void
from test_experts_gpu import offsets_of
from test_linear_cpu import within
from test_linear_gpu import feed_forward64, rand, weight

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
