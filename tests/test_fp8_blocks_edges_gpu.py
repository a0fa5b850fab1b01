"""Linear layers with dense 8-bit weights in scaled blocks on a B200: operands that change from call to call."""
import pytest
import torch

import void_b200 as void
from void_b200 import _lib
from test_fp8_blocks_gpu import _gen, _weights

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("experts, n", [(6, 90), (6, 700), (40, 90), (40, 3000)])
def test_runs_weights_and_biases_written_just_before_by_a_few_blocks(experts, n):
    """Every call has other runs, scales, biases and tokens, written by kernels of a few blocks right before it: nothing that a multiprocessor read in the
    call before may be used again, an old run least of all."""
    m, k = 130, 200
    given = []
    for s in range(5):
        w = [_weights(m, k, 10 * s + e) for e in range(experts)]
        cuts = torch.randint(0, n + 1, (experts - 1,), generator=_gen(s), device="cuda").sort().values
        given.append((torch.stack([p.values.view(torch.uint8) for p in w]), torch.stack([p.scales for p in w]),
                      torch.cat([cuts.new_zeros(1), cuts, cuts.new_full((1,), n)]), torch.randn(experts, m, generator=_gen(20 + s), device="cuda"),
                      torch.randn(n, k, generator=_gen(30 + s), device="cuda")))
    want = [void.void_expert_linear(void.FP8BlockTensor(v.view(torch.float8_e4m3fn), s), x, o, b, 3) for v, s, o, b, x in given]
    values, scales, offsets, bias, x = (t.clone() for t in given[0])
    w = void.FP8BlockTensor(values.view(torch.float8_e4m3fn), scales)
    got = []
    for i in range(40):
        for to, new in zip((w.values.view(torch.uint8), w.scales, x, bias, offsets), (given[i % 5][j] for j in (0, 1, 4, 3, 2))):
            to.copy_(new)
        got.append(void.void_expert_linear(w, x, offsets, bias, 3))
    for i, y in enumerate(got):
        assert torch.equal(y, want[i % 5]), i
    void.check_device_status()


@pytest.mark.parametrize("n", [8, 50, 200])
def test_residuals_and_biases_written_just_before_by_a_few_blocks(n):
    m, k = 130, 1200
    w = _weights(m, k, 1)
    given = [(torch.randn(n, k, generator=_gen(s), device="cuda"), torch.randn(m, generator=_gen(10 + s), device="cuda"),
              torch.randn(n, m, generator=_gen(20 + s), device="cuda")) for s in range(5)]
    want = [void.void_linear(w, x, b, residual=r) for x, b, r in given]
    x, bias, residual = (t.clone() for t in given[0])
    got = []
    for i in range(40):
        for to, new in zip((x, bias, residual), given[i % 5]):
            to.copy_(new)
        got.append(void.void_linear(w, x, bias, residual=residual))
    for i, y in enumerate(got):
        assert torch.equal(y, want[i % 5]), i


def test_tangents_are_refused():
    import torch.autograd.forward_ad as fwd
    w, experts = _weights(256, 256, 1), void.quantize_fp8_blocks(torch.randn(2, 256, 256, generator=_gen(1), device="cuda"))
    x, bias, offsets = torch.randn(4, 256, device="cuda"), torch.randn(256, device="cuda"), torch.tensor([0, 1, 4], device="cuda")
    quantised = void.quantize_fp8_blocks(x, 1)
    with fwd.dual_level():
        x_dual, bias_dual, biases = fwd.make_dual(x, x), fwd.make_dual(bias, bias), fwd.make_dual(bias.expand(2, 256).contiguous(), bias.expand(2, 256).contiguous())
        scales = [fwd.make_dual(t.scales, torch.ones_like(t.scales)) for t in (w, quantised)]
        for call in (lambda: void.void_linear(w, x_dual), lambda: void.void_linear(w, x, bias_dual), lambda: void.void_linear(w, quantised, residual=x_dual),
                     lambda: void.void_linear(void.FP8BlockTensor(w.values, scales[0]), x), lambda: void.void_linear(w, void.FP8BlockTensor(quantised.values, scales[1])),
                     lambda: void.void_expert_linear(experts, x_dual, offsets), lambda: void.void_expert_linear(experts, x, offsets, biases),
                     lambda: void.quantize_fp8_blocks(x_dual), lambda: void.quantize_fp8_blocks(x_dual, 1),
                     lambda: void.quantize_fp8_blocks(x_dual.expand(2, 4, 256))):
            with pytest.raises(NotImplementedError, match="tangent"):
                call()
    assert void.void_linear(w, x, bias).shape == (4, 256)


def test_too_many_columns_are_refused():
    for cols, dtype in ((16776961, torch.bfloat16), (33553924, torch.float32), (67107848, torch.float16)):   # (odd rows; rows in whole 16-byte pieces)
        with pytest.raises(_lib.VoidB200Error, match="documented maximum"):
            void.quantize_fp8_blocks(torch.empty(1, cols, dtype=dtype, device="cuda"), 1)
    x = torch.ones(1, 16776959, dtype=torch.bfloat16, device="cuda")
    q = void.quantize_fp8_blocks(x, 1)
    assert (q.values.float() * 2.0 ** -8 == 1).all() and (q.scales == 2.0 ** -8).all()


def test_the_status_word_is_that_of_the_device():
    """Values that were replaced by some of another device (here: of the host first) take their status word with them."""
    w, x = _weights(256, 256, 1), torch.randn(4, 256, generator=_gen(1), device="cuda")
    want = void.void_linear(w, x)
    w._status = torch.zeros(1, dtype=torch.int32)
    assert torch.equal(void.void_linear(w, x), want) and w._status is _lib.status_word(x.device)
