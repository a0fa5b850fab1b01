"""Linear layers with dense 8-bit weights in scaled blocks on a B200: operands that change from call to call."""
import pytest
import torch

import void_b200 as void
from void_b200 import _lib
from test_fp8_blocks_gpu import TYPES, _check, _dense, _gen, _weights

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


# runs, rows behind them, M, K: few work items with eight blocks of k or more, which clusters share; of 24, 64 and more tokens an expert on average, empty runs
# (clusters with nothing to do), results in rows on 32 bytes and off them, plans by the product and (33 experts and more) by a launch of their own
SHARED = [([3, 0, 5, 1], 2, 130, 1024), ([10, 0, 20, 0, 7], 5, 128, 4096), ([0, 1, 0], 0, 257, 1030), ([60, 0, 40], 0, 256, 2048), ([64, 1, 33, 0], 9, 131, 1500),
          ([200, 0, 150, 0], 13, 304, 1500), ([130, 0, 257], 40, 255, 4096), ([0, 300], 1, 64, 3000), ([4] * 33, 3, 64, 1024), ([100] * 35, 0, 200, 1300),
          ([70, 2] * 18, 5, 129, 1100), ([0, 0, 0], 30, 128, 1024), ([0] * 40, 20, 128, 1024)]


@pytest.mark.parametrize("runs, spare, m, k", SHARED)
def test_experts_whose_blocks_are_shared(runs, spare, m, k):
    experts, n = len(runs), sum(runs) + spare
    parts = [_weights(m, k, e) for e in range(experts)]
    w = void.FP8BlockTensor(torch.stack([p.values.view(torch.uint8) for p in parts]).view(torch.float8_e4m3fn), torch.stack([p.scales for p in parts]))
    a = _dense(w)
    ends = torch.tensor([0] + runs).cumsum(0)
    used = sum(runs)
    for i, dtype in enumerate(TYPES):
        x = torch.randn(n, k, generator=_gen(5), device="cuda").to(dtype)
        x[used:] = float("nan")
        xd = _dense(void.quantize_fp8_blocks(x, 1))
        bias = torch.randn(experts, m, generator=_gen(6), device="cuda").to(dtype) if i != 2 else None
        act = (experts + i) % 4
        got = void.void_expert_linear(w, x, ends.to((torch.int32, torch.int64)[i % 2]).cuda(), bias, act)
        for e in range(experts):
            if runs[e]:
                _check(got[ends[e]:ends[e + 1]], xd[ends[e]:ends[e + 1]], a[e], None if bias is None else bias[e], act, None, dtype)
        assert (got[used:] == 0).all()
        outer = torch.full((n, m + 7), 5.0, dtype=dtype, device="cuda")     # (rows that lie anyhow)
        void.void_expert_linear(w, x, ends.cuda(), bias, act, out=outer[:, 3:m + 3])
        assert torch.equal(outer[:used, 3:m + 3], got[:used]) and (outer[used:] == 5).all() and (outer[:, :3] == 5).all() and (outer[:, m + 3:] == 5).all()
    void.check_device_status()


@pytest.mark.parametrize("n, m, k", [(40, 300, 1100), (8, 300, 5000), (200, 300, 700), (200, 300, 1100), (200, 301, 1100), (300, 2500, 700)])
def test_waits_that_run_out_are_reported(n, m, k):
    """The first stage of every ring is never filled, of both kernels, alone and in clusters: they give up after a tenth of a second and say so, and the next
    product is right."""
    import ctypes
    w, x = _weights(m, k, 1), void.quantize_fp8_blocks(torch.randn(n, k, generator=_gen(2), device="cuda"), 1)
    want = void.void_linear(w, x)
    out = torch.empty_like(want)
    status = _lib.status_word(x.device)
    a = _lib.Fp8Args(a=w.values.data_ptr(), lda=w.values.stride(0), a_scale=w.scales.data_ptr(), a_scale_row=w.scales.stride(0), a_scale_col=1,
                     x=x.values.data_ptr(), ldx=x.values.stride(0), x_scale=x.scales.data_ptr(), x_scale_row=x.scales.stride(0),
                     x_scale_col=x.scales.stride(1), out=out.data_ptr(), ldc=m, M=m, K=k, N=n, test_hooks=100 | 1 << 16, status=status.data_ptr())
    assert _lib.load().void_fp8_linear(ctypes.byref(a), None, _lib.stream_ptr(x.device)) == 0
    with pytest.raises(_lib.VoidB200Error, match="wait gave up"):
        void.check_device_status()
    assert torch.equal(void.void_linear(w, x), want)
    void.check_device_status()


def test_a_token_s_result_in_other_batches():
    """A token's result is the same in every batch for which the blocks of k are cut alike: here twelve of them, in threes (by three CTAs of a cluster)."""
    w = _weights(700, 1500, 1)
    x = torch.randn(600, 1500, generator=_gen(2), device="cuda")
    for most, cuts in ((600, ((0, 200), (100, 300), (129, 590))), (64, ((0, 40), (20, 60), (31, 64))), (32, ((0, 1), (5, 9), (17, 32)))):
        want = void.void_linear(w, x[:most])
        for lo, hi in cuts:
            assert torch.equal(void.void_linear(w, x[lo:hi]), want[lo:hi]), (most, lo, hi)


@pytest.mark.parametrize("dtype", TYPES)
def test_weights_of_experts_are_quantised_into_one_place(dtype):
    from torch.utils._python_dispatch import TorchDispatchMode

    class Calls(TorchDispatchMode):
        def __init__(self):
            super().__init__()
            self.names = set()

        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            self.names.add(func.overloadpacket._qualified_op_name)
            return func(*args, **(kwargs or {}))

    for experts, m, k in ((1, 1, 1), (3, 130, 200), (5, 128, 256), (2, 300, 1111)):
        x = (torch.randn(experts, m, k, generator=_gen(m), device="cuda") * torch.logspace(-2, 2, experts, device="cuda")[:, None, None]).to(dtype)
        for given in (x, x.transpose(1, 2).contiguous().transpose(1, 2), torch.empty(experts + 1, m, k + 3, dtype=dtype, device="cuda")[1:, :, 1:k + 1].copy_(x)):
            with Calls() as calls:
                got = void.quantize_fp8_blocks(given)
            if given is x:
                assert not calls.names & {"aten::copy_", "aten::stack", "aten::cat", "aten::clone"}, calls.names
            assert got.shape == (experts, m, k) and got.n_experts == experts and got.block_rows == 128
            for e in range(experts):
                want = void.quantize_fp8_blocks(x[e])
                assert torch.equal(got.scales[e], want.scales) and torch.equal(got.values[e].view(torch.uint8), want.values.view(torch.uint8))
    with pytest.raises(ValueError):
        void.quantize_fp8_blocks(x, 1)


@pytest.mark.parametrize("chunk", [32, 64, 128])
@pytest.mark.parametrize("runs, spare, m, k", [([17, 0, 70, 1], 3, 130, 500), ([130, 33], 0, 256, 1100), ([0, 65, 64, 0, 2], 5, 300, 2048)])
def test_experts_by_chunks_of_any_length(runs, spare, m, k, chunk):
    """What the entry point takes: chunks of 32, 64 and 128 tokens, whatever the experts have on average."""
    import ctypes
    experts, n, used = len(runs), sum(runs) + spare, sum(runs)
    parts = [_weights(m, k, e) for e in range(experts)]
    w = void.FP8BlockTensor(torch.stack([p.values.view(torch.uint8) for p in parts]).view(torch.float8_e4m3fn), torch.stack([p.scales for p in parts]))
    x = void.quantize_fp8_blocks(torch.randn(n, k, generator=_gen(2), device="cuda"), 1)
    bias = torch.randn(experts, m, generator=_gen(3), device="cuda")
    ends = torch.tensor([0] + runs).cumsum(0)
    offsets = ends.cuda()
    out = torch.full((n, m), 5.0, device="cuda")
    status = _lib.status_word(x.device)
    a = _lib.Fp8Args(a=w.values.data_ptr(), lda=w.values.stride(1), expert_stride=w.values.stride(0), a_scale=w.scales.data_ptr(), a_scale_row=w.scales.stride(1),
                     a_scale_col=1, a_scale_expert=w.scales.stride(0), x=x.values.data_ptr(), ldx=x.values.stride(0), x_scale=x.scales.data_ptr(),
                     x_scale_row=x.scales.stride(0), x_scale_col=x.scales.stride(1), bias=bias.data_ptr(), out=out.data_ptr(), ldc=m, M=m, K=k, N=n,
                     status=status.data_ptr())
    plan = _lib.Experts(plan=offsets.data_ptr(), n_experts=experts, chunk=chunk, offset_bytes=8)
    assert _lib.load().void_fp8_linear(ctypes.byref(a), ctypes.byref(plan), _lib.stream_ptr(x.device)) == 0
    void.check_device_status()
    xd, wd = _dense(x), _dense(w)
    for e in range(experts):
        if runs[e]:
            _check(out[ends[e]:ends[e + 1]], xd[ends[e]:ends[e + 1]], wd[e], bias[e], 0, None, torch.float32)
    assert (out[used:] == 5).all()


def test_the_status_word_is_not_made_by_a_capture():
    """A process whose first launch is a captured product: the word that kernels report in is there before, and no replay clears what is reported."""
    import os
    import subprocess
    import sys
    code = """
import torch, void_b200 as void
from void_b200 import _lib
w = void.FP8BlockTensor(torch.ones(256, 256, device="cuda").to(torch.float8_e4m3fn), torch.ones(2, 2, device="cuda"))
x = torch.ones(4, 256, device="cuda")
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    y = void.void_linear(w, x)
void.check_device_status()
graph.replay()
assert (y == 256).all()
_lib.status_word("cuda:0").fill_(1)
graph.replay()
try:
    void.check_device_status()
except _lib.VoidB200Error:
    print("reported")
"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    run = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=300)
    assert run.returncode == 0 and run.stdout.strip() == "reported", (run.stdout, run.stderr[-2000:])


@pytest.mark.parametrize("experts, m", [(3, 128), (37, 512), (149, 100)])
@pytest.mark.parametrize("each", [16, 24, 25, 48, 49, 65])
def test_experts_on_either_side_of_the_rule(experts, m, each):
    """Tokens an expert has on average, and matrices, around what decides between items of 32 and of 128 tokens; one expert has the tokens of three."""
    k, n = 200, experts * each
    counts = [each] * experts
    counts[0] += 2 * each
    counts[1] -= each
    counts[2] -= each
    w = void.quantize_fp8_blocks(torch.randn(experts, m, k, generator=_gen(1), device="cuda"))
    x = torch.randn(n, k, generator=_gen(2), device="cuda")
    ends = torch.tensor([0] + counts).cumsum(0)
    got = void.void_expert_linear(w, x, ends.cuda(), None, 2)
    xd, a = _dense(void.quantize_fp8_blocks(x, 1)), _dense(w)
    for e in range(experts):
        if counts[e]:
            _check(got[ends[e]:ends[e + 1]], xd[ends[e]:ends[e + 1]], a[e], None, 2, None, torch.float32)
    void.check_device_status()
