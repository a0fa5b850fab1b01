"""Dense 8-bit weights with scales of blocks, what needs no GPU: refusals of the operators and copies of the tensor."""
import copy
import io

import pytest
import torch

import void_b200 as void
from void_b200 import _lib
from test_fp8_blocks_cpu import ALIGN, TOO_LARGE, _linear

E4M3 = torch.float8_e4m3fn
WEIGHT = void.FP8BlockTensor(torch.ones(256, 256).to(E4M3), torch.ones(2, 2))
EXPERTS = void.FP8BlockTensor(torch.ones(2, 256, 256).to(E4M3), torch.ones(2, 2, 2))
OFFSETS = torch.tensor([0, 2, 4])


@pytest.mark.parametrize("call", [
    lambda x: void.void_linear(WEIGHT, x), lambda x: void.void_linear(WEIGHT, torch.ones(4, 256), residual=x), lambda x: void.void_expert_linear(EXPERTS, x, OFFSETS),
    lambda x: void.quantize_fp8_blocks(x, 1).scales, lambda x: void.quantize_fp8_blocks(x).scales, lambda x: void.sort_by_expert((x > 0).int(), 2).offsets],
    ids=["linear", "residual", "experts", "quantise tokens", "quantise weights", "sort"])
def test_transforms_are_refused(call):
    x = torch.ones(4, 256)
    for transform in (lambda: torch.func.vmap(call)(x[None]), lambda: torch.func.jvp(call, (x,), (x,)), lambda: torch.func.grad(lambda t: call(t).float().sum())(x)):
        with pytest.raises(RuntimeError, match="torch.func"):
            transform()


def test_copies_hold_the_fields_alone():
    """What a product keeps with a tensor (the device's status word) stays behind: a copy of the word would be one that nobody looks at."""
    w = void.FP8BlockTensor(torch.randn(200, 130).to(E4M3), torch.randn(2, 2))
    w._status = torch.zeros(1, dtype=torch.int32)
    file = io.BytesIO()   # (torch's own way: pickle by itself does not bring 8-bit tensors back)
    torch.save(w, file)
    file.seek(0)
    for copied in (copy.copy(w), copy.deepcopy(w), torch.load(file, weights_only=False)):
        assert copied._status is None and (copied.shape, copied.block_rows, copied.n_experts) == ((200, 130), 128, None)
        assert torch.equal(copied.values.view(torch.uint8), w.values.view(torch.uint8)) and torch.equal(copied.scales, w.scales)
        assert copied.values.stride() == (144, 1)
    assert copy.copy(w).values is w.values


def test_addresses_that_hold_no_element_are_refused():
    for bad in (dict(a_scale=4098), dict(x_scale=4098), dict(status=4098), dict(bias=4098), dict(bias=4097, bias_elem=2), dict(out=4098), dict(out=4097, out_elem=1),
                dict(residual=4098, ldr=64), dict(residual=4097, ldr=64, residual_elem=2)):
        assert _linear(**bad) == ALIGN, bad
    for bad in (dict(x=4098, elem=0), dict(x=4097, elem=1), dict(scales=4098, elem=2)):
        v = dict(dict(x=4096, elem=0, scales=4096), **bad)
        assert _lib.load().void_quant_fp8_blocks(v["x"], v["elem"], 100, 4, 100, 1, 4096, 112, v["scales"], 1, 4, None) == ALIGN, bad


def test_sizes_whose_ends_are_no_numbers_are_refused():
    for bad in (dict(M=2 ** 31 - 1, ldc=2 ** 31), dict(M=2 ** 31 - 255, ldc=2 ** 31), dict(N=2 ** 30 + 1), dict(N=2 ** 31 - 1)):
        assert _linear(**bad) == TOO_LARGE, bad
