"""Dense 8-bit weights with scales of blocks, what needs no GPU: refusals of the operators and copies of the tensor."""
import copy
import io

import pytest
import torch

import void_b200 as void

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
