"""Dense 8-bit weights with scales of blocks, what needs no GPU: refusals of the operators and copies of the tensor."""
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
