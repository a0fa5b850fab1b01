"""Layer norm on B200: what stands in front of a sparse layer in a transformer block.

The reference has no layers around its products; this is an extension.  Forward and backward are hand-written kernels
(csrc/norm.cu), statistics and sums over tokens are fp32, and the gradients do not depend on the order blocks ran in.
"""
from typing import Optional

import torch

from . import _lib


def void_layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None, eps: float = 1e-5,
                    out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """y = (x - mean) / sqrt(var + eps) * weight + bias over the last dimension of x [..., D] (float32, float16 or bfloat16), y in
    x's type.  weight and bias [D] are of x's type or float32, both of one; each may be left out.  Differentiable once in x, weight
    and bias.  ``out`` (contiguous; may be x itself, or share memory with an operand in another way) takes the result where nothing is
    differentiated."""
    if torch._C._are_functorch_transforms_active():
        raise RuntimeError("the layer norm cannot be used inside torch.func transforms (vmap, grad, jvp, ...)")
    _lib.require_cuda(x, weight, bias, out)
    return _lib.native().layer_norm(x, weight, bias, eps, out)


class VOIDLayerNorm(torch.nn.Module):
    """void_layer_norm as a module with a weight of ones and a bias of zeros (``bias=False``: none)."""

    def __init__(self, features: int, eps: float = 1e-5, bias: bool = True, dtype: Optional[torch.dtype] = None, device="cuda"):
        super().__init__()
        self.features, self.eps = features, eps
        self.weight = torch.nn.Parameter(torch.ones(features, dtype=dtype, device=device))
        if bias:
            self.bias = torch.nn.Parameter(torch.zeros(features, dtype=dtype, device=device))
        else:
            self.register_parameter("bias", None)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return void_layer_norm(x, self.weight, self.bias, self.eps)

    def extra_repr(self) -> str:
        return f"features={self.features}, eps={self.eps}, bias={self.bias is not None}"


__all__ = ["void_layer_norm", "VOIDLayerNorm"]
