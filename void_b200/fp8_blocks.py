"""Dense e4m3 matrices with a scale for each block of 128 columns: weights of linear layers and of experts on B200.

The reference's FP8 tensors are 32x32 tiles with a scale each (void/fp8.py:438-570); this is an extension for dense weights, whose blocks are
128 x 128, and for tokens, whose blocks are one token's 128 features.  ops.void_linear and experts.void_expert_linear take them
(csrc/fp8_blocks.cu): products on the FP8 tensor cores, both scales applied to each block's fp32 sum.  Inference only, like the other
quantised products.
"""
from typing import Optional

import torch

from . import _lib

BLOCK = 128


def _rows_on_16_bytes(values: torch.Tensor) -> torch.Tensor:
    """The values themselves where their rows start on 16-byte boundaries, else a copy whose rows do."""
    cols = values.shape[-1]
    if values.data_ptr() % 16 == 0 and (cols <= 1 or values.stride(-1) == 1) and all(
            s % 16 == 0 and s >= cols for n, s in zip(values.shape[:-1], values.stride()[:-1]) if n > 1):
        return values
    copy = torch.empty(*values.shape[:-1], (cols + 15) // 16 * 16, dtype=values.dtype, device=values.device)[..., :cols]
    copy.view(torch.uint8).copy_(values.view(torch.uint8))
    return copy


class FP8BlockTensor:
    """A matrix [rows, cols], or the matrices of experts [experts, rows, cols], in float8_e4m3fn (``values``) with float32 ``scales``
    [..., ceil(rows / 128), ceil(cols / 128)] (weights) or [rows, ceil(cols / 128)] (tokens): the matrix stands for values * scale of their
    block.  ``values`` and ``scales`` are the tensors given (values with rows that do not start on 16-byte boundaries: a copy), and products
    read them as they are at the time of the call."""
    __slots__ = ("values", "scales", "block_rows", "shape", "n_experts", "_status")

    def __init__(self, values: torch.Tensor, scales: torch.Tensor):
        if values.dtype is not torch.float8_e4m3fn:
            raise _lib.VoidB200Error("an FP8BlockTensor holds float8_e4m3fn values, got %s" % values.dtype)
        if scales.dtype is not torch.float32:
            raise _lib.VoidB200Error("an FP8BlockTensor's scales are float32, got %s" % scales.dtype)
        if values.dim() not in (2, 3) or scales.dim() != values.dim() or 0 in values.shape:
            raise ValueError("an FP8BlockTensor is a matrix or a stack of matrices with scales of as many dimensions, none of them empty, got %s and %s"
                             % (tuple(values.shape), tuple(scales.shape)))
        if values.device != scales.device:
            raise _lib.VoidB200Error("values and scales are on different devices")
        rows, cols = values.shape[-2:]
        across, down = (cols + BLOCK - 1) // BLOCK, (rows + BLOCK - 1) // BLOCK
        if tuple(scales.shape) == (*values.shape[:-2], down, across):
            self.block_rows = BLOCK
        elif values.dim() == 2 and tuple(scales.shape) == (rows, across):
            self.block_rows = 1
        else:
            raise ValueError("scales of a %s matrix must be %s (or, of tokens, %s), got %s" % (
                tuple(values.shape), (*values.shape[:-2], down, across), (rows, across), tuple(scales.shape)))
        self.values, self.scales, self._status = _rows_on_16_bytes(values), scales, None
        self.shape = tuple(values.shape)                                       # (experts, rows, columns), or without the first
        self.n_experts: Optional[int] = self.shape[0] if len(self.shape) == 3 else None
        if values.is_cuda and not torch.cuda.is_current_stream_capturing():   # (made inside a capture, the device's status word would be cleared by its replays)
            _lib.status_word(values.device)

    def __reduce__(self):
        """Copies and files hold the fields; the status word is the device's."""
        return FP8BlockTensor, (self.values, self.scales)

    @property
    def device(self) -> torch.device:
        return self.values.device

    @property
    def memory_bytes(self) -> int:
        return self.values.numel() + 4 * self.scales.numel()

    def to(self, device) -> "FP8BlockTensor":
        return FP8BlockTensor(self.values.to(device), self.scales.to(device))

    def cuda(self) -> "FP8BlockTensor":
        return self.to("cuda")

    def dequantize(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        """The matrix it stands for, values * scale in float32 rounded to ``dtype``."""
        rows, cols = self.values.shape[-2:]
        scales = self.scales.repeat_interleave(BLOCK, -1)[..., :cols]
        if self.block_rows != 1:
            scales = scales.repeat_interleave(self.block_rows, -2)[..., :rows, :]
        return (self.values.float() * scales).to(dtype)

    def _product(self, x, offsets, bias, activation, out, out_dtype, residual) -> torch.Tensor:
        if _lib.transforms_active():
            _lib.no_transforms("a layer with 8-bit weights")
        values, x_scales = self.values, None
        if type(x) is FP8BlockTensor:
            x, x_scales = x.values, x.scales
        if not (values.is_cuda and x.is_cuda):
            _lib.require_cuda(values, x)
        status = self._status
        if status is None or status.get_device() != x.get_device():
            status = self._status = _lib.status_word(x.device)
        return _lib.native().fp8_linear(values, self.scales, x, x_scales, offsets, bias, activation, out, out_dtype, residual, status)

    def __repr__(self) -> str:
        return f"FP8BlockTensor(shape={self.shape}, block={(self.block_rows, BLOCK)}, device={self.values.device})"


def quantize_fp8_blocks(x: torch.Tensor, block_rows: int = BLOCK) -> FP8BlockTensor:
    """x [rows, cols] (float32, float16 or bfloat16) in e4m3 with a scale for each 128 x 128 block (weights; also of x [experts, rows, cols]), or with
    ``block_rows=1`` for each row's 128 columns (tokens, as void_linear and void_expert_linear take them).  A scale is the smallest
    power of two that keeps its block within 448, so that only the quotients are rounded, once; a block that holds an infinity or NaN gets a
    scale of NaN."""
    if _lib.transforms_active():
        _lib.no_transforms("the quantiser of blocks")
    if block_rows not in (1, BLOCK):
        raise ValueError("blocks have 1 or %d rows, got %s" % (BLOCK, block_rows))
    if x.dim() not in (2, 3) or (x.dim() == 3 and block_rows == 1) or 0 in x.shape:
        raise ValueError("quantize_fp8_blocks takes a matrix (or, of weights, a stack of them) that is not empty, got %s" % (tuple(x.shape),))
    _lib.require_cuda(x)
    return FP8BlockTensor(*_lib.native().quant_fp8_blocks(x, block_rows))


__all__ = ["FP8BlockTensor", "quantize_fp8_blocks"]
