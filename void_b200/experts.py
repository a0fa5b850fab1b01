"""Linear layers of experts on B200: tokens sorted by expert, every run of tokens multiplied with its expert's VOID weight.

The reference has no such layer; this is an extension next to its linear layers (ops.void_linear, autograd.SparseLinear).  The
weights of all experts are one list of tiles and one packed store; a run may have any number of tokens, none included, and the
offsets stay on the device (csrc/experts.cu).
"""
from dataclasses import dataclass
from typing import Optional, Sequence, Tuple

import torch

from . import _lib
from .autograd import _require_operands, tile_grad_items
from .format import Derived, VOIDTensor, build_tile_index
from .fusion import layer_activation
from .ops import _KIND_DTYPE, packed_fp, product_kind


@dataclass
class VOIDExperts(Derived):
    """The weights [out, in] of experts, one VOIDTensor whose tile rows are theirs one expert after the other."""
    tensor: VOIDTensor          # shape (n_experts * padded rows, in)
    n_experts: int
    shape: Tuple[int, int]      # of one expert's weight

    @property
    def tile_rows(self) -> int:
        """Tile rows of one expert."""
        return (self.shape[0] + 31) // 32

    @property
    def values(self) -> torch.Tensor:
        return self.tensor.values

    @property
    def dtype(self) -> torch.dtype:
        return self.tensor.dtype

    @property
    def device(self) -> torch.device:
        return self.tensor.values.device

    def to(self, device) -> "VOIDExperts":
        return VOIDExperts(self.tensor.to(device), self.n_experts, self.shape)

    def to_dtype(self, dtype: torch.dtype) -> "VOIDExperts":
        return VOIDExperts(self.tensor.to_dtype(dtype), self.n_experts, self.shape)


def rows_by_length(row_ptr: torch.Tensor, n_experts: int) -> torch.Tensor:
    """Tile rows of every expert by falling tile count (int32 [n_experts * tile rows], each within its expert)."""
    counts = (row_ptr[1:] - row_ptr[:-1]).view(n_experts, -1)
    return counts.argsort(dim=1, descending=True, stable=True).to(torch.int32).flatten().contiguous()


def _row_order(packed, n_experts: int) -> torch.Tensor:
    """rows_by_length of a packed store, kept with it: where a captured graph reads the store, both stay."""
    kept = packed.__dict__.setdefault("_expert_orders", {})
    order = kept.get(n_experts)
    if order is None:
        dev = packed.row_ptr.device
        with torch.cuda.device(dev):
            order = rows_by_length(packed.row_ptr, n_experts)
            if packed.stable and not torch.cuda.is_current_stream_capturing():
                torch.cuda.current_stream(dev).synchronize()     # (other streams may read it from now on)
                kept[n_experts] = order
    return order


def stack_experts(weights: Sequence[VOIDTensor]) -> VOIDExperts:
    """The weights of experts, VOIDTensors of one shape, type and device, as one VOIDExperts (tiles in the order given)."""
    weights = list(weights)
    if not weights:
        raise ValueError("stack_experts needs at least one weight")
    first = weights[0]
    for w in weights:
        if not isinstance(w, VOIDTensor):
            raise TypeError("stack_experts takes VOIDTensors, got %s" % type(w).__name__)
        if tuple(w.tile_size) != (32, 32):
            raise NotImplementedError("void_b200 kernels are built for 32x32 tiles, got tile_size=%s" % (w.tile_size,))
        if tuple(w.shape) != tuple(first.shape) or w.values.dtype != first.values.dtype or w.values.device != first.values.device:
            raise ValueError("stack_experts takes weights of one shape, type and device, got %s %s on %s and %s %s on %s" % (
                tuple(first.shape), first.values.dtype, first.values.device, tuple(w.shape), w.values.dtype, w.values.device))
    rows, cols = (first.shape[0] + 31) // 32, first.shape[1]
    block_rows = torch.cat([w.block_rows for w in weights]).to(torch.int32)
    if block_rows.numel():
        low, high = torch.stack(block_rows.aminmax()).tolist()
        if low < 0 or high >= rows:                        # (they would be another expert's)
            raise ValueError("invalid VOID tile list: block rows outside the block grid of %s" % (tuple(first.shape),))
    counts = torch.tensor([w.block_rows.numel() for w in weights], device=block_rows.device)
    block_rows += torch.repeat_interleave(torch.arange(len(weights), dtype=torch.int32, device=block_rows.device) * rows, counts,
                                          output_size=block_rows.numel())
    tensor = VOIDTensor(values=torch.cat([w.values for w in weights]), block_rows=block_rows,
                        block_cols=torch.cat([w.block_cols.to(torch.int32) for w in weights]),
                        morton_codes=torch.empty(0, dtype=torch.int64, device=first.values.device), shape=(len(weights) * rows * 32, cols),
                        tile_size=(32, 32), nnz_original=sum(w.nnz_original for w in weights), n_blocks=sum(w.n_blocks for w in weights),
                        density=sum(w.density for w in weights) / len(weights), dtype=first.values.dtype)
    return VOIDExperts(tensor, len(weights), tuple(first.shape))


def void_expert_linear(experts: VOIDExperts, x: torch.Tensor, offsets: torch.Tensor, bias: Optional[torch.Tensor] = None, activation: int = 0,
                       out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """y[t] = act(x[t] @ A_e^T + bias[e]) for the tokens offsets[e] <= t < offsets[e + 1] of every expert e; x [tokens, in] in
    float32 (multiplied as TF32), float16 or bfloat16, sorted by expert, y [tokens, out] in x's type.  ``offsets`` is int32 or int64
    [n_experts + 1] on x's device and is not read by the host: a captured call may be replayed with others.  ``bias`` is
    [n_experts, out].  Rows in no run (before the first offset, behind the last) are zeros; with ``out`` (which must have no memory in common with an operand)
    they are left as they are.
    Offsets that fall or lie outside the batch are taken as empty runs and reported by check_device_status.  Inference form of
    SparseExperts: nothing is differentiated."""
    if not isinstance(experts, VOIDExperts):
        raise TypeError("void_expert_linear takes a VOIDExperts (stack_experts), got %s" % type(experts).__name__)
    assert x.dim() == 2 and x.shape[1] == experts.shape[1], f"Dimension mismatch: the experts are {experts.shape}, x is {tuple(x.shape)}"
    tensor = experts.tensor
    _lib.require_cuda(tensor.values, x, offsets, bias, out)
    M, n_experts = experts.shape[0], experts.n_experts
    if bias is not None:
        assert bias.shape == (n_experts, M), f"bias must have shape {(n_experts, M)}, got {tuple(bias.shape)}"
    dtype = x.dtype
    if dtype not in _lib.OUT_DTYPE_CODE:
        raise _lib.VoidB200Error("void_expert_linear: x must be float32, float16 or bfloat16, got %s" % dtype)
    if out is not None and out.dtype != dtype:
        raise _lib.VoidB200Error("void_expert_linear: out must be of x's type, got %s" % out.dtype)
    if out is not None and tuple(out.shape) != (x.shape[0], M):
        raise _lib.VoidB200Error("void_expert_linear: out must be a row-major [%d, %d] tensor, got %s" % (x.shape[0], M, tuple(out.shape)))
    kind = product_kind(tensor, x)
    packed = packed_fp(tensor, kind)
    order = _row_order(packed, n_experts)
    if dtype is not _KIND_DTYPE[kind]:
        y = _lib.native().expert_linear(packed.native, n_experts, M, x.to(_KIND_DTYPE[kind]), offsets, bias, activation, None, order).to(dtype)
        return y if out is None else _copy_runs(out, y, offsets)
    return _lib.native().expert_linear(packed.native, n_experts, M, x, offsets, bias, activation, out, order)


def _copy_runs(out: torch.Tensor, y: torch.Tensor, offsets: torch.Tensor) -> torch.Tensor:
    """``out`` with the rows of all runs taken from ``y``."""
    at = torch.arange(y.shape[0], device=y.device)
    last = offsets.cummax(0).values[-1]
    return out.copy_(torch.where(((at >= offsets[0]) & (at < last))[:, None], y, out))


_EXPERT_STRUCTURE = {}
_EXPERT_STRUCTURE_MAX = 64


def _expert_structure(block_rows, block_cols, n_experts, shape, n_blocks):
    """The index arrays of all experts' tiles, of their weights and of the weights' transposes, as autograd._structure has them (built in 0.6 ms for
    13000 tiles, 1.3 for 26000; kept for the last 64 tile lists, whether their layers live or not)."""
    key = (block_rows.data_ptr(), block_cols.data_ptr(), block_rows._version, block_cols._version, shape[0], shape[1], n_experts, n_blocks,
           block_rows.is_contiguous() or block_rows.stride(), block_cols.is_contiguous() or block_cols.stride())
    hit = _EXPERT_STRUCTURE.get(key)
    if hit is None:
        _lib.require_cuda(block_rows, block_cols)
        nbr, nbc = (shape[0] + 31) // 32, (shape[1] + 31) // 32
        rows, cols = block_rows.to(torch.int32), block_cols.to(torch.int32)
        row_ptr, block_indices = build_tile_index(rows, cols, n_experts * nbr, nbc)
        expert = torch.div(rows, nbr, rounding_mode="floor")
        inner = rows - expert * nbr
        row_ptr_t, block_indices_t = build_tile_index(expert * nbc + cols, inner, n_experts * nbc, nbr)
        st = _lib.native().structure(row_ptr, block_indices, cols[block_indices.long()].contiguous(), row_ptr_t, block_indices_t,
                                     inner[block_indices_t.long()].contiguous(), tile_grad_items(row_ptr), _lib.status_word(block_rows.device),
                                     shape[0], shape[1], n_blocks, rows_by_length(row_ptr, n_experts), rows_by_length(row_ptr_t, n_experts),
                                     n_experts)
        torch.cuda.current_stream(block_rows.device).synchronize()    # (other streams may read the arrays from now on)
        hit = (st, block_rows, block_cols)     # keeps the keys alive
        if len(_EXPERT_STRUCTURE) >= _EXPERT_STRUCTURE_MAX:
            for old in list(_EXPERT_STRUCTURE):
                if not _lib.native().structure_captured(_EXPERT_STRUCTURE[old][0]):
                    _EXPERT_STRUCTURE.pop(old, None)
                    break
        _EXPERT_STRUCTURE[key] = hit
    return hit[0]


class SparseExperts(torch.nn.Module):
    """A linear layer of experts with VOID weights, y[t] = act(x[t] W_e^T + b_e) for the tokens offsets[e] <= t < offsets[e + 1], zeros
    for tokens in no run.  Differentiable in x, the stored tiles and the biases, once; experts without tokens get zero gradients.
    Parameters: ``values`` [tiles, 32, 32], expert after expert, and ``bias`` [n_experts, out]."""

    def __init__(self, experts: VOIDExperts, bias: bool = True, activation: str = "none", dtype: Optional[torch.dtype] = None):
        super().__init__()
        self.n_experts, self.shape, self.activation = experts.n_experts, experts.shape, activation
        self.out_features, self.in_features = experts.shape
        self._activation = layer_activation(activation)
        self.values = torch.nn.Parameter(experts.values.clone())
        self.register_buffer("block_rows", experts.tensor.block_rows)
        self.register_buffer("block_cols", experts.tensor.block_cols)
        self.n_blocks = experts.tensor.n_blocks
        if bias:
            self.bias = torch.nn.Parameter(torch.zeros(self.n_experts, self.out_features, dtype=dtype or experts.dtype, device=experts.device))
        else:
            self.register_parameter("bias", None)

    def forward(self, x: torch.Tensor, offsets: torch.Tensor) -> torch.Tensor:
        _require_operands(self.values, (32, 32), x)
        assert x.dim() == 2 and x.shape[1] == self.in_features, f"Dimension mismatch: the experts are {self.shape}, x is {tuple(x.shape)}"
        _lib.require_cuda(offsets)
        st = _expert_structure(self.block_rows, self.block_cols, self.n_experts, self.shape, self.n_blocks)
        return _lib.native().expert_values_product(st, self.values, x, offsets, self.bias, self._activation)

    def get_experts(self) -> VOIDExperts:
        """The weights for void_expert_linear: they share memory with the parameter and follow its changes."""
        rows = (self.out_features + 31) // 32
        tensor = VOIDTensor(values=self.values.detach(), block_rows=self.block_rows, block_cols=self.block_cols,
                            morton_codes=torch.empty(0, dtype=torch.int64, device=self.values.device),
                            shape=(self.n_experts * rows * 32, self.in_features), tile_size=(32, 32), nnz_original=0, n_blocks=self.n_blocks,
                            density=0.0, dtype=self.values.dtype)
        return VOIDExperts(tensor, self.n_experts, self.shape)

    def extra_repr(self) -> str:
        return (f"n_experts={self.n_experts}, in_features={self.in_features}, out_features={self.out_features}, "
                f"activation={self.activation}, bias={self.bias is not None}")


__all__ = ["VOIDExperts", "stack_experts", "void_expert_linear", "SparseExperts"]
