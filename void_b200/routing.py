"""Tokens on their way to experts and back on B200: the router that chooses a token's experts, the tokens brought into runs by expert as
layers of experts read them (experts.void_expert_linear, SparseExperts), and the experts' rows brought back with their weights.

The reference has no such operators; this is an extension next to its linear layers.  Forward and backward are hand-written kernels
(csrc/route.cu); the offsets stay on the device, sums are fp32 and taken in the order of a token's choices, and no result depends on the
order in which blocks ran.
"""
from typing import Optional, Tuple

import torch

from . import _lib


class ExpertRoutes:
    """Where tokens went that were sorted by expert: ``offsets`` (int32 [n_experts + 1], the ends of the experts' runs) and ``position`` (int32
    [tokens, top_k], the row of every choice, -1 for a dropped one).  Made by sort_by_expert and void_dispatch; not to be written to."""
    __slots__ = ("offsets", "position", "n_experts", "_versions")

    def __init__(self, offsets: torch.Tensor, position: torch.Tensor, n_experts: int):
        self.offsets, self.position, self.n_experts = offsets, position, n_experts
        self._versions = None if position.is_inference() else offsets._version + position._version

    def check(self):
        """Raises where the routes were written to since they were made: rows would be left that no choice has."""
        if self._versions is not None and self._versions != self.offsets._version + self.position._version:   # (they only grow)
            raise _lib.VoidB200Error("the routes have been written to since the tokens were sorted: drop choices (-1) before they are sorted")

    def __reduce__(self):
        """Copies and files hold the routes; their tensors count what is written to them anew."""
        self.check()
        return ExpertRoutes, (self.offsets, self.position, self.n_experts)

    @property
    def n_tokens(self) -> int:
        return self.position.shape[0]

    @property
    def top_k(self) -> int:
        return self.position.shape[1]

    def __repr__(self) -> str:
        return f"ExpertRoutes(n_tokens={self.n_tokens}, top_k={self.top_k}, n_experts={self.n_experts})"


def void_route(scores: torch.Tensor, top_k: int, normalize: bool = True) -> Tuple[torch.Tensor, torch.Tensor]:
    """The ``top_k`` (at most 32) experts of each token with the largest scores [tokens, experts] (float32, float16 or bfloat16, up to 1024
    experts) as int32 [tokens, top_k], largest first, ties to the lowest index, and their weights, float32 [tokens, top_k]: the softmax of the
    scores over the chosen experts, or with ``normalize=False`` over all.  A score of -inf is never chosen: where fewer than ``top_k``
    others are left, the expert is -1 (which void_dispatch drops) and the weight 0.  NaN counts as the largest and makes a token's weights NaN.
    Differentiable once in the scores."""
    if _lib.transforms_active():
        _lib.no_transforms("the router")
    if not scores.is_cuda:
        _lib.require_cuda(scores)
    return _lib.native().route(scores, top_k, normalize)


def sort_by_expert(experts: torch.Tensor, n_experts: int) -> ExpertRoutes:
    """Sorts the choices ``experts`` (int32 or int64 [tokens, top_k]) by expert, in the order of the tokens within an expert.  A choice
    outside [0, n_experts) is dropped: it belongs to no run.  At most 1024 experts; nothing is read by the host, so a captured call may be
    replayed with other choices."""
    if _lib.transforms_active():
        _lib.no_transforms("the sort by expert")
    _lib.require_cuda(experts)
    return ExpertRoutes(*_lib.native().sort_by_expert(experts, n_experts), n_experts)


def void_dispatch(x: torch.Tensor, experts: torch.Tensor, n_experts: int, out: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, ExpertRoutes]:
    """Tokens x [tokens, features] (float32, float16 or bfloat16) copied into the run of each of their experts: rows [tokens * top_k, features]
    sorted by expert, as void_expert_linear and SparseExperts take them, and the routes (sort_by_expert).  Rows behind the last run, one for
    every dropped choice, are zeros; with ``out`` (row-major) they are left as they are.  Differentiable once in x."""
    if _lib.transforms_active():
        _lib.no_transforms("the dispatch of tokens")
    if not (x.is_cuda and experts.is_cuda):
        _lib.require_cuda(x, experts)
    rows, offsets, position = _lib.native().dispatch(x, experts, n_experts, out)
    return rows, ExpertRoutes(offsets, position, n_experts)


def void_combine(rows: torch.Tensor, routes: ExpertRoutes, weights: Optional[torch.Tensor] = None, residual: Optional[torch.Tensor] = None,
                 out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """y[t] = residual[t] + sum_j weights[t, j] rows[position[t, j]]: the experts' rows [tokens * top_k, features] brought back to their tokens,
    in rows' type.  ``weights`` [tokens, top_k] and ``residual`` [tokens, features] are float32, float16 or bfloat16; without weights the rows
    are added.  A dropped choice adds nothing, whatever its weight.  Differentiable once in rows, weights and residual.  ``out`` (row-major;
    may be the residual, or share memory with an operand in another way) takes the result where nothing is differentiated."""
    if _lib.transforms_active():
        _lib.no_transforms("the combination of experts' rows")
    if not isinstance(routes, ExpertRoutes):
        raise TypeError("void_combine takes ExpertRoutes (sort_by_expert, void_dispatch), got %s" % type(routes).__name__)
    if not rows.is_cuda:
        _lib.require_cuda(rows)
    routes.check()
    return _lib.native().combine(rows, routes.position, routes.offsets, weights, residual, out)


__all__ = ["ExpertRoutes", "void_route", "sort_by_expert", "void_dispatch", "void_combine"]
