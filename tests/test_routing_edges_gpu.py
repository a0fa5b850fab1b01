"""Tokens to experts and back on a B200: operands that change from call to call, and calls that are refused."""
import pytest
import torch

import void_b200 as void
from void_b200 import _lib
from test_routing_gpu import _gen, _sorted

pytestmark = pytest.mark.gpu


def test_tokens_and_choices_written_just_before_by_a_few_blocks():
    """Every call has other tokens and other choices, written by kernels of a few blocks right before it: nothing that a multiprocessor read in the call
    before may be used again."""
    n, top, d, experts = 700, 2, 8, 24
    for dtype, index in ((torch.float32, torch.int64), (torch.bfloat16, torch.int32)):
        x, ids = torch.empty(n, d, dtype=dtype, device="cuda"), torch.empty(n, top, dtype=index, device="cuda")
        given = [(torch.randn(n, d, generator=_gen(s), device="cuda").to(dtype), torch.randint(-1, experts, (n, top), generator=_gen(10 + s), device="cuda").to(index))
                 for s in range(5)]
        sorted_ids = [_sorted(ids_, experts) for _, ids_ in given]
        got = []
        for i in range(60):
            x.copy_(given[i % 5][0])
            ids.copy_(given[i % 5][1])
            got.append(void.void_dispatch(x, ids, experts))
        for i, (rows, routes) in enumerate(got):
            tokens = given[i % 5][0]
            offsets, position = sorted_ids[i % 5]
            assert torch.equal(routes.offsets, offsets) and torch.equal(routes.position, position), i
            at = position.flatten()
            want = torch.zeros(n * top, d, dtype=dtype, device="cuda")
            want[at[at >= 0].long()] = tokens.repeat_interleave(top, 0)[at >= 0]
            assert torch.equal(rows, want), i


def test_too_many_features_are_refused_with_the_limit():
    x, ids = torch.empty(1, 67107833, dtype=torch.bfloat16, device="cuda"), torch.zeros(1, 1, dtype=torch.int32, device="cuda")
    with pytest.raises(_lib.VoidB200Error, match="at most 67107832 features, got 67107833"):
        void.void_dispatch(x, ids, 1)
    with pytest.raises(_lib.VoidB200Error, match="at most 67107832 features, got 67107833"):
        void.void_combine(x, void.sort_by_expert(ids, 1))
    most = torch.ones(1, 67107832, dtype=torch.bfloat16, device="cuda")
    rows, routes = void.void_dispatch(most, ids, 1)
    assert torch.equal(rows, most) and torch.equal(void.void_combine(rows, routes), most)


@pytest.mark.parametrize("tokens, top", [(1, 1), (64, 8), (513, 1), (57, 9), (128, 8)])
@pytest.mark.parametrize("experts", [1, 7, 51, 52, 64, 65, 249, 300, 1024])
def test_dispatch_on_either_side_of_few_choices_and_experts(tokens, top, experts):
    ids = torch.randint(-1, experts + 1, (tokens, top), generator=_gen(tokens + experts), device="cuda")
    x = torch.randn(tokens, 24, generator=_gen(3), device="cuda").bfloat16()
    offsets, position = _sorted(torch.where(ids < experts, ids, -1), experts)
    for index in (torch.int32, torch.int64):
        rows, routes = void.void_dispatch(x, ids.to(index), experts)
        assert torch.equal(routes.offsets, offsets) and torch.equal(routes.position, position)
        alone = void.sort_by_expert(ids.to(index), experts)
        assert torch.equal(alone.offsets, offsets) and torch.equal(alone.position, position)
        at = position.flatten()
        want = torch.zeros_like(rows)
        want[at[at >= 0].long()] = x.repeat_interleave(top, 0)[at >= 0]
        assert torch.equal(rows, want)


def test_few_choices_of_many_experts_cost_what_the_sort_costs():
    """1024 choices of 1024 experts: not the many passes of one block over all choices (53 us on a B200) that the form for few experts would take."""
    ids = torch.randint(0, 1024, (128, 8), generator=_gen(1), device="cuda")
    x = torch.randn(128, 256, generator=_gen(2), device="cuda").bfloat16()

    def us(call):
        call()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            kept = [call() for _ in range(20)]
        best = float("inf")
        for _ in range(5):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            graph.replay()
            b.record()
            b.synchronize()
            best = min(best, a.elapsed_time(b) * 1e3 / len(kept))
        return best
    assert us(lambda: void.void_dispatch(x, ids, 1024)) < 2 * us(lambda: void.sort_by_expert(ids, 1024))


def test_an_argument_without_a_truth_is_refused():
    with pytest.raises(RuntimeError, match="ambiguous"):
        void.void_route(torch.randn(4, 8, device="cuda"), 2, torch.tensor([1, 0]))


@pytest.mark.parametrize("count, experts", [(8192, 1024), (8193, 1024), (32768, 1023), (32769, 1024), (200001, 1024), (140000, 1)])
def test_sorts_of_many_choices_of_many_experts(count, experts):
    ids = torch.randint(-1, experts, (count, 1), generator=_gen(count), device="cuda", dtype=torch.int32)
    flat = ids.flatten()
    order = torch.where(flat < 0, experts, flat).sort(stable=True).indices[: int((flat >= 0).sum())]
    position = torch.full((count,), -1, dtype=torch.int32, device="cuda")
    position[order] = torch.arange(order.numel(), dtype=torch.int32, device="cuda")
    ends = torch.bincount(flat[flat >= 0], minlength=experts).cumsum(0).int()
    routes = void.sort_by_expert(ids, experts)
    assert torch.equal(routes.position.flatten(), position) and routes.offsets[0] == 0 and torch.equal(routes.offsets[1:], ends)
