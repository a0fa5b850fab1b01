"""Routing and 8-bit layers: a kernel that starts beside the end of the kernel before it waits for that one as a whole, every thread
of it and before anything else, and reads nothing of an operand ahead of the wait."""
import re

import pytest

from test_kernel_rules_cpu import KERNELS, WAIT

FILES = ("route.cu", "fp8_blocks.cu")
# members of the parameters that are sizes and rules of the launch, not addresses
SIZES = {"pitch", "stages", "wait_limit_ms", "splits", "k_blocks"}
MINE = [k for k in KERNELS if k[0] in FILES]


def _depth(text):
    return text.count("{") - text.count("}")


def test_the_kernels_are_found():
    assert {"route_kernel", "sort_cluster_kernel", "sort_count_kernel", "sort_place_kernel", "dispatch_kernel", "combine_kernel", "combine_grad_kernel",
            "quant_rows_kernel", "quant_blocks_kernel", "fp8_block_kernel", "fp8_wide_kernel"} <= {k[1] for k in MINE}


@pytest.mark.parametrize("kernel", MINE, ids=lambda k: k[1])
def test_all_threads_wait_before_they_read(kernel):
    _, name, _, body = kernel
    waits = list(WAIT.finditer(body))
    assert len(waits) == 1, name
    before = body[:waits[0].start()]
    assert _depth(before) == 0 and before.strip()[-1:] in ("", ";", "}"), (name, "the wait has a condition")
    assert set(re.findall(r"\bp\.(\w+)", before)) <= SIZES, name
    assert not re.search(r"\b(item_at|items_of|find_runs|tma_load_\dd|bulk_load|reinterpret_cast<const T)\b", before), name
