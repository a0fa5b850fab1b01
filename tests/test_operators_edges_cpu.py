"""What layers of experts refuse at an edge, without a GPU."""
import pytest
import torch

import void_b200 as void
from test_experts_cpu import _cpu_weight


def test_stacking_refuses_tiles_of_another_expert():
    a, b = _cpu_weight(70, 96), _cpu_weight(70, 96, 5)
    for row in (3, -1):                       # 70 outputs are three tile rows: the fourth would be the next expert's first
        bad = void.VOIDTensor(b.values, b.block_rows.clone(), b.block_cols, b.morton_codes, b.shape, (32, 32), 0, b.n_blocks, 0.0)
        bad.block_rows[1] = row
        for weights in ([a, bad], [bad, a]):
            with pytest.raises(ValueError, match="invalid VOID tile list"):
                void.stack_experts(weights)
    e = void.stack_experts([a, b])
    assert torch.equal(e.tensor.block_rows, torch.cat([a.block_rows, b.block_rows + 3])) and e.tensor.block_rows.dtype == torch.int32
    assert void.stack_experts([void.VOIDTensor(a.values[:0], a.block_rows[:0], a.block_cols[:0], a.morton_codes[:0], a.shape, (32, 32), 0, 0, 0.0)] * 2).tensor.n_blocks == 0
