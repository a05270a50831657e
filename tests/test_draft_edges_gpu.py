"""Calls of the drafts' operators at the edges of what their documentation allows, against 64 bits on the CPU (`draft_reference.py`, where the
bounds are derived)."""
import pytest
import torch

import draft_reference as plain
from test_draft_tree_gpu import check

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from fllm_amd.kernels import Ops
    return Ops()


@pytest.mark.parametrize("dim,rows,dtype", [(128, 16, torch.bfloat16), (128, 32, torch.bfloat16), (128, 64, torch.bfloat16), (128, 128, torch.bfloat16), (64, 16, torch.bfloat16),
                                            (64, 64, torch.bfloat16), (40, 0, torch.bfloat16), (64, 0, torch.float32), (128, 0, torch.float32)])
@pytest.mark.parametrize("window", [1, 16, 100])
def test_a_window_goes_by_positions_wherever_the_nodes_lie(ops, dim, rows, window, dtype):
    """Positions above and below the slots: a node is seen or not by its `row_pos`, its value comes from its slot."""
    case = plain.TreeCase([(1000, 6), (40, 70), (130, 33), (0, 9), (64, 64)], 8, 2, dim, 8 if dim == 40 else 16, dtype, seed=dim + window)
    for s, shift in enumerate((95, 17, -60, 4000, 120)):
        case.row_pos[int(case.seg_start[s]): int(case.seg_start[s + 1])] += shift
    ops.set_option("attention.tree_rows", rows)
    try:
        check(ops, case, window=window)
        check(ops, case, window=window, sinks=True)
        # a sibling that is not finite stays where it is seen
        case.seen_of[0] = [{0}, {0, 1}, {2}, {0, 3}, {0, 4}, {0, 2, 5}]
        case.values[0][1000 + 1] = float("nan")
        case.put(0, 1001)
        row_pos = case.row_pos[:6].clone()
        case.row_pos[:6] = 1095
        check(ops, case, window=window)
        case.row_pos[:6] = row_pos
    finally:
        ops.set_option("attention.tree_rows", 0)
