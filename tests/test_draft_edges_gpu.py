"""Calls of the drafts' operators at the edges of what their documentation allows, against 64 bits on the CPU (`draft_reference.py`, where the
bounds are derived)."""
import pytest
import torch

import draft_reference as plain
from test_draft_tree_gpu import attend, check

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


@pytest.mark.parametrize("heads,kv_heads,dim,page", [(4, 2, 128, 16), (32, 8, 128, 16), (6, 6, 64, 8), (32, 8, 64, 64)])
@pytest.mark.parametrize("slots,positions", [("run", "depths"), ("run", "run"), ("scattered", "run"), ("reversed", "run"), ("run", "below"), ("short", "depths")])
def test_eight_rows_that_lie_together_are_found_by_their_slots(ops, heads, kv_heads, dim, page, slots, positions):
    """Batches of 256 rows and more store the values of eight neighbouring slots together, wherever the rows' positions are.

    Values are copied: bit for bit.  A rotated lane is a c - b s in float32 (roundings of 2^-24 of |a c| + |b s|, fewer than eight of them) and is
    rounded to bfloat16 once (2^-8 of the value)."""
    gen = torch.Generator().manual_seed(heads + dim)
    each, kept, width = 152, 8, 200 // page + 1
    rows = 2 * each + 1
    qkv = torch.randn((rows, (heads + 2 * kv_heads) * dim), generator=gen).to(torch.bfloat16)
    tables = torch.randperm(2 * width, generator=gen).to(torch.int32).reshape(2, width)
    angles = torch.randn((400, dim // 2), generator=gen)
    row_seg = torch.tensor([0] * each + [1] * each + [-1], dtype=torch.int32)
    own = {"run": list(range(each)), "scattered": torch.randperm(each, generator=gen).tolist(), "reversed": list(range(each))[::-1],
           "short": [i + i // 7 for i in range(each)]}[slots]          # seven neighbours, then a gap
    slot = torch.tensor([kept + n for n in own] * 2 + [0], dtype=torch.int32)
    at = {"depths": [kept + n // 3 for n in range(each)], "run": [kept + n for n in range(each)], "below": [n % 8 for n in range(each)]}[positions]
    pos = torch.tensor(at * 2 + [0], dtype=torch.int32)
    k = torch.zeros((2 * width, kv_heads, dim // 8, page, 8), dtype=torch.bfloat16)
    v = torch.zeros((2 * width, kv_heads, dim, page), dtype=torch.bfloat16)
    got, got_k, got_v = qkv.cuda(), k.cuda(), v.cuda()
    ops.rope_kv_store(got, pos.cuda(), row_seg.cuda(), tables.cuda(), angles.cos().cuda(), angles.sin().cuda(), got_k, got_v, heads, kv_heads, dim, dim, 1, page,
                      row_slot=slot.cuda())
    got, got_k, got_v = got.cpu(), got_k.cpu(), got_v.cpu()
    x = qkv[: 2 * each, : (heads + kv_heads) * dim].double().reshape(2 * each, heads + kv_heads, dim // 2, 2)
    c, s = angles.cos().double()[pos[: 2 * each].long()][:, None], angles.sin().double()[pos[: 2 * each].long()][:, None]
    a, b = x[..., 0], x[..., 1]
    want = torch.stack([a * c - b * s, b * c + a * s], -1).reshape(2 * each, heads + kv_heads, dim)
    size = torch.stack([(a * c).abs() + (b * s).abs(), (b * c).abs() + (a * s).abs()], -1).reshape_as(want)
    near = lambda value, r, part: bool(((value.double() - want[r, part]).abs() <= want[r, part].abs() * 2.0 ** -8 + size[r, part] * 2.0 ** -21).all())
    written_k, written_v = torch.zeros_like(got_k, dtype=torch.bool), torch.zeros_like(got_v, dtype=torch.bool)
    values = qkv[:, (heads + kv_heads) * dim:].reshape(rows, kv_heads, dim)
    for r in range(2 * each):
        p, off = int(tables[int(row_seg[r]), int(slot[r]) // page]), int(slot[r]) % page
        assert near(got[r, : heads * dim].view(heads, dim), r, slice(0, heads))
        assert near(got_k[p, :, :, off].reshape(kv_heads, dim), r, slice(heads, None))
        assert torch.equal(got_v[p, :, :, off], values[r])
        written_k[p, :, :, off] = True
        written_v[p, :, :, off] = True
    assert bool((got_k[~written_k] == 0).all()) and bool((got_v[~written_v] == 0).all())
    assert torch.equal(got[2 * each], qkv[2 * each])


LONG = {3: (2500, 40), 64: (3100, 17), 65: (1100, 33), 100: (6000, 5), 127: (1500, 16), 128: (2100, 49), 149: (4000, 20)}


@pytest.mark.parametrize("heads,kv_heads,window", [(8, 1, 0), (6, 2, 0), (6, 3, 700), (8, 1, 1500)])
def test_more_requests_than_a_wave_has_lanes_are_cut(ops, heads, kv_heads, window):
    """Tiles of 128 rows look the requests' lengths over 64 at a time: long ones among the first 64, at the edges and behind them."""
    requests = [LONG.get(i, (7 * i % 60, 0 if i % 11 == 5 else 1 + i % 5)) for i in range(150)]
    case = plain.TreeCase(requests, heads, kv_heads, 128, 16, torch.bfloat16, seed=heads + kv_heads)
    ops.set_option("attention.tree_rows", 128)
    try:
        first = check(ops, case, window=window)
        assert bool((attend(ops, case, 128 ** -0.5, window=window).cpu() == first).all()), "a second call gives other bits"
    finally:
        ops.set_option("attention.tree_rows", 0)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("heads,kv_heads,dim,page", [(8, 2, 32, 16), (6, 3, 96, 16), (4, 2, 256, 16), (72, 1, 64, 16), (8, 2, 64, 128), (8, 2, 128, 4)])
def test_shapes_of_the_plain_kernel_over_long_contexts(ops, heads, kv_heads, dim, page, dtype):
    case = plain.TreeCase([(3100, 11), (1, 5), (1023, 2)], heads, kv_heads, dim, page, dtype, seed=dim + page)
    check(ops, case)
    check(ops, case, window=1024, sinks=True)


def test_a_request_that_ends_and_choices_that_are_refused(ops):
    """The step's kernels behind what the engine's own tests do on the CPU: a batch of which one request has ended, a choice of the wrong type."""
    import numpy as np
    import plain_llama
    import tiny_configs as tc
    from fllm_amd.engine import StepEntry, TreeEntry
    from fllm_amd.kernels import KernelError
    from test_draft_steps_gpu import TOL, runner_of
    runner, cfg, weights = runner_of("E", "float32")
    prompts = {r: tc.random_ids(n, cfg["vocab_size"], n) for r, n in (("a", 17), ("b", 30), ("c", 5))}
    newest = dict(zip(prompts, runner.step([StepEntry(r, p, want=(len(p) - 1,)) for r, p in prompts.items()]).argmax(dim=1).tolist()))
    second = {r: int(np.argmax(plain_llama.forward(cfg, weights, prompts[r] + [newest[r]])[-1])) for r in prompts}
    chosen = runner.step_tree([TreeEntry(r, [newest[r], 1, second[r]], [-1, 0, 0]) for r in prompts]).argmax(dim=1)
    with pytest.raises(KernelError):
        runner.keep_tree(chosen)                   # 64-bit numbers: refused ahead of the first move
    runner.free_request("b")
    kept = runner.keep_tree(chosen.int())
    assert kept[0][0] == [0, 2] and kept[1] == ([], -1) and kept[2][0] == [0, 2]
    got = runner.step([StepEntry(r, [kept[i][1]], want=(0,)) for i, r in ((0, "a"), (2, "c"))]).cpu().numpy()
    for row, (i, r) in zip(got, ((0, "a"), (2, "c"))):
        want = plain_llama.forward(cfg, weights, prompts[r] + [newest[r], second[r], kept[i][1]])[-1]
        assert np.abs(row - want).max() <= TOL["float32"] * np.abs(want).max()
    runner.cache.check_invariants()


@pytest.mark.parametrize("pairs", [63, 64, 399, 401, 447, 448, 449, 895, 897])
def test_copies_at_the_edges_of_a_launch(ops, pairs):
    store = torch.arange(2 * 2000 * 12, dtype=torch.float32).reshape(2, 2000, 12)
    pages = torch.randperm(2000, generator=torch.Generator().manual_seed(pairs)).tolist()
    source, target = pages[:pairs], pages[1000:1000 + pairs]
    device = store.cuda()
    ops.copy_pages((device,), source, target)
    store[:, target] = store[:, source]
    assert torch.equal(device.cpu(), store)
