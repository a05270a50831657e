"""Trees of drafted tokens over the paged cache: attention, the walk, moving and copying, against 64 bits on the CPU
(`draft_reference.py`, where the bounds are derived)."""
import random

import pytest
import torch

import draft_reference as plain

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from fllm_amd.kernels import Ops
    return Ops()


def attend(ops, case, scale, window=0, sinks=False, max_nodes=None, max_context=None, out=None):
    dev = lambda t: t.cuda()
    joint = dev(case.joint)
    out = torch.full((case.rows, case.heads * case.v_dim), 7.0, dtype=case.dtype, device="cuda") if out is None else out
    most = max([k + n for k, n in case.requests] + [0]) if max_context is None else max_context
    got = ops.tree_attention(joint[:, : case.heads * case.dim], dev(case.k_pages), dev(case.v_pages), dev(case.tables), dev(case.row_pos),
                             dev(case.seg_start), dev(case.kept), dev(case.seen), out, case.heads, case.kv_heads, case.dim, case.page, scale, most,
                             window=window or None, sinks=dev(case.sinks) if sinks else None, v_dim=case.v_dim, key_chunk=case.key_chunk,
                             max_nodes=max_nodes)
    assert got is out
    return got


def check(ops, case, scale=None, window=0, sinks=False, **more):
    scale = case.dim ** -0.5 if scale is None else scale
    want, bound = case.expected(scale, window, sinks)
    got = attend(ops, case, scale, window, sinks, **more).cpu()
    assert plain.compare(got[: case.live_rows], want[: case.live_rows], bound[: case.live_rows]) <= 1.0
    assert bool((got[case.live_rows:] == 7.0).all()), "rows behind the last segment have changed"
    return got


RAGGED = [(0, 1), (1, 1), (5, 3), (0, 9), (63, 2), (64, 33), (127, 1), (200, 17), (257, 5)]
SHAPES = [(8, 2, 128), (8, 8, 64), (14, 2, 64), (40, 2, 32), (36, 2, 128), (9, 3, 24), (130, 2, 64), (4, 1, 256)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("heads,kv_heads,dim", SHAPES)
@pytest.mark.parametrize("page", [8, 16, 32, 64])
def test_attention_of_ragged_trees(ops, heads, kv_heads, dim, page, dtype):
    check(ops, plain.TreeCase(RAGGED, heads, kv_heads, dim, page, dtype, seed=heads + dim + page, spare_rows=3))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("dim,page", [(128, 16), (64, 32), (64, 8), (40, 5)])
@pytest.mark.parametrize("window", [1, 2, 7, 64, 130, 5000])
def test_attention_with_a_window_and_sinks(ops, dim, page, window, dtype):
    case = plain.TreeCase(RAGGED + [(600, 40)], 8, 2, dim, page, dtype, seed=window + dim, words=3)
    check(ops, case, window=window, sinks=True)
    check(ops, case, window=window)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_attention_over_long_contexts_is_split_and_joined(ops, dtype):
    for kept, nodes, heads, kv_heads, dim in [(5000, 8, 8, 2, 128), (9001, 16, 8, 2, 64), (3001, 70, 8, 1, 128), (4097, 1, 4, 4, 128)]:
        case = plain.TreeCase([(kept, nodes), (kept // 3, 3)], heads, kv_heads, dim, 16, dtype, seed=kept)
        first = check(ops, case, sinks=True)
        again = check(ops, case, sinks=True)
        assert torch.equal(first, again), "a second call gives other bits"
    torch.cuda.synchronize()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("nodes", [1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 100, 128, 129, 200])
def test_attention_of_trees_of_any_size(ops, nodes, dtype):
    check(ops, plain.TreeCase([(70, nodes), (3, max(1, nodes // 2))], 8, 2, 64, 16, dtype, seed=nodes))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("dim,heads,kv_heads", [(128, 8, 2), (64, 4, 4), (24, 4, 2)])
def test_what_a_row_does_not_see_does_not_reach_it(ops, dim, heads, kv_heads, dtype):
    """Siblings that hold NaN and infinities, a row that sees nothing at all, a table entry that names no page."""
    case = plain.TreeCase([(100, 12), (0, 6), (40, 4)], heads, kv_heads, dim, 16, dtype, seed=dim)
    case.seen_of[0] = [{i} if i % 3 == 0 else {0, 3, i} if i % 3 == 1 else set(range(0, 12, 3)) for i in range(12)]
    for j, value in ((1, float("nan")), (2, float("inf")), (4, float("-inf")), (5, float("nan"))):
        case.values[0][100 + j] = value
        case.put(0, 100 + j)
    case.seen_of[0][1], case.seen_of[0][4] = {0}, {3, 6}
    case.keys[0][100 + 2] = float("nan")
    case.keys[0][100 + 5] = float("inf")
    case.put(0, 102), case.put(0, 105)
    case.seen_of[0][2], case.seen_of[0][5], case.seen_of[0][8] = {0}, {9}, {11}
    case.seen_of[1] = [set(), {0, 1}, set(), {3}, {63}, {5}]          # rows that see nothing; a bit behind the last node
    case.tables[2, 0] = case.k_pages.shape[0]                        # no such page: its sixteen tokens are not there
    case.tables[2, 1] = -5
    got = check(ops, case)
    assert bool(torch.isfinite(got[: case.live_rows].float()).all())
    assert bool((got[12] == 0).all()) and bool((got[14] == 0).all()) and bool((got[16] == 0).all())
    check(ops, case, sinks=True)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("dim,rows", [(64, 0), (128, 0), (128, 64), (128, 128), (64, 64)])
def test_what_a_row_sees_does_reach_it(ops, dim, rows, dtype):
    case = plain.TreeCase([(100, 12)], 4, 2, dim, 16, dtype, seed=3)
    ops.set_option("attention.tree_rows", rows)
    case.seen_of[0] = [{0, i} for i in range(12)]
    for j, value in ((1, float("nan")), (2, float("inf")), (3, float("-inf"))):
        case.values[0][100 + j] = value
        case.put(0, 100 + j)
    try:
        got = attend(ops, case, 0.125).float().cpu()
    finally:
        ops.set_option("attention.tree_rows", 0)
    assert bool(torch.isnan(got[1]).all()) and bool((got[2] == float("inf")).all()) and bool((got[3] == float("-inf")).all())
    assert bool(torch.isfinite(got[[0] + list(range(4, 12))]).all())


@pytest.mark.parametrize("scale", [0.0, -0.2, 3.0])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_attention_with_other_scales(ops, scale, dtype):
    check(ops, plain.TreeCase([(300, 9)], 8, 2, 64, 16, dtype, seed=1), scale=scale)


def test_attention_with_widths_of_their_own(ops):
    check(ops, plain.TreeCase(RAGGED, 6, 2, 96, 16, torch.bfloat16, seed=1, v_dim=40))
    check(ops, plain.TreeCase(RAGGED, 6, 2, 36, 16, torch.float32, seed=2, v_dim=300, key_chunk=1))


def test_rows_beyond_the_bound_and_empty_calls(ops):
    case = plain.TreeCase([(50, 10), (20, 2)], 8, 2, 64, 16, torch.bfloat16, seed=5)
    got = attend(ops, case, 0.125, max_nodes=0)
    assert bool((got == 7.0).all())
    want, bound = case.expected(0.125)
    got = attend(ops, case, 0.125, max_nodes=10, max_context=1)          # a bound that is too low costs time, not keys
    assert plain.compare(got, want, bound) <= 1.0


@pytest.mark.parametrize("plain_kernels", [False, True])
def test_the_plain_kernel_and_the_fast_one(ops, plain_kernels):
    case = plain.TreeCase(RAGGED, 8, 2, 128, 16, torch.bfloat16, seed=11)
    ops.set_fast_kernels(not plain_kernels)
    try:
        check(ops, case, sinks=True)
    finally:
        ops.set_fast_kernels(True)


@pytest.mark.parametrize("rows", [16, 32, 64, 128])
@pytest.mark.parametrize("heads,kv_heads,dim,page", [(8, 2, 128, 16), (8, 1, 128, 8), (14, 2, 128, 32), (36, 2, 128, 64), (8, 2, 64, 16), (40, 2, 64, 8), (8, 8, 128, 64)])
def test_tiles_of_any_number_of_rows(ops, rows, heads, kv_heads, dim, page):
    """What the launch chooses by the number of tiles and the reach of their rows, asked for by hand."""
    ops.set_option("attention.tree_rows", rows)
    try:
        case = plain.TreeCase(RAGGED + [(900, 70)], heads, kv_heads, dim, page, torch.bfloat16, seed=rows + dim + page, spare_rows=2)
        check(ops, case)
        check(ops, case, window=50, sinks=True)
        check(ops, case, scale=-0.1)
        case = plain.TreeCase([(3000, 30), (1, 90)], heads, kv_heads, dim, page, torch.bfloat16, seed=rows + dim)
        assert torch.equal(check(ops, case, sinks=True), check(ops, case, sinks=True))
        test_what_a_row_does_not_see_does_not_reach_it(ops, dim, heads, kv_heads, torch.bfloat16)
    finally:
        ops.set_option("attention.tree_rows", 0)


# ---- the walk --------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("sizes,most", [([1], 1), ([1, 2, 3], 4), ([64], 70), ([65, 0, 7, 130, 63], 9), ([300, 200], 16), ([40] * 70, 3), ([0], 2)])
@pytest.mark.parametrize("seed", [0, 1, 2])
def test_the_walk(ops, sizes, most, seed):
    rng = random.Random(seed + 100 * most)
    parents, drafted, chosen, want = [], [], [], []
    for n in sizes:
        mine = plain.random_tree(n, rng, 0.6) if n else []
        tokens, picks = [rng.randrange(6) for _ in range(n)], [rng.randrange(6) for _ in range(n)]
        for i in range(n):
            children = [c for c in range(i + 1, n) if mine[c] == i]
            if children and rng.random() < 0.85:
                picks[i] = tokens[rng.choice(children)]
        want.append(plain.follow(mine, tokens, picks, most))
        parents += mine
        drafted += tokens
        chosen += picks
    starts = [0]
    for n in sizes:
        starts.append(starts[-1] + n)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
    path = torch.full((len(sizes), most), 77, dtype=torch.int32, device="cuda")
    length, newest = i32([9] * len(sizes)), i32([9] * len(sizes))
    ops.follow_tree(i32(drafted), i32(parents), i32(starts), i32(chosen), path, length, newest)
    assert path.tolist() == [p + [-1] * (most - len(p)) for p, _ in want]
    assert length.tolist() == [len(p) for p, _ in want] and newest.tolist() == [t for _, t in want]


# ---- moving and copying -----------------------------------------------------------------------------------------------------
def stores(shape_k, shape_v, dtype, seed):
    gen = torch.Generator().manual_seed(seed)
    make = lambda shape: torch.randn(shape, generator=gen).to(dtype)
    return make(shape_k), make(shape_v) if shape_v else None


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("page,dim,v_dim,chunk", [(16, 128, 128, 8), (8, 64, 64, 8), (64, 32, 48, 8), (5, 12, 7, 1), (16, 72, 0, 0), (32, 576, 0, 8)])
def test_moving(ops, page, dim, v_dim, chunk, dtype):
    """Paths whose targets are later sources, that cross pages, that stay where they are, that do not rise, of length zero, and slots without
    a page."""
    rng = random.Random(page * dim)
    layers, kv_heads = 3, 2
    kept = [0, 3, page - 1, 2 * page + 1, 7, 4, 10, 1]
    paths = [[0, 1, 2], [0, 2, 5, 11], [0, 1, 3, 4], [3, 4, 5, 6, 9, 12], [0, 5, 4, 9], [-1, 2], [0, 2 * page], []]
    lengths = [3, 4, 4, 6, 4, 2, 2, 0]
    most = 7
    width = 4 + 12 // page
    pages = len(kept) * width + 2
    order = rng.sample(range(pages), len(kept) * width)
    tables = torch.tensor(order, dtype=torch.int32).reshape(len(kept), width)
    tables[6, (10 + 2 * page) // page] = -1            # the second move of that request has no source
    shape_k = (layers, pages, kv_heads, dim // chunk, page, chunk) if chunk else (layers, pages, kv_heads, page, dim)
    k, v = stores(shape_k, (layers, pages, kv_heads, v_dim, page) if v_dim else None, dtype, seed=dim)
    wants = [t.clone() if t is not None else None for t in (k, v)]
    for old, new, token_axis in ((k, wants[0], -2), (v, wants[1], -1)):
        if old is None:
            continue
        old, new = old.movedim(token_axis, 2), new.movedim(token_axis, 2)      # [layers, pages, token, ...]
        for s, path in enumerate(paths):
            last = -1
            for i, node in enumerate(path[: lengths[s]]):
                if node <= last:
                    break
                last = node
                (a, b), (c, d) = divmod(kept[s] + node, page), divmod(kept[s] + i, page)
                if a < width and int(tables[s, a]) >= 0 and int(tables[s, c]) >= 0:
                    new[:, int(tables[s, c]), d] = old[:, int(tables[s, a]), b]
    dev_k, dev_v = k.cuda(), v.cuda() if v is not None else None
    i32 = lambda t: torch.tensor(t, dtype=torch.int32, device="cuda")
    ops.move_tokens(dev_k, dev_v, tables.cuda(), i32(kept), i32([p + [-1] * (most - len(p)) for p in paths]), i32(lengths))
    assert torch.equal(dev_k.cpu(), wants[0])
    assert v is None or torch.equal(dev_v.cpu(), wants[1])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_moving_a_long_path(ops, dtype):
    """A chain of 150 of 200 nodes, every other one, all layers of several heads."""
    k, v = stores((2, 60, 3, 8, 16, 8), (2, 60, 3, 64, 16), dtype, seed=4)
    path = [i for i in range(200) if i % 4 != 2]
    tables = torch.randperm(60, generator=torch.Generator().manual_seed(1))[:14].to(torch.int32)[None]
    kept = 9
    flat = lambda t, axis: t.movedim(axis, 2)[:, tables[0].long()].flatten(1, 2)          # [layers, slot, ...]
    want_k, want_v = flat(k, 4).clone(), flat(v, 4).clone()
    source = [kept + n for n in path]
    want_k[:, kept:kept + len(path)] = flat(k, 4)[:, source]
    want_v[:, kept:kept + len(path)] = flat(v, 4)[:, source]
    dev_k, dev_v = k.cuda(), v.cuda()
    i32 = lambda t: torch.tensor(t, dtype=torch.int32, device="cuda")
    ops.move_tokens(dev_k, dev_v, tables.cuda(), i32([kept]), i32([path]), i32([len(path)]))
    assert torch.equal(flat(dev_k.cpu(), 4), want_k) and torch.equal(flat(dev_v.cpu(), 4), want_v)


@pytest.mark.parametrize("pairs", [0, 1, 3, 130, 300])
@pytest.mark.parametrize("shapes", [[((3, 700), (2, 16, 16, 8)), ((3, 700), (2, 128, 16))], [((1, 640), (3, 5))], [((2, 620), (7,)), ((5, 610), (2, 33, 3))]])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_copying(ops, pairs, shapes, dtype):
    rng = random.Random(pairs)
    chosen = rng.sample(range(600), pairs + max(1, pairs // 3))
    target, some = chosen[:pairs], chosen[pairs:]
    source = [rng.choice(some) for _ in range(pairs)]            # a page may be copied several times
    gen = torch.Generator().manual_seed(pairs)
    host = [torch.randn((*lead, *rest), generator=gen).to(dtype) for lead, rest in shapes]
    device = [t.cuda() for t in host]
    ops.copy_pages(device, source, target)
    for t in host:
        t[:, target] = t[:, source]
    for a, b in zip(host, device):
        assert torch.equal(a, b.cpu())


def test_copying_more_pages_than_a_launch_takes(ops):
    rng = random.Random(7)
    chosen = rng.sample(range(2000), 1300)
    source, target = chosen[:30] * 33, chosen[310:1300]
    store = torch.randn((2, 2000, 3, 8), generator=torch.Generator().manual_seed(1))
    device = store.cuda()
    ops.copy_pages((device,), source, target)
    store[:, target] = store[:, source]
    assert torch.equal(device.cpu(), store)


def test_rotary_positions_that_are_not_slots(ops):
    """`rope_kv_store(row_slot=)` stores at the slot what the call without it stores at the position."""
    from fllm_amd.kernels import KernelError
    gen = torch.Generator().manual_seed(2)
    for dtype, rows, dim, page, pairing in ((torch.bfloat16, 20, 64, 16, 1), (torch.bfloat16, 300, 128, 16, 1), (torch.float32, 9, 32, 8, 0), (torch.bfloat16, 9, 20, 8, 1)):
        chunk = 8 if dim % 8 == 0 else 1
        heads, kv_heads, width = 4, 2, 60
        qkv = torch.randn((rows, (heads + 2 * kv_heads) * dim), generator=gen).to(dtype)
        tables = torch.randperm(2 * width, generator=gen).to(torch.int32).reshape(2, width)
        angles = torch.randn((400, dim // 2), generator=gen)
        half = rows // 2
        row_seg = torch.tensor([0] * half + [1] * (rows - half - 1) + [-1], dtype=torch.int32)
        slot = torch.tensor([5 + i for i in range(half)] + [8 + i for i in range(rows - half)], dtype=torch.int32)
        pos = torch.tensor([5 + i // 2 for i in range(half)] + [8 + i // 3 for i in range(rows - half)], dtype=torch.int32)
        k = torch.zeros((2 * width, kv_heads, dim // chunk, page, chunk), dtype=dtype)
        v = torch.zeros((2 * width, kv_heads, dim, page), dtype=dtype)
        dev = lambda t: t.cuda()

        def call(positions, cos, sin, **more):
            a, b, c = dev(qkv), dev(k), dev(v)
            ops.rope_kv_store(a, dev(positions), dev(row_seg), dev(tables), dev(cos), dev(sin), b, c, heads, kv_heads, dim, dim, pairing, page, key_chunk=chunk, **more)
            return a.cpu(), b.cpu(), c.cpu()

        # the same angles at the slots' own places: what the rows of two requests need of the table is gathered a row at a time
        got = call(pos, angles.cos(), angles.sin(), row_slot=slot.cuda())
        for seg in (0, 1):
            mine = (row_seg == seg)
            cos, sin = angles.cos().clone(), angles.sin().clone()
            cos[slot[mine].long()], sin[slot[mine].long()] = angles.cos()[pos[mine].long()], angles.sin()[pos[mine].long()]
            want = call(slot, cos, sin)
            assert torch.equal(got[0][mine], want[0][mine])
            pages = tables[seg].long()
            assert torch.equal(got[1][pages], want[1][pages]) and torch.equal(got[2][pages], want[2][pages])
        with pytest.raises(KernelError):
            call(pos, angles.cos(), angles.sin(), row_slot=slot[1:].cuda())


# ---- what is refused --------------------------------------------------------------------------------------------------------
def test_refusals(ops):
    from fllm_amd.kernels import KernelError
    case = plain.TreeCase([(20, 4), (3, 2)], 4, 2, 32, 16, torch.bfloat16, seed=1)
    dev = lambda t: t.cuda()
    good = dict(q=dev(case.joint[:, :128]).contiguous(), k_pages=dev(case.k_pages), v_pages=dev(case.v_pages), tables=dev(case.tables), row_pos=dev(case.row_pos),
                seg_start=dev(case.seg_start), kept=dev(case.kept), seen=dev(case.seen), out=torch.empty((6, 128), dtype=torch.bfloat16, device="cuda"),
                heads=4, kv_heads=2, head_dim=32, page_size=16, scale=0.2, max_context=24)
    ops.tree_attention(**good)
    for wrong in (dict(q=good["q"].float()), dict(q=good["q"].half()), dict(q=case.joint[:, :128]), dict(q=good["q"].t()), dict(out=good["out"][:5]), dict(out=good["out"].cpu()),
                  dict(seen=good["seen"].int()), dict(seen=good["seen"][:, :0]), dict(kept=good["kept"][:1]), dict(seg_start=good["seg_start"][1:]),
                  dict(tables=good["tables"].long()), dict(tables=good["tables"][:, ::2]), dict(row_pos=good["row_pos"][1:]), dict(page_size=8), dict(kv_heads=4),
                  dict(heads=3), dict(head_dim=16), dict(k_pages=good["k_pages"].float()), dict(v_pages=good["v_pages"][:, :1]), dict(max_nodes=65), dict(max_nodes=-1),
                  dict(sinks=torch.zeros(3, device="cuda")), dict(window=-4), dict(key_chunk=5), dict(max_context=-1)):
        with pytest.raises(KernelError):
            ops.tree_attention(**dict(good, **wrong))
    i32 = lambda *shape: torch.zeros(shape, dtype=torch.int32, device="cuda")
    walk = dict(drafted=i32(6), parents=i32(6), seg_start=good["seg_start"], chosen=i32(6), path=i32(2, 3), length=i32(2), newest=i32(2))
    ops.follow_tree(**walk)
    for wrong in (dict(drafted=i32(5)), dict(parents=i32(6).long()), dict(chosen=i32(6).cpu()), dict(path=i32(3, 3)), dict(path=i32(2, 0)), dict(length=i32(3)),
                  dict(newest=i32(1)), dict(seg_start=i32(2, 2))):
        with pytest.raises(KernelError):
            ops.follow_tree(**dict(walk, **wrong))
    k, v = good["k_pages"][None].clone(), good["v_pages"][None].clone()
    move = dict(k_store=k, v_store=v, tables=good["tables"], kept=good["kept"], path=i32(2, 3), length=i32(2))
    ops.move_tokens(**move)
    for wrong in (dict(k_store=k[0, 0]), dict(k_store=k.half()), dict(v_store=v.float()), dict(v_store=v[:, :1]), dict(v_store=v[0]), dict(kept=i32(3)), dict(path=i32(2, 0)), dict(path=i32(3, 3)),
                  dict(length=i32(2).cpu()), dict(tables=good["tables"][0]), dict(k_store=k.transpose(1, 2))):
        with pytest.raises(KernelError):
            ops.move_tokens(**dict(move, **wrong))
    pages = k.shape[1]
    for stores_given, source, target in (((k, v), [0], [1, 2]), ((k, v), [0], [pages]), ((k, v), [-1], [0]), ((k, v), [0, 1], [2, 2]), ((k, v), [0, 1], [1, 2]), ((), [0], [1]),
                                         ((k,) * 9, [0], [1]), ((k.cpu(),), [0], [1]), ((k.transpose(3, 4),), [0], [1]), ((k.view(-1),), [0], [1])):
        with pytest.raises(KernelError):
            ops.copy_pages(stores_given, source, target)


# ---- together, captured, and in a large cache -------------------------------------------------------------------------------
@pytest.mark.parametrize("dim", [64, 128])
def test_a_captured_run_of_all(ops, dim):
    """Attention over a split context, the walk and the move in one graph, replayed with other inputs and with eager calls (other sizes, the same
    workspace) between the replays; a second graph shares the workspace with it."""
    cases = [plain.TreeCase([(2500, 20), (900, 7)], 8, 2, dim, 16, torch.bfloat16, seed=s) for s in range(3)]
    other = plain.TreeCase([(3300, 9)], 8, 2, dim, 16, torch.bfloat16, seed=9)
    rng = random.Random(dim)
    walks = []
    for case in cases:
        drafted, picks, want = [], [], []
        for parents in case.parents:
            tokens, mine = [rng.randrange(4) for _ in parents], [rng.randrange(4) for _ in parents]
            want.append(plain.follow(parents, tokens, mine, 6))
            drafted += tokens
            picks += mine
        walks.append((drafted, picks, want))
    dev = lambda t: t.clone().cuda()
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
    static = dict(q=dev(cases[0].joint[:, : 8 * dim]), k=dev(cases[0].k_pages)[None], v=dev(cases[0].v_pages)[None], tables=dev(cases[0].tables),
                  pos=dev(cases[0].row_pos), seen=dev(cases[0].seen), parents=i32([p for t in cases[0].parents for p in t]), drafted=i32(walks[0][0]), chosen=i32(walks[0][1]))
    starts, kept = dev(cases[0].seg_start), dev(cases[0].kept)
    out = torch.zeros((27, 8 * dim), dtype=torch.bfloat16, device="cuda")
    path, length, newest = i32([[0] * 6] * 2), i32([0, 0]), i32([0, 0])

    def run():
        ops.tree_attention(static["q"], static["k"][0], static["v"][0], static["tables"], static["pos"], starts, kept, static["seen"], out, 8, 2, dim, 16, dim ** -0.5, 2520)
        ops.follow_tree(static["drafted"], static["parents"], starts, static["chosen"], path, length, newest)
        ops.move_tokens(static["k"], static["v"], static["tables"], kept, path, length)

    graphs = []
    run()
    torch.cuda.synchronize()
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            run()
        graphs.append(graph)
    for turn in range(6):
        case, (drafted, picks, want) = cases[turn % 3], walks[turn % 3]
        static["q"].copy_(case.joint[:, : 8 * dim]), static["k"][0].copy_(case.k_pages), static["v"][0].copy_(case.v_pages), static["tables"].copy_(case.tables)
        static["pos"].copy_(case.row_pos), static["seen"].copy_(case.seen), static["parents"].copy_(i32([p for t in case.parents for p in t]))
        static["drafted"].copy_(i32(drafted)), static["chosen"].copy_(i32(picks))
        check(ops, other)                                   # eager work in the same workspace
        graphs[turn % 2].replay()
        torch.cuda.synchronize()
        expected, bound = case.expected(dim ** -0.5)
        assert plain.compare(out, expected, bound) <= 1.0
        assert length.tolist() == [len(p) for p, _ in want] and newest.tolist() == [t for _, t in want]
        for s, (steps, _) in enumerate(want):               # what the walk kept lies behind the kept tokens
            for i, node in enumerate(steps):
                slot = case.requests[s][0] + i
                page = int(case.tables[s, slot // 16])
                assert torch.equal(static["v"][0, page, :, :, slot % 16].cpu(), case.values[s][case.requests[s][0] + node])
                assert torch.equal(static["k"][0, page, :, :, slot % 16].cpu().reshape(2, dim), case.keys[s][case.requests[s][0] + node])


@pytest.mark.parametrize("dtype,dim,rows", [(torch.bfloat16, 128, 16), (torch.bfloat16, 128, 64), (torch.bfloat16, 128, 128), (torch.bfloat16, 64, 64), (torch.float32, 64, 0), (torch.float32, 40, 0)])
def test_offsets_beyond_32_bits(ops, dtype, dim, rows):
    """The last pages of a cache of more than 2^32 bytes, and a second layer behind it."""
    case = plain.TreeCase([(150, 20), (33, 5)], 8, 8, dim, 16, dtype, seed=dim + rows)
    small = case.k_pages.shape[0]
    pages = -(-(1 << 31) // (8 * dim * 16)) + 5 + small            # more than 2^31 elements of keys, and as many values
    k = torch.empty((2, pages, 8, dim // 8, 16, 8), dtype=dtype, device="cuda")
    v = torch.empty((2, pages, 8, dim, 16), dtype=dtype, device="cuda")
    first = pages - small
    for layer in range(2):
        k[layer, first:], v[layer, first:] = case.k_pages.cuda(), case.v_pages.cuda()
    tables = torch.where(case.tables >= 0, case.tables + first, case.tables).cuda()
    want, bound = case.expected(0.1)
    ops.set_option("attention.tree_rows", rows)
    try:
        for layer in range(2):
            out = torch.zeros((case.rows, 8 * dim), dtype=dtype, device="cuda")
            ops.tree_attention(case.joint[:, : 8 * dim].cuda(), k[layer], v[layer], tables, case.row_pos.cuda(), case.seg_start.cuda(), case.kept.cuda(), case.seen.cuda(), out, 8, 8, dim, 16,
                               0.1, 170)
            assert plain.compare(out, want, bound) <= 1.0
    finally:
        ops.set_option("attention.tree_rows", 0)
    path, length = torch.tensor([[0, 3, 19], [0, 4, -1]], dtype=torch.int32, device="cuda"), torch.tensor([3, 2], dtype=torch.int32, device="cuda")
    ops.move_tokens(k, v, tables, case.kept.cuda(), path, length)
    for s, i, node in ((0, 1, 3), (0, 2, 19), (1, 1, 4)):
        slot = case.requests[s][0] + i
        page = int(tables[s, slot // 16])
        for layer in range(2):
            assert torch.equal(v[layer, page, :, :, slot % 16].cpu(), case.values[s][case.requests[s][0] + node])
            assert torch.equal(k[layer, page, :, :, slot % 16].cpu().reshape(8, dim), case.keys[s][case.requests[s][0] + node])
    k[1, pages - 1], v[1, pages - 1] = 3.0, 4.0
    ops.copy_pages((k, v), [pages - 1], [first - 1])
    assert bool((k[1, first - 1] == 3.0).all()) and bool((v[1, first - 1] == 4.0).all())


def test_another_stream_is_refused(ops):
    """As for every kernel that meets others in the device workspace."""
    from fllm_amd.kernels import KernelError
    case = plain.TreeCase([(20, 4)], 4, 2, 64, 16, torch.bfloat16, seed=1)
    check(ops, case)
    with torch.cuda.stream(torch.cuda.Stream()):
        with pytest.raises(KernelError, match="stream"):
            attend(ops, case, 0.1)
        with pytest.raises(KernelError, match="stream"):
            ops.copy_pages((torch.zeros((1, 4, 8), device="cuda"),), [0], [1])
    torch.cuda.synchronize()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("dim,rows", [(64, 0), (128, 0), (128, 64), (128, 128), (64, 64), (40, 0)])
@pytest.mark.parametrize("scale", [0.1, 2.0])
def test_scores_of_minus_infinity(ops, dim, rows, scale, dtype):
    """Keys that make a score minus infinity weigh nothing: whole blocks of them ahead of, between and behind others, with scales on both sides of 1."""
    case = plain.TreeCase([(700, 9), (90, 20)], 4, 2, dim, 16 if dim != 40 else 8, dtype, seed=dim)
    case.joint = case.joint.abs() + 0.1                # times minus infinity: that, in every lane
    case.joint *= 0.25
    none = {0: set(range(0, 300)) | set(range(420, 500)) | set(range(650, 700)), 1: set(range(0, 64)) | {92}}
    visible = case.visible
    case.visible = lambda s, i, window: [t for t in visible(s, i, window) if t not in none[s]]
    for s, slots in none.items():
        for t in slots:
            case.keys[s][t, :, 3] = float("-inf")
            case.put(s, t)
    ops.set_option("attention.tree_rows", rows)
    try:
        check(ops, case, scale=scale)
    finally:
        ops.set_option("attention.tree_rows", 0)


UNEVEN = [(3000, 6), (0, 1), (700, 35), (64, 0), (9, 33), (1500, 17)]


@pytest.mark.parametrize("heads,kv_heads", [(4, 1), (16, 2), (6, 3), (8, 4), (16, 8), (9, 9), (60, 20)])
@pytest.mark.parametrize("window", [0, 1000])
def test_uneven_requests_share_the_device(ops, heads, kv_heads, window):
    """The tiles of 128 rows cut the requests by their lengths: any number of key/value heads on the dies, requests without nodes, the same bits
    each time."""
    ops.set_option("attention.tree_rows", 128)
    try:
        case = plain.TreeCase(UNEVEN, heads, kv_heads, 128, 16, torch.bfloat16, seed=kv_heads)
        first = check(ops, case, window=window)
        for _ in range(3):
            again = attend(ops, case, 128 ** -0.5, window=window).cpu()
            assert bool((again == first).all())
        # bounds that the requests do not reach, and a bound on the nodes that cuts some of them
        check(ops, case, window=window, max_context=100000, max_nodes=64)
        short = attend(ops, case, 128 ** -0.5, window=window, max_nodes=7).cpu()
    finally:
        ops.set_option("attention.tree_rows", 0)
    for s, (kept, nodes) in enumerate(UNEVEN):
        row0 = int(case.seg_start[s])
        assert bool((short[row0 + 7: row0 + nodes] == 7.0).all())
        want, bound = case.expected(128 ** -0.5, window)
        assert plain.compare(short[row0: row0 + min(nodes, 7)], want[row0: row0 + min(nodes, 7)], bound[row0: row0 + min(nodes, 7)]) <= 1.0


@pytest.mark.parametrize("dim,rows", [(128, 128), (128, 64), (64, 64)])
def test_many_requests(ops, dim, rows):
    """More requests and key/value heads than workgroups at a time, one request much longer than the others."""
    ops.set_option("attention.tree_rows", rows)
    try:
        for requests in ([(5 * i % 90, 1 + i % 7) for i in range(70)], [(3 * i % 50, 1 + i % 9) for i in range(39)] + [(4500, 3)] + [(20, 0), (50, 2)]):
            case = plain.TreeCase(requests, 16, 8, dim, 16, torch.bfloat16, seed=len(requests))
            first = check(ops, case)
            assert bool((attend(ops, case, dim ** -0.5).cpu() == first).all())
    finally:
        ops.set_option("attention.tree_rows", 0)
