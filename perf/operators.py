"""Work on trees of drafted tokens over the paged cache, as cases that can be timed and compared with 64-bit arithmetic.

A request has `kept` tokens in its pages; a draft adds a tree of candidate continuations, whose nodes are computed together in one
step.  Node 0 is the request's newest token, every other node names its parent, a node of a lower number.  Node i lies in the slot
`kept + i` of the cache, its position (rotary, windows) is `kept` + its depth.  Four operators:

* `attend`  the nodes' attention over the kept tokens and their own ancestors (`Ops.tree_attention`);
* `follow`  which drafted tokens the model chose itself: the walk from the root (`Ops.follow_tree`);
* `move`    the walked nodes' keys and values move up behind the kept tokens, in every layer (`Ops.move_tokens`);
* `copy`    pages are copied in every layer, for a request that goes on in two ways (`Ops.copy_pages`).

With `own` false the operators are computed from elementary torch operations.
"""
import random

import torch

own = False

PAGE = 16
_DTYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}
_HEADS = {"8b": (32, 8, 128, 32), "1b": (32, 8, 64, 16), "70b": (64, 8, 128, 80)}      # heads, key/value heads, lanes, layers


def _attend(name, sizes, requests, nodes, kept, dtype="bfloat16", window=0, sinks=False, page=PAGE):
    heads, kv_heads, dim, _ = _HEADS[sizes] if isinstance(sizes, str) else sizes
    return dict(name=name, op="attend", heads=heads, kv_heads=kv_heads, dim=dim, requests=requests, nodes=nodes, kept=kept, dtype=dtype,
                window=window, sinks=sinks, page=page)


def _move(name, sizes, requests, nodes, accepted, kept, dtype="bfloat16", page=PAGE):
    _, kv_heads, dim, layers = _HEADS[sizes] if isinstance(sizes, str) else sizes
    return dict(name=name, op="move", kv_heads=kv_heads, dim=dim, layers=layers, requests=requests, nodes=nodes, accepted=accepted, kept=kept,
                dtype=dtype, page=page)


def _copy(name, sizes, pairs, pages, fork=False, dtype="bfloat16", page=PAGE):
    _, kv_heads, dim, layers = _HEADS[sizes] if isinstance(sizes, str) else sizes
    return dict(name=name, op="copy", kv_heads=kv_heads, dim=dim, layers=layers, pairs=pairs, pages=pages, fork=fork, dtype=dtype,
                page=page)


def listed():
    return [
        # one request, a small draft behind a short prompt: an interactive answer, where latency counts
        _attend("attend-one", "8b", requests=1, nodes=8, kept=1000),
        # a serving batch of ragged drafts (up to 26 nodes) at chat lengths
        _attend("attend-batch", "8b", requests=8, nodes=26, kept=2048),
        # two requests over long documents with wide trees; eight query heads a key/value head
        _attend("attend-long", "70b", requests=2, nodes=64, kept=32768),
        # a full batch with wide trees: the largest; heads of 64
        _attend("attend-many", "1b", requests=32, nodes=64, kept=6144),
        # windowed layers with sinks, drafts behind contexts far longer than the window, pages of 32 tokens
        _attend("attend-window", "8b", requests=16, nodes=24, kept=9000, window=1024, sinks=True, page=32),
        # the 32-bit path of the engine
        _attend("attend-float32", "1b", requests=4, nodes=13, kept=1500, dtype="float32"),
        # one request's draft of 32 nodes, five accepted, in all layers of a model
        _move("move-one", "8b", requests=1, nodes=32, accepted=5, kept=1003),
        # a batch with wide trees
        _move("move-batch", "1b", requests=48, nodes=64, accepted=9, kept=517),
        # an answer goes on in seven more ways: the tail page of its prompt is copied seven times
        _copy("copy-fork", "8b", pairs=7, pages=64, fork=True),
        # a cache is packed: hundreds of pages move
        _copy("copy-many", "1b", pairs=400, pages=1024),
        # one request's draft of 16 nodes
        _follow("follow-one", requests=1, nodes=16, deepest=8),
        # a full batch of wide trees
        _follow("follow-many", requests=256, nodes=64, deepest=16),
    ]


def _follow(name, requests, nodes, deepest):
    return dict(name=name, op="follow", requests=requests, nodes=nodes, deepest=deepest)


def _spread(rng, low, high):
    """A whole number between the two, even over its logarithm."""
    return max(low, min(high, round(low * (high / low) ** rng.random())))


def draw(rng):
    op = rng.choice(["attend", "attend", "attend", "move", "copy", "follow"])
    dtype = "float32" if rng.random() < 0.2 else "bfloat16"
    page = rng.choice([8, 16, 16, 32, 64])
    if op == "follow":
        nodes = _spread(rng, 2, 128)
        case = _follow(None, requests=_spread(rng, 1, 256), nodes=nodes, deepest=rng.randint(1, min(nodes, 24)))
    elif op == "attend":
        heads, kv_heads = rng.choice([(32, 8), (64, 8), (16, 16), (28, 4), (12, 2), (24, 8)])
        while True:
            case = _attend(None, (heads, kv_heads, rng.choice([64, 128]), 1), requests=_spread(rng, 1, 32), nodes=_spread(rng, 1, 96),
                           kept=_spread(rng, 1, 32768), dtype=dtype, window=rng.choice([0, 0, 0, _spread(rng, 16, 4096)]),
                           sinks=rng.random() < 0.3, page=page)
            if work(case)["flops"] <= 8e10 and work(case)["bytes"] <= 4e8:
                break
    elif op == "move":
        nodes = _spread(rng, 6, 96)
        while True:
            case = _move(None, (0, rng.choice([2, 4, 8]), rng.choice([64, 128]), rng.randint(1, 40)), requests=_spread(rng, 1, 48), nodes=nodes,
                         accepted=rng.randint(2, min(12, nodes // 2)), kept=_spread(rng, 1, 2048), dtype=dtype, page=page)
            if _cache_bytes(case, sum(_pages_of(case))) <= 2.5e9:
                break
    else:
        while True:
            pairs = _spread(rng, 1, 400)
            case = _copy(None, (0, rng.choice([2, 4, 8]), rng.choice([64, 128]), rng.randint(1, 40)), pairs=pairs, pages=2 * pairs + rng.randint(1, 40),
                         fork=rng.random() < 0.4, dtype=dtype, page=page)
            if _cache_bytes(case, case["pages"]) <= 1e9 and work(case)["bytes"] <= 4e8:
                break
    del case["name"]
    return case


# ---- what a case comes to ------------------------------------------------------------------------------------------------
def _lengths(case):
    """(kept tokens, nodes) of every request: the first as the case says, the others between half of that and that."""
    rng = random.Random(case["requests"] * 1009 + case["nodes"])
    out = []
    for r in range(case["requests"]):
        share = 1.0 if r == 0 else 0.5 + 0.5 * rng.random()
        kept = case.get("kept", 0)
        out.append((max(min(kept, 1), round(kept * share)), max(1, round(case["nodes"] * (1.0 if r == 0 else 0.5 + 0.5 * rng.random())))))
    return out


def _pages_of(case):
    return [-(-(kept + nodes) // case["page"]) for kept, nodes in _lengths(case)]


def _size(case):
    return 4 if case["dtype"] == "float32" else 2


def _cache_bytes(case, pages):
    return 2 * case["layers"] * pages * case["kv_heads"] * case["dim"] * case["page"] * _size(case)


def _paths(case):
    """Per request the rising nodes that are kept; those behind the root have numbers beyond the places they move to, as in a
    tree that is numbered level by level and wider than it is deep."""
    rng = random.Random(case["nodes"] * 7919 + case["accepted"])
    out = []
    for _, nodes in _lengths(case):
        length = max(1, min(case["accepted"], (nodes + 1) // 2))
        out.append([0] + sorted(rng.sample(range(length, nodes), length - 1)))
    return out


def work(case):
    """A tree's rows are counted with the kept tokens and themselves; their ancestors, a few, are left out."""
    if case["op"] == "follow":
        nodes = sum(n for _, n in _lengths(case))
        return {"bytes": 4 * (3 * nodes + case["requests"] * (3 + case["deepest"])), "flops": nodes}
    if case["op"] == "copy":
        return {"bytes": _cache_bytes(case, case["pairs"] + (1 if case["fork"] else case["pairs"])), "flops": 0}
    if case["op"] == "move":
        moved = sum(sum(1 for i, n in enumerate(path) if i != n) for path in _paths(case))
        return {"bytes": 2 * 2 * case["layers"] * moved * case["kv_heads"] * case["dim"] * _size(case), "flops": 0}
    tokens = keys = rows = 0
    for kept, nodes in _lengths(case):
        reach = min(kept, case["window"] - 1) if case["window"] else kept
        tokens += reach + nodes
        keys += nodes * (reach + 1)
        rows += nodes
    return {"bytes": _size(case) * case["dim"] * (2 * tokens * case["kv_heads"] + 2 * rows * case["heads"]),
            "flops": 4 * keys * case["heads"] * case["dim"]}


# ---- inputs ---------------------------------------------------------------------------------------------------------------
def _tree(nodes, deepest, rng):
    """Parents and depths of a tree that is numbered level by level."""
    deepest = max(1, min(deepest, nodes))
    depths = [0] + sorted(list(range(1, deepest)) + [rng.randint(1, max(1, deepest - 1)) for _ in range(nodes - deepest)])
    depths = depths[:nodes]
    levels = {}
    for i, d in enumerate(depths):
        levels.setdefault(d, []).append(i)
    parents = [-1 if d == 0 else rng.choice(levels[d - 1]) for d in depths]
    return parents, depths


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _cuts(lengths):
    cuts = [0]
    for _, nodes in lengths:
        cuts.append(cuts[-1] + nodes)
    return cuts


def prepare(case, seed):
    rng = random.Random(seed)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    state = {"case": case}
    if own:
        from fllm_amd.kernels import Ops
        state["ops"] = Ops()
    if case["op"] == "copy":
        shape = (case["layers"], case["pages"], case["kv_heads"])
        sources = 1 if case["fork"] else case["pairs"]      # a fork copies one page to many, a packing each page once
        chosen = rng.sample(range(case["pages"]), sources + case["pairs"])
        state["source"], state["target"] = [chosen[i % sources] for i in range(case["pairs"])], chosen[sources:]
        state["k"], state["v"] = _stores(case, shape, gen)
        return state
    lengths = _lengths(case)
    cuts = _cuts(lengths)
    state["lengths"], state["cuts"], state["seg_start"] = lengths, cuts, _int32(cuts)
    if case["op"] == "follow":
        parents, drafted, chosen = [], [], []
        for _, nodes in lengths:
            mine, depths = _tree(nodes, case["deepest"], rng)
            tokens = [rng.randrange(128256) for _ in range(nodes)]
            picks = [rng.randrange(128256) for _ in range(nodes)]
            for i in range(nodes):      # most nodes' choice is one of their children, where they have some
                children = [c for c in range(i + 1, nodes) if mine[c] == i]
                if children and rng.random() < 0.8:
                    picks[i] = tokens[rng.choice(children)]
            parents += mine
            drafted += tokens
            chosen += picks
        state["parents"], state["drafted"], state["chosen"] = _int32(parents), _int32(drafted), _int32(chosen)
        state["path"] = torch.empty((case["requests"], case["deepest"]), dtype=torch.int32, device="cuda")
        state["length"] = torch.empty(case["requests"], dtype=torch.int32, device="cuda")
        state["newest"] = torch.empty(case["requests"], dtype=torch.int32, device="cuda")
        return state
    pages_of = _pages_of(case)
    total = sum(pages_of) + 1
    order = list(range(total))
    rng.shuffle(order)
    width = max(pages_of)
    table, at = [], 0
    for pages in pages_of:
        table.append(order[at:at + pages] + [-1] * (width - pages))
        at += pages
    state["host_table"], state["tables"] = table, _int32(table)
    state["kept"] = _int32([kept for kept, _ in lengths])
    layers = case.get("layers", 1)
    state["k"], state["v"] = _stores(case, (layers, total, case["kv_heads"]), gen)
    if case["op"] == "move":
        paths = _paths(case)
        state["path"] = _int32([path + [-1] * (case["accepted"] - len(path)) for path in paths])
        state["length"] = _int32([len(path) for path in paths])
        state["paths"] = paths
        return state
    rows, heads, dim = cuts[-1], case["heads"], case["dim"]
    words = (max(n for _, n in lengths) + 63) // 64
    seen, positions = [], []
    for kept, nodes in lengths:
        parents, depths = _tree(nodes, rng.randint(1, 12), rng)
        bits = []
        for i, p in enumerate(parents):
            bits.append((bits[p] if p >= 0 else 0) | 1 << i)
        for b in bits:
            seen.append([(b >> 64 * w & (1 << 64) - 1) - (1 << 64 if b >> 64 * w + 63 & 1 else 0) for w in range(words)])
        positions += [kept + d for d in depths]
    state["seen"] = torch.tensor(seen, dtype=torch.int64, device="cuda")
    state["positions"] = _int32(positions)
    # the queries as the fused product leaves them: the first columns of a wider matrix
    joint = torch.randn((rows, (heads + 2 * case["kv_heads"]) * dim), generator=gen, device="cuda").to(_DTYPES[case["dtype"]])
    state["q"] = joint[:, : heads * dim]
    state["sinks"] = torch.randn(heads, generator=gen, device="cuda") if case["sinks"] else None
    state["out"] = torch.empty((rows, heads * dim), dtype=_DTYPES[case["dtype"]], device="cuda")
    state["most"] = max(n for _, n in lengths)
    state["context"] = max(kept + n for kept, n in lengths)
    return state


def _stores(case, shape, gen):
    """Keys [layers, pages, key/value heads, lanes / 8, tokens, 8] and values [.., lanes, tokens]."""
    dim, page, dtype = case["dim"], case["page"], _DTYPES[case["dtype"]]
    return (torch.randn((*shape, dim // 8, page, 8), generator=gen, device="cuda", dtype=dtype),
            torch.randn((*shape, dim, page), generator=gen, device="cuda", dtype=dtype))


# ---- a pass ---------------------------------------------------------------------------------------------------------------
def run(state):
    case = state["case"]
    return {"attend": _run_attend, "move": _run_move, "copy": _run_copy, "follow": _run_follow}[case["op"]](case, state)


def _run_copy(case, state):
    if own:
        state["ops"].copy_pages((state["k"], state["v"]), state["source"], state["target"])
    else:
        source = torch.tensor(state["source"], device="cuda")
        target = torch.tensor(state["target"], device="cuda")
        for store in (state["k"], state["v"]):
            store.index_copy_(1, target, store.index_select(1, source))
    return state["k"], state["v"]


def _run_move(case, state):
    if own:
        state["ops"].move_tokens(state["k"], state["v"], state["tables"], state["kept"], state["path"], state["length"])
        return state["k"], state["v"]
    page = case["page"]
    places = torch.arange(case["accepted"], device="cuda")
    live = places[None, :] < state["length"][:, None]
    base = state["kept"].long()[:, None]
    source, target = (base + state["path"].long())[live], (base + places[None, :])[live]
    request = torch.arange(case["requests"], device="cuda")[:, None].expand_as(live)[live]
    tables = state["tables"].long()
    source_page, target_page = tables[request, source // page], tables[request, target // page]
    for layer in range(case["layers"]):
        k, v = state["k"][layer], state["v"][layer]
        k[target_page, :, :, target % page] = k[source_page, :, :, source % page]
        v[target_page, :, :, target % page] = v[source_page, :, :, source % page]
    return state["k"], state["v"]


def _run_follow(case, state):
    if own:
        state["ops"].follow_tree(state["drafted"], state["parents"], state["seg_start"], state["chosen"], state["path"], state["length"],
                                 state["newest"])
        return state["path"], state["length"], state["newest"]
    starts, ends = state["seg_start"][:-1].long(), state["seg_start"][1:].long()
    most = max(n for _, n in state["lengths"])
    numbers = torch.arange(most, device="cuda")
    rows = starts[:, None] + numbers[None, :]
    inside = rows < ends[:, None]
    rows = torch.where(inside, rows, torch.zeros_like(rows))
    parents = torch.where(inside, state["parents"].long()[rows], torch.full_like(rows, -2))
    drafted = state["drafted"].long()[rows]
    at = torch.zeros_like(starts)
    going = torch.ones_like(starts, dtype=torch.bool)
    path = torch.full((case["requests"], case["deepest"]), -1, dtype=torch.int32, device="cuda")
    path[:, 0] = 0
    length = torch.ones_like(starts)
    for step in range(1, case["deepest"]):
        picked = state["chosen"].long()[starts + at]
        fits = (parents == at[:, None]) & (drafted == picked[:, None]) & (numbers[None, :] > 0)
        child = torch.where(fits, numbers[None, :], torch.full_like(rows, most)).amin(dim=1)
        going = going & (child < most)
        at = torch.where(going, child, at)
        path[:, step] = torch.where(going, child, torch.full_like(child, -1)).int()
        length = length + going.long()
    return path, length.int(), state["chosen"][starts + at]


def _visible(state, s, positions, seen):
    """[nodes, kept + nodes]: what the nodes of request s see."""
    case = state["case"]
    kept, nodes = state["lengths"][s]
    first, last = state["cuts"][s], state["cuts"][s + 1]
    mine = positions[first:last].long()
    numbers = torch.arange(nodes, device="cuda")
    own_nodes = (seen[first:last][:, numbers // 64] >> (numbers % 64)[None, :]) & 1
    keys = torch.cat([torch.arange(kept, device="cuda"), mine])
    visible = torch.cat([torch.ones((nodes, kept), dtype=torch.bool, device="cuda"), own_nodes.bool()], dim=1)
    if case["window"]:
        visible &= keys[None, :] > mine[:, None] - case["window"]
    return visible


def _run_attend(case, state):
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    if own:
        return state["ops"].tree_attention(state["q"], state["k"][0], state["v"][0], state["tables"], state["positions"], state["seg_start"],
                                           state["kept"], state["seen"], state["out"], heads, kv_heads, dim, case["page"], dim ** -0.5,
                                           state["context"], window=case["window"] or None, sinks=state["sinks"], max_nodes=state["most"])
    group = heads // kv_heads
    for s, (kept, nodes) in enumerate(state["lengths"]):
        n, first, last = kept + nodes, state["cuts"][s], state["cuts"][s + 1]
        pages = state["tables"][s, : -(-n // case["page"])].long()
        k = state["k"][0][pages].permute(1, 2, 4, 0, 3).reshape(kv_heads, dim, -1)[:, :, :n].float().contiguous()
        v = state["v"][0][pages].permute(1, 0, 3, 2).reshape(kv_heads, -1, dim)[:, :n].float().contiguous()
        q = state["q"][first:last].float().reshape(nodes, kv_heads, group, dim).permute(1, 2, 0, 3).reshape(kv_heads, group * nodes, dim)
        scores = torch.bmm(q, k).reshape(kv_heads, group, nodes, n) * dim ** -0.5
        scores = scores.masked_fill(~_visible(state, s, state["positions"], state["seen"]), float("-inf"))
        top = scores.amax(dim=-1, keepdim=True)
        if state["sinks"] is not None:
            sinks = state["sinks"].reshape(kv_heads, group, 1, 1)
            top = torch.maximum(top, sinks)
        weights = torch.exp(scores - top)
        below = weights.sum(dim=-1, keepdim=True)
        if state["sinks"] is not None:
            below = below + torch.exp(sinks - top)
        mixed = torch.bmm(weights.reshape(kv_heads, group * nodes, n), v).reshape(kv_heads, group, nodes, dim) / below
        state["out"][first:last] = mixed.permute(2, 0, 1, 3).reshape(nodes, heads * dim).to(state["out"].dtype)
    return state["out"]


# ---- the definition in 64 bits --------------------------------------------------------------------------------------------
def exact(case, seed):
    """Attention head by head over one token after another of the pages' order; a copied value is itself."""
    if case["op"] == "follow":
        return None
    state = prepare(case, seed)
    if case["op"] != "attend":
        before, after = (state["k"], state["v"]), (state["k"].double(), state["v"].double())
        for old, new in zip(before, after):
            if case["op"] == "copy":
                for source, target in zip(state["source"], state["target"]):
                    new[:, target] = old[:, source]
                continue
            for (kept, _), table, path in zip(state["lengths"], state["host_table"], state["paths"]):
                for i, n in enumerate(path):
                    (from_page, at), (to_page, to) = divmod(kept + n, case["page"]), divmod(kept + i, case["page"])
                    if old.dim() == 6:
                        new[:, table[to_page], :, :, to] = old[:, table[from_page], :, :, at].double()
                    else:
                        new[:, table[to_page], ..., to] = old[:, table[from_page], ..., at].double()
        return after
    heads, dim, page = case["heads"], case["dim"], case["page"]
    out = torch.zeros((state["cuts"][-1], heads, dim), dtype=torch.float64, device="cuda")
    for s, (kept, nodes) in enumerate(state["lengths"]):
        first, last = state["cuts"][s], state["cuts"][s + 1]
        slots = torch.arange(kept + nodes, device="cuda")
        pages = state["tables"][s].long()[slots // page]
        bits = (state["seen"][first:last, :, None] >> torch.arange(64, device="cuda")) & 1
        hidden = torch.zeros((nodes, kept + nodes), dtype=torch.bool, device="cuda")
        hidden[:, kept:] = bits.reshape(nodes, -1)[:, :nodes] == 0
        if case["window"]:
            places = torch.cat([slots[:kept], state["positions"][first:last].long()])
            hidden |= state["positions"][first:last, None] - places[None, :] >= case["window"]
        for h in range(heads):
            g = h // (heads // case["kv_heads"])
            keys = state["k"][0][pages, g, :, slots % page].reshape(-1, dim).double()
            values = state["v"][0][pages, g, :, slots % page].double()
            z = state["q"][first:last, h * dim:(h + 1) * dim].double() @ keys.t().contiguous() / dim ** 0.5
            z[hidden] = float("-inf")
            if state["sinks"] is not None:
                z = torch.cat([z, state["sinks"][h].double().expand(nodes, 1)], dim=1)
                values = torch.cat([values, torch.zeros((1, dim), dtype=torch.float64, device="cuda")])
            out[first:last, h] = torch.softmax(z, dim=1) @ values
    return out.reshape(-1, heads * dim)
