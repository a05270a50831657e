"""Trees of drafted tokens without a GPU: the interface's version, the rows of a tree, what the entry points refuse before a launch."""
import ctypes
import hashlib
import os
import random
import re

import pytest

import draft_reference as plain
from fllm_amd.kernels import load_library, tree_rows

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

# version -> the first of the digest of csrc/draft_api.h's declarations (comments and spaces aside).  An entry point that is added, taken away
# or given other arguments needs a new version in csrc/tree_attention.hip and kernels/__init__.py, and a line here.
DECLARATIONS = {1: "0d14cc4899e33c87"}


def source(*path):
    with open(os.path.join(ROOT, "fllm_amd", *path)) as fh:
        return fh.read()


def test_the_version_is_that_of_the_entry_points():
    text = re.sub(r"//[^\n]*|/\*.*?\*/", " ", source("csrc", "draft_api.h"), flags=re.S)
    found = sorted(" ".join(d.split()) for d in re.findall(r"\b[\w \*]+\bfllm_\w+\s*\([^;{]*\)\s*;", text))
    assert len(found) == 6
    version = int(re.search(r"fllm_draft_abi_version\(void\) \{ return (\d+); \}", source("csrc", "tree_attention.hip")).group(1))
    assert int(re.search(r"^DRAFT_ABI_VERSION = (\d+)", source("kernels", "__init__.py"), re.M).group(1)) == version
    assert hashlib.sha256("\n".join(found).encode()).hexdigest()[:16] == DECLARATIONS.get(version)


@pytest.mark.parametrize("nodes", [0, 1, 2, 63, 64, 65, 200])
def test_the_rows_of_a_tree(nodes):
    parents = plain.random_tree(nodes, random.Random(nodes)) if nodes else []
    depths, seen = tree_rows(parents)
    assert len(depths) == len(seen) == nodes
    for i in range(nodes):
        line, at = {i}, i
        while at:
            at = parents[at]
            line.add(at)
        assert depths[i] == len(line) - 1
        assert seen[i] == plain.signed_words(sum(1 << j for j in line), max(1, -(-nodes // 64)))
        assert all(-(1 << 63) <= w < 1 << 63 for w in seen[i])
    assert tree_rows(parents, 5)[1] == [row + [0] * (5 - len(row)) for row in seen]


def test_a_tree_that_is_none():
    for parents in ([-1, 1], [-1, 0, 2], [-1, -1], [-1, 0, 5]):
        with pytest.raises(ValueError, match="lower number"):
            tree_rows(parents)
    with pytest.raises(ValueError, match="more than 1 words"):
        tree_rows([0] * 65, 1)


# a call of every entry point that is right, and what is refused in its place; nothing is launched for sizes of zero
ATTEND = dict(q=0, q_stride=128, k=0, v=0, tables=0, table_stride=4, row_pos=0, seg_start=0, num_segs=1, kept=0, seen=0, words=1, out=0, rows=0,
              heads=2, kv_heads=1, head_dim=64, v_dim=64, page_size=16, num_pages=9, scale=1.0, window=0, key_chunk=8, sinks=0, dtype=1,
              max_nodes=1, max_context=10, stream=0)
MOVE = dict(k=0, v=1, layers=0, num_pages=9, kv_heads=1, k_dim=64, v_dim=64, page_size=16, key_chunk=8, elem_bytes=2, tables=0, table_stride=4,
            num_segs=1, kept=0, path=0, max_path=3, length=0, stream=0)
FOLLOW = dict(drafted=0, parents=0, seg_start=0, num_segs=0, chosen=0, rows=0, path=0, max_path=1, length=0, newest=0, stream=0)


@pytest.mark.parametrize("name,right,wrong,message", [
    ("fllm_tree_attention", ATTEND, dict(heads=0), "bad sizes"), ("fllm_tree_attention", ATTEND, dict(rows=-1), "bad sizes"),
    ("fllm_tree_attention", ATTEND, dict(page_size=0), "bad sizes"), ("fllm_tree_attention", ATTEND, dict(num_pages=0), "bad sizes"),
    ("fllm_tree_attention", ATTEND, dict(table_stride=0), "bad sizes"), ("fllm_tree_attention", ATTEND, dict(words=0), "words"),
    ("fllm_tree_attention", ATTEND, dict(window=-1), "window"), ("fllm_tree_attention", ATTEND, dict(max_nodes=-1), "bounds"),
    ("fllm_tree_attention", ATTEND, dict(kv_heads=3), "not a multiple"), ("fllm_tree_attention", ATTEND, dict(key_chunk=7), "chunks of 7"),
    ("fllm_tree_attention", ATTEND, dict(q_stride=100), "q_stride"), ("fllm_tree_attention", ATTEND, dict(dtype=2), "dtype"),
    ("fllm_tree_attention", ATTEND, dict(v_dim=513), "too wide"), ("fllm_tree_attention", ATTEND, dict(heads=70000, kv_heads=1, q_stride=70000 * 64), "too many heads"),
    ("fllm_move_tokens", MOVE, dict(page_size=0), "bad sizes"), ("fllm_move_tokens", MOVE, dict(max_path=0), "bad sizes"),
    ("fllm_move_tokens", MOVE, dict(key_chunk=5), "chunks of 5"), ("fllm_move_tokens", MOVE, dict(elem_bytes=8), "8 bytes"),
    ("fllm_move_tokens", MOVE, dict(v=0), "values are missing"), ("fllm_move_tokens", MOVE, dict(num_pages=0), "bad sizes"),
    ("fllm_follow_tree", FOLLOW, dict(max_path=0), "bad sizes"), ("fllm_follow_tree", FOLLOW, dict(rows=-1), "bad sizes"),
])
def test_what_is_refused(name, right, wrong, message):
    lib = load_library()
    call = getattr(lib, name)
    assert call(*right.values()) == 0
    assert call(*dict(right, **wrong).values()) != 0
    assert message in lib.fllm_last_error().decode()


def test_pages_that_are_not_copied():
    """Pages outside the store, and a page onto itself, are refused before anything is launched."""
    lib = load_library()
    i64, i32 = ctypes.c_int64, ctypes.c_int32
    stores, layers, pages, size = (ctypes.c_void_p * 1)(0), (i64 * 1)(0), (i64 * 1)(10), (i64 * 1)(64)
    call = lambda source, target, stores_given=1: lib.fllm_copy_pages(stores, layers, pages, size, stores_given, (i32 * 1)(source), (i32 * 1)(target), 1, None)
    assert call(1, 2) == 0             # a store without layers: nothing to do
    for source, target in ((10, 1), (1, 10), (-1, 1), (1, -1), (3, 3)):
        assert call(source, target) != 0 and "of 10" in lib.fllm_last_error().decode()
    assert call(1, 2, 9) != 0 and "9 stores" in lib.fllm_last_error().decode()


# ---- a request that goes on in two ways -------------------------------------------------------------------------------------
def group(window=None, page_size=4):
    from fllm_amd.cache import GroupSpec
    return GroupSpec(entries=(0,), kv_heads=2, k_dim=16, v_dim=16, window=window, page_size=page_size)


def test_a_fork_holds_full_pages_and_copies_the_last():
    from fllm_amd.cache import CacheManager, OutOfPages
    m = CacheManager([group(), group(window=6)], [6, 6], max_requests=4)
    m.add_request("a"), m.reserve("a", 14), m.commit("a", 10)
    m.add_request("b")
    copies = m.fork_request("a", "b")
    assert m.length("b") == 10 and len(m.table("b", 0)) == 3 and len(m.table("a", 0)) == 4
    assert m.table("b", 0)[:2] == m.table("a", 0)[:2] and copies[0] == (m.table("a", 0)[2], m.table("b", 0)[2]) and copies[0][0] != copies[0][1]
    assert m.table("b", 1)[0] == m.table("a", 1)[0] == -1 and m.table("b", 1)[1] == m.table("a", 1)[1] and copies[1][0] == m.table("a", 1)[2]
    m.check_invariants()
    m.add_request("c")
    with pytest.raises(OutOfPages):                       # a group without a page: nothing is changed
        m.reserve("a", 17), m.fork_request("a", "c")
    assert m.length("c") == 0 and m.table("c", 0) == [] and m.table("c", 1) == []
    m.check_invariants()
    m.free_request("a")
    m.reserve("b", 11), m.commit("b", 1)
    m.check_invariants()
    for wrong in (("b", "b"), ("c", "b")):
        with pytest.raises(ValueError):
            m.fork_request(*wrong)
    with pytest.raises(KeyError):
        m.fork_request("nobody", "c")
    m.free_request("b"), m.free_request("c")
    assert m.free_pages(0) == 6 and m.free_pages(1) == 6
    m.check_invariants()


def test_a_fork_on_a_pages_edge_and_of_nothing():
    from fllm_amd.cache import CacheManager
    m = CacheManager([group()], [4], max_requests=3)
    m.add_request("a"), m.reserve("a", 8), m.commit("a", 8)
    m.add_request("b")
    assert m.fork_request("a", "b") == [None] and m.table("b", 0) == m.table("a", 0) and m.free_pages() == 2
    m.add_request("c"), m.free_request("b"), m.add_request("b")
    assert m.fork_request("c", "b") == [None] and m.length("b") == 0
    m.check_invariants()


@pytest.mark.parametrize("seed", range(6))
def test_forks_in_random_orders_keep_the_books(seed):
    from fllm_amd.cache import CacheManager, OutOfPages
    rng = random.Random(seed)
    prefixes = seed % 2 == 0
    m = CacheManager([group()] if prefixes else [group(), group(window=7)], [30] if prefixes else [30, 30], max_requests=6)
    if prefixes:
        m.enable_prefix_cache()
    tokens, number, forks = {}, 0, 0
    for _ in range(500):
        what = rng.random()
        if what < 0.2 and len(tokens) < 6:
            m.add_request(number)
            tokens[number] = [rng.randrange(2) for _ in range(40)]
            if prefixes:
                m.adopt_prefix(number, tokens[number][:20])
            number += 1
        elif what < 0.45 and tokens and len(tokens) < 6:
            src = rng.choice(list(tokens))
            m.add_request(number)
            try:
                copies = m.fork_request(src, number)
                tokens[number] = list(tokens[src])
                forks += 1
                assert [c is not None for c in copies] == [m.length(src) % 4 != 0] * len(m.groups)
            except OutOfPages:
                m.free_request(number)
            number += 1
        elif what < 0.85 and tokens:
            r = rng.choice(list(tokens))
            n = min(rng.randint(1, 9), 40 - m.length(r))
            if n and m.can_reserve(r, m.length(r) + n):
                m.reserve(r, m.length(r) + n)
                m.commit(r, rng.randint(0, n))
                if rng.random() < 0.5:
                    m.trim(r, m.length(r))
                if prefixes:
                    m.remember_prefix(r, tokens[r][: m.length(r)])
        elif tokens:
            r = rng.choice(list(tokens))
            m.free_request(r)
            del tokens[r]
        m.check_invariants()
    assert forks > 10
    for r in tokens:
        m.free_request(r)
    m.check_invariants()
