"""Steps on trees of drafted tokens and forks on the CPU, with plain kernels: what a request holds after a tree that was left behind, a step that
failed part of the way, a request that ended meanwhile."""
import random

import numpy as np
import pytest
import torch

import draft_reference as plain
import plain_llama
import tiny_configs as tc
from draft_ops import PlainTreeOps
from fllm_amd.engine import ModelRunner, StepEntry, StepError, TreeEntry
from fllm_amd.registry import model_spec_from_config
from fllm_amd.weights import random_tensors


def runner_of(name, max_tokens=400, ops=None, **more):
    cfg = tc.CONFIGS[name]
    _, spec = model_spec_from_config(cfg)
    tensors = random_tensors(spec, 7, torch.float32, with_optional=(name == "C"))
    args = dict(dtype="float32", device="cpu", page_size=tc.PAGE_SIZES[name], max_tokens=max_tokens, max_requests=8)
    return ModelRunner(spec, tensors, ops=ops or PlainTreeOps(), **dict(args, **more)), cfg, tc.to_float64(tensors)


def free_pages(runner):
    return [runner.cache.free_pages(g) for g in range(len(runner.cache.groups))]


def tree_of(req_id, nodes, vocab, seed=1):
    rng = random.Random(seed)
    return TreeEntry(req_id, [rng.randrange(vocab) for _ in range(nodes)], plain.random_tree(nodes, rng))


def own_tokens(cfg, weights, tokens, count):
    """Greedy continuations of `tokens`."""
    out = []
    for _ in range(count):
        out.append(int(np.argmax(plain_llama.forward(cfg, weights, tokens + out)[-1])))
    return out


def next_logits(cfg, weights, tokens, got):
    want = plain_llama.forward(cfg, weights, tokens)[-1]
    assert np.abs(got.numpy() - want).max() <= 2e-5 * np.abs(want).max()


@pytest.mark.parametrize("name", ["A", "E"])
def test_a_tree_and_what_is_kept_of_it(name):
    """Logits of every node, and the next step on what was kept, against the plain implementation."""
    runner, cfg, weights = runner_of(name)
    prompt = tc.random_ids(45, cfg["vocab_size"], 1)
    newest, *more = own_tokens(cfg, weights, prompt, 4)
    runner.step([StepEntry("a", prompt)])
    entry = TreeEntry("a", [newest, 3, more[0], 5, more[1], 7], [-1, 0, 0, 2, 2, 4])
    logits = runner.step_tree([entry])
    for node, line in enumerate(([], [1], [2], [2, 3], [2, 4], [2, 4, 5])):
        next_logits(cfg, weights, prompt + [newest] + [entry.tokens[i] for i in line], logits[node])
    (path, token), = runner.keep_tree(logits.argmax(dim=1).int())
    assert (path, token) == ([0, 2, 4], more[2]) and runner.length("a") == 48
    next_logits(cfg, weights, prompt + [newest] + more, runner.step([StepEntry("a", [token], want=(0,))])[0])
    runner.cache.check_invariants()


def failing(runner, monkeypatch, when):
    """The next forward passes of the model fail, ahead of or behind their launches."""
    real = runner.model.forward

    def forward(ctx):
        if when == "after":
            real(ctx)
        raise MemoryError("no room for the logits")
    monkeypatch.setattr(runner.model, "forward", forward)


@pytest.mark.parametrize("when", ["before", "after"])
def test_a_tree_step_that_fails_leaves_the_trees_before_it_behind(monkeypatch, when):
    """Its nodes may lie in the slots of theirs."""
    runner, cfg, weights = runner_of("A")
    prompt = tc.random_ids(21, cfg["vocab_size"], 2)
    runner.step([StepEntry("a", prompt)])
    entry = tree_of("a", 6, cfg["vocab_size"])
    chosen = runner.step_tree([entry]).argmax(dim=1).int()
    with monkeypatch.context() as patch:
        failing(runner, patch, when)
        with pytest.raises(MemoryError):
            runner.step_tree([tree_of("a", 9, cfg["vocab_size"], seed=5)])
    with pytest.raises(StepError, match="follows a step_tree"):
        runner.keep_tree(chosen)
    assert runner.length("a") == 21
    runner.cache.check_invariants()
    next_logits(cfg, weights, prompt + [9], runner.step([StepEntry("a", [9], want=(0,))])[0])


def test_keeping_that_fails_part_of_the_way_is_not_done_twice():
    """A path that has been moved in one group's pages and is moved again takes other nodes' keys and values."""
    class Ops(PlainTreeOps):
        calls, fail_at, refuse = 0, None, False

        def follow_tree(self, *args):
            if self.refuse:
                raise ValueError("refused")
            super().follow_tree(*args)

        def move_tokens(self, *args):
            self.calls += 1
            if self.calls == self.fail_at:
                raise MemoryError("a launch that failed")
            super().move_tokens(*args)

    ops = Ops()
    runner, cfg, weights = runner_of("E", ops=ops)
    assert len(runner.cache.groups) == 2
    prompt = tc.random_ids(30, cfg["vocab_size"], 3)
    newest, *more = own_tokens(cfg, weights, prompt, 4)
    entry = TreeEntry("a", [newest, 3, more[0], 5, more[1]], [-1, 0, 0, 2, 2])
    runner.step([StepEntry("a", prompt)])
    chosen = runner.step_tree([entry]).argmax(dim=1).int()
    ops.refuse = True
    with pytest.raises(ValueError):
        runner.keep_tree(chosen)                  # refused ahead of the first move: the trees are still there
    ops.refuse, ops.fail_at = False, 2
    with pytest.raises(MemoryError):
        runner.keep_tree(chosen)
    with pytest.raises(StepError, match="follows a step_tree"):
        runner.keep_tree(chosen)
    assert runner.length("a") == 30 and ops.calls == 2
    chosen = runner.step_tree([entry]).argmax(dim=1).int()
    (path, token), = runner.keep_tree(chosen)
    assert (path, token) == ([0, 2, 4], more[2])
    next_logits(cfg, weights, prompt + [newest] + more, runner.step([StepEntry("a", [token], want=(0,))])[0])
    runner.cache.check_invariants()


@pytest.mark.parametrize("what", ["pages", "state"])
def test_a_fork_whose_copies_fail_leaves_nothing(monkeypatch, what):
    """The request that was to go on holds a last page that nobody filled."""
    class Ops(PlainTreeOps):
        fails = False

        def copy_pages(self, *args):
            if self.fails:
                raise MemoryError("a launch that failed")
            super().copy_pages(*args)

    ops = Ops()
    runner, cfg, weights = runner_of("E", ops=ops)
    prompt = tc.random_ids(37, cfg["vocab_size"], 4)
    runner.step([StepEntry("a", prompt)])
    before = free_pages(runner), runner.cache.free_slots()

    def arenas():
        raise MemoryError("a copy that failed")
    ops.fails = what == "pages"
    with monkeypatch.context() as patch:
        if what == "state":
            patch.setattr(runner.model, "state_arenas", arenas)
        with pytest.raises(MemoryError):
            runner.fork_request("a", "b")
    assert runner.cache.requests() == ["a"] and (free_pages(runner), runner.cache.free_slots()) == before
    ops.fails = False
    with pytest.raises(ValueError):
        runner.fork_request("a", "a")
    assert runner.cache.requests() == ["a"]       # a name that is taken is not given up
    runner.fork_request("a", "b")
    got = runner.step([StepEntry("a", [3], want=(0,)), StepEntry("b", [8], want=(0,))])
    next_logits(cfg, weights, prompt + [3], got[0])
    next_logits(cfg, weights, prompt + [8], got[1])
    runner.cache.check_invariants()


@pytest.mark.parametrize("name", ["A", "E"])
@pytest.mark.parametrize("how", ["step", "step of another", "step_tree", "step_tree of another", "failing step_tree", "free", "free another", "keep"])
def test_trees_that_are_left_behind_give_their_pages_back(monkeypatch, name, how):
    runner, cfg, weights = runner_of(name)
    vocab = cfg["vocab_size"]
    prompts = {r: tc.random_ids(n, vocab, n) for r, n in (("a", 17), ("b", 30), ("c", 5))}
    runner.step([StepEntry(r, p) for r, p in prompts.items()])
    before = free_pages(runner)
    chosen = runner.step_tree([tree_of("a", 40, vocab), tree_of("b", 40, vocab)]).argmax(dim=1).int()
    assert all(now < then for now, then in zip(free_pages(runner), before))
    if how == "step":
        runner.step([StepEntry("a", [3])])
    elif how == "step of another":
        runner.step([StepEntry("c", [3])])
    elif how == "step_tree":
        runner.step_tree([tree_of("a", 2, vocab)])
    elif how == "step_tree of another":
        runner.step_tree([tree_of("c", 2, vocab)])
    elif how == "failing step_tree":
        with monkeypatch.context() as patch:
            failing(runner, patch, "after")
            with pytest.raises(MemoryError):
                runner.step_tree([tree_of("a", 50, vocab), tree_of("c", 40, vocab)])
    elif how == "free":
        runner.free_request("a")
        runner.step([StepEntry("c", [3])])
    elif how == "free another":
        runner.free_request("c")
        runner.step([StepEntry("b", [3])])
    else:
        runner.keep_tree(chosen)
    runner.cache.check_invariants()
    size = tc.PAGE_SIZES[name]
    for r in runner.cache.requests():              # no more pages than the tokens of each need, and those of a tree that is still there
        more = 2 if how == "step_tree" and r == "a" or how == "step_tree of another" and r == "c" else 0
        for g in range(len(runner.cache.groups)):
            assert len(runner.cache.table(r, g)) == -(-(runner.length(r) + more) // size), (r, g)
    if "free" not in how and how != "keep":
        tail = {"a": [3] if how == "step" else [], "b": [], "c": [3] if how == "step of another" else []}
        got = runner.step([StepEntry(r, [8], want=(0,)) for r in prompts])
        for row, (r, p) in zip(got, prompts.items()):
            next_logits(cfg, weights, p + tail[r] + [8], row)


def test_a_step_gets_the_pages_of_trees_that_it_leaves_behind():
    from fllm_amd.cache import OutOfPages
    runner, cfg, _ = runner_of("A", max_tokens=6 * 16)
    vocab = cfg["vocab_size"]
    runner.step([StepEntry("a", tc.random_ids(10, vocab, 1)), StepEntry("b", tc.random_ids(10, vocab, 2))])
    runner.step_tree([tree_of("a", 70, vocab)])   # 5 pages of 6, and "b" has the sixth
    runner.step([StepEntry("b", tc.random_ids(40, vocab, 3))])
    runner.step_tree([tree_of("a", 20, vocab)])
    runner.step_tree([tree_of("b", 30, vocab)])   # 80 tokens: five pages, one of them what "a" had for its tree
    with pytest.raises(OutOfPages):
        runner.step_tree([tree_of("a", 40, vocab)])
    assert free_pages(runner) == [1]
    runner.cache.check_invariants()


@pytest.mark.parametrize("end", ["step", "keep"])
def test_what_was_reserved_ahead_of_a_tree_stays(end):
    """Pages that the caller has reserved for a request are not a tree's."""
    runner, cfg, _ = runner_of("A")
    runner.step([StepEntry("a", tc.random_ids(10, cfg["vocab_size"], 1))])
    runner.cache.reserve("a", 90)
    chosen = runner.step_tree([tree_of("a", 100, cfg["vocab_size"])]).argmax(dim=1).int()
    assert len(runner.cache.table("a", 0)) == 7
    if end == "step":
        runner.step([StepEntry("a", [3])])
    else:
        runner.keep_tree(chosen)
    assert len(runner.cache.table("a", 0)) == 6
    runner.cache.check_invariants()


@pytest.mark.parametrize("again", [False, True])
@pytest.mark.parametrize("ended", [["a"], ["b"], ["c"], ["a", "c"], ["a", "b", "c"], ["d"]])
def test_requests_that_end_between_a_tree_and_what_is_kept_of_it(ended, again):
    """The other requests' nodes are kept; pages that have gone to other requests since are not written."""
    runner, cfg, weights = runner_of("E", max_tokens=16 * 16)
    vocab = cfg["vocab_size"]
    prompts = {r: tc.random_ids(n, vocab, n) for r, n in (("a", 17), ("b", 30), ("c", 5), ("d", 4))}
    runner.step([StepEntry(r, p) for r, p in prompts.items()])
    own = {r: own_tokens(cfg, weights, prompts[r], 4) for r in "abc"}
    entries = [TreeEntry(r, [t[0], 3, t[1], 5, t[2]], [-1, 0, 0, 2, 2]) for r, t in own.items()]
    entries[1] = TreeEntry("b", own["b"][:1], [-1])           # one node: its segment lies behind the others
    chosen = runner.step_tree(entries).argmax(dim=1).int()
    for r in ended:
        runner.free_request(r)
        if again:                                             # a new request of the same name, in the pages that are free now
            runner.add_request(r)
    pages = [runner.model.k_store[g].clone() for g in range(2)]
    held = [{p for r in runner.cache.requests() for p in runner.cache.table(r, g) if p >= 0} for g in range(2)]
    kept = runner.keep_tree(chosen)
    for g in range(2):
        for page in set(range(pages[g].shape[1])) - held[g]:
            assert torch.equal(runner.model.k_store[g][:, page], pages[g][:, page])
    for entry, got in zip(entries, kept):
        r = entry.req_id
        if r in ended:
            assert got == ([], -1) and (runner.length(r) == 0 if again else not runner.cache.has_request(r))
            continue
        nodes = [0] if r == "b" else [0, 2, 4]
        assert got == (nodes, own[r][len(nodes)]) and runner.length(r) == len(prompts[r]) + len(nodes)
        row, = runner.step([StepEntry(r, [got[1]], want=(0,))])
        next_logits(cfg, weights, prompts[r] + own[r][: len(nodes) + 1], row)
    runner.cache.check_invariants()
    with pytest.raises(StepError):
        runner.keep_tree(chosen)


def test_a_caller_may_go_on_with_its_lists():
    """The record of a step on trees is its own: lists that the caller changes meanwhile change nothing."""
    runner, cfg, weights = runner_of("A")
    vocab = cfg["vocab_size"]
    prompts = {"a": tc.random_ids(20, vocab, 1), "b": tc.random_ids(7, vocab, 2)}
    runner.step([StepEntry(r, p) for r, p in prompts.items()])
    own = {r: own_tokens(cfg, weights, p, 3) for r, p in prompts.items()}
    entries = [TreeEntry("a", own["a"][:1], [-1]), TreeEntry("b", [own["b"][0], 3, own["b"][1]], [-1, 0, 0])]
    chosen = runner.step_tree(entries).argmax(dim=1).int()
    entries[0].tokens.append(9), entries[1].tokens.clear(), entries[1].parents.clear()
    entries[0].req_id = "c"
    entries.pop()
    assert runner.keep_tree(chosen) == [([0], own["a"][1]), ([0, 2], own["b"][2])]
    got = runner.step([StepEntry("a", [own["a"][1]], want=(0,)), StepEntry("b", [own["b"][2]], want=(0,))])
    next_logits(cfg, weights, prompts["a"] + own["a"][:2], got[0])
    next_logits(cfg, weights, prompts["b"] + own["b"], got[1])
    runner.cache.check_invariants()
