"""Whole steps on trees of drafted tokens and requests that go on in two ways: every logit against the plain implementation over the
sequence from the first token to the node, the walk and the moved cache against steps that took the same tokens one by one.
Tolerances: those of the replays (`test_replay_gpu.py`), the same computation in another order."""
import random

import numpy as np
import pytest
import torch

import draft_reference as plain
import plain_llama
import tiny_configs as tc

pytestmark = pytest.mark.gpu
TOL = {"float32": 3e-6, "bfloat16": 1.5e-2}


def runner_of(name, dtype, **more):
    from fllm_amd.engine import ModelRunner
    from fllm_amd.registry import model_spec_from_config
    from fllm_amd.weights import random_tensors
    cfg = tc.CONFIGS[name]
    _, spec = model_spec_from_config(cfg)
    tensors = {k: v.to(torch.float32) for k, v in random_tensors(spec, seed=5 + ord(name), dtype=torch.bfloat16, with_optional=(name == "C")).items()}
    args = dict(dtype=dtype, page_size=tc.PAGE_SIZES[name], max_tokens=2000, max_requests=8)
    return ModelRunner(spec, tensors, **dict(args, **more)), cfg, tc.to_float64(tensors)


def lines(parents):
    """Node -> the nodes from the root to it."""
    out = []
    for i, p in enumerate(parents):
        out.append((out[p] if i else []) + [i])
    return out


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("name", list(tc.CONFIGS))
def test_logits_of_trees(name, dtype):
    from fllm_amd.engine import StepEntry, TreeEntry
    runner, cfg, weights = runner_of(name, dtype)
    rng = random.Random(ord(name))
    vocab = cfg["vocab_size"]
    prompts = [tc.random_ids(n, vocab, 7 + n) for n in (50, 3, 33)]
    runner.step([StepEntry(i, p) for i, p in enumerate(prompts)])
    sizes = (13, 1, 24)
    trees = [plain.random_tree(n, rng) for n in sizes]
    tokens = [[rng.randrange(vocab) for _ in range(n)] for n in sizes]
    got = runner.step_tree([TreeEntry(i, tokens[i], trees[i]) for i in range(3)]).cpu().numpy()
    at = 0
    for i in range(3):
        for node, line in enumerate(lines(trees[i])):
            want = plain_llama.forward(cfg, weights, prompts[i] + [tokens[i][j] for j in line])[-1]
            assert np.abs(got[at] - want).max() <= TOL[dtype] * np.abs(want).max(), (i, node)
            at += 1
    assert runner.length(0) == 50                  # nothing is committed


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("name", ["A", "D", "E", "F"])
def test_drafted_generation_is_generation(name, dtype):
    """Greedy tokens of steps on trees (some of whose drafts are what the model says, most are not) are the tokens that steps of one token each
    make, and the cache they leave gives the same logits."""
    from fllm_amd.engine import StepEntry, TreeEntry
    runner, cfg, weights = runner_of(name, dtype)
    rng = random.Random(3)
    vocab = cfg["vocab_size"]
    prompts = {f"p{i}": tc.random_ids(n, vocab, n) for i, n in enumerate((20, 41))}
    goal = 30
    logits = runner.step([StepEntry(r, p, want=(len(p) - 1,)) for r, p in prompts.items()])
    newest = dict(zip(prompts, logits.argmax(dim=1).tolist()))
    for r in prompts:                              # the same request once more, token by token
        runner.fork_request(r, r + "'")
    want = {r: [newest[r]] for r in prompts}
    rows = {}
    while any(len(w) < goal + 14 for w in want.values()):
        logits = runner.step([StepEntry(r + "'", [want[r][-1]], want=(0,)) for r in prompts])
        for r, row in zip(prompts, logits):
            rows[r, len(want[r]) - 1] = row.cpu()
            want[r].append(int(row.argmax()))
    made = {r: [newest[r]] for r in prompts}
    steps = 0
    while any(len(m) < goal for m in made.values()):
        live = [r for r in prompts if len(made[r]) < goal]
        entries = []
        for r in live:
            n = rng.randint(1, 12)
            parents = plain.random_tree(n, rng, 0.6)
            line = lines(parents)
            tokens = [made[r][-1]]
            for i in range(1, n):                  # a node that continues the model's own tokens says the next of them, two times in three
                own = all(tokens[j] == want[r][len(made[r]) - 1 + d] for d, j in enumerate(line[i][:-1]))
                tokens.append(want[r][len(made[r]) - 1 + len(line[i]) - 1] if own and rng.random() < 0.67 else rng.randrange(vocab))
            entries.append(TreeEntry(r, tokens, parents))
        before = {r: runner.length(r) for r in live}
        logits = runner.step_tree(entries)
        chosen = logits.argmax(dim=1).to(torch.int32)
        at = 0
        kept = runner.keep_tree(chosen)
        for e, (path, token) in zip(entries, kept):
            assert path == plain.follow([-1] + list(e.parents[1:]), e.tokens, chosen[at:at + len(e.tokens)].tolist(), 99)[0]
            at += len(e.tokens)
            assert runner.length(e.req_id) == before[e.req_id] + len(path)
            made[e.req_id] += [e.tokens[j] for j in path[1:]] + [token]
        runner.cache.check_invariants()
        steps += 1
    for r in prompts:
        n = min(len(made[r]), len(want[r]))
        if dtype == "float32":                     # (in bfloat16 two tokens may be as likely as each other)
            assert made[r][:n] == want[r][:n]
    assert steps < sum(len(m) for m in made.values()) / 2
    # what lies in the cache after all the moves: the next token's logits, against the plain implementation
    logits = runner.step([StepEntry(r, [made[r][-1]], want=(0,)) for r in prompts]).cpu().numpy()
    for got, r in zip(logits, prompts):
        plainly = plain_llama.forward(cfg, weights, prompts[r] + made[r])[-1]
        assert np.abs(got - plainly).max() <= TOL[dtype] * np.abs(plainly).max()


@pytest.mark.parametrize("name", ["A", "E", "F"])
def test_a_fork_goes_on_by_itself(name):
    from fllm_amd.engine import StepEntry
    runner, cfg, weights = runner_of(name, "float32")
    vocab = cfg["vocab_size"]
    prompt, one, two = tc.random_ids(45, vocab, 1), tc.random_ids(9, vocab, 2), tc.random_ids(12, vocab, 3)
    runner.step([StepEntry("a", prompt)])
    runner.fork_request("a", "b")
    runner.step([StepEntry("a", one[:5]), StepEntry("b", two[:7])])
    runner.fork_request("b", "c")
    got = runner.step([StepEntry("a", one[5:], want=(3,)), StepEntry("b", two[7:], want=(4,)), StepEntry("c", one, want=(8,))]).cpu().numpy()
    for row, tail in zip(got, (one, two, two[:7] + one)):
        want = plain_llama.forward(cfg, weights, prompt + tail)[-1]
        assert np.abs(row - want).max() <= TOL["float32"] * np.abs(want).max()
    runner.cache.check_invariants()
    for r in "abc":
        runner.free_request(r)
    assert runner.cache.free_pages(0) == runner.pages_per_group[0]


def test_refusals():
    from fllm_amd.cache import OutOfPages
    from fllm_amd.engine import StepEntry, StepError, TreeEntry
    runner, cfg, _ = runner_of("D", "bfloat16", max_tokens=64, max_requests=2)
    with pytest.raises(StepError):
        runner.step_tree([TreeEntry("a", [1, 2], [-1, 0])])                # no prompt
    runner.step([StepEntry("a", [1, 2, 3])])
    for tokens, parents in (([1, 2], [-1, 1]), ([1, 2], [-1]), ([], []), ([1, 9999], [-1, 0]), ([1, 2, 3], [-1, 0, -2])):
        with pytest.raises(StepError):
            runner.step_tree([TreeEntry("a", tokens, parents)])
    with pytest.raises(StepError):
        runner.keep_tree(torch.zeros(2, dtype=torch.int32, device="cuda"))  # no tree before it
    runner.step_tree([TreeEntry("a", [4, 5], [-1, 0])])
    with pytest.raises(StepError):
        runner.keep_tree(torch.zeros(3, dtype=torch.int32, device="cuda"))
    runner.step([StepEntry("a", [4])])                                      # leaves the tree behind
    with pytest.raises(StepError):
        runner.keep_tree(torch.zeros(2, dtype=torch.int32, device="cuda"))
    runner.step_tree([TreeEntry("a", [4, 5], [-1, 0])])
    with pytest.raises(KeyError):
        runner.fork_request("nobody", "c")
    with pytest.raises(ValueError):
        runner.fork_request("a", "a")
    assert runner.cache.requests() == ["a"]
    runner.step([StepEntry("b", list(range(1, 49)))])                       # 48 tokens: the three pages that "a" has left
    with pytest.raises(OutOfPages):
        runner.step_tree([TreeEntry("a", [4] + [5] * 20, [-1] + [0] * 20)])
    runner.free_request("b")
    runner.step([StepEntry("a", list(range(1, 52)))])                       # every page is taken
    with pytest.raises(OutOfPages):
        runner.fork_request("a", "c")
    assert runner.cache.requests() == ["a"]
    runner.cache.check_invariants()
