"""Requests that go on in two ways, for every family of models: pages, pooled blocks and states of fixed size of the fork are its own."""
import numpy as np
import torch

import dovudra_configs
import dumizen_configs
import menitar_configs
import plain_dovudra
import plain_dumizen
import plain_menitar
import plain_purivik
import plain_venadra
import plain_zoguzen
import purivik_configs
import venadra_configs
import zoguzen_configs

FAMILIES = {"venadra": (venadra_configs, plain_venadra), "zoguzen": (zoguzen_configs, plain_zoguzen), "purivik": (purivik_configs, plain_purivik),
            "dumizen": (dumizen_configs, plain_dumizen), "dovudra": (dovudra_configs, plain_dovudra), "menitar": (menitar_configs, plain_menitar)}
CASES = [(family, name) for family, (configs, _) in FAMILIES.items() for name in configs.CONFIGS]


def check_forks(family, name, lengths, tolerance, **kw):
    """Forks behind prompts of these lengths: each way's logits against the plain implementation over its own tokens."""
    from fllm_amd.engine import ModelRunner, StepEntry
    from fllm_amd.registry import model_spec_from_config
    configs, plain = FAMILIES[family]
    cfg = configs.CONFIGS[name]
    tensors = configs.named_weights(name, 3) if hasattr(configs, "named_weights") else configs.weights(cfg, 3)
    _, spec = model_spec_from_config(cfg)
    runner = ModelRunner(spec, {n: t.to(torch.float32) for n, t in tensors.items()}, page_size=configs.PAGE_SIZES[name],
                         **{"max_tokens": 600, "max_requests": 5, "max_context": 512, **kw})
    w64 = configs.to_float64(tensors)
    vocab = runner.vocab_size
    for length in lengths:
        tokens = {"a": configs.random_ids(length, vocab, length)}
        runner.step([StepEntry("a", tokens["a"])])
        more = {r: configs.random_ids(40, vocab, 100 * length + i) for i, r in enumerate("abcd")}

        def step(count):
            for _ in range(count):
                for r in tokens:
                    tokens[r] = tokens[r] + [more[r].pop()]
                logits = runner.step([StepEntry(r, [t[-1]], want=(0,)) for r, t in tokens.items()]).cpu().numpy().copy()
            for r, got in zip(tokens, logits):
                want = plain.forward(cfg, w64, tokens[r])[-1]
                assert np.abs(got - want).max() <= tolerance * np.abs(want).max(), (length, r)

        for src, dst, count in (("a", "b", 3), ("b", "c", 2), ("a", "d", 11)):      # a fork, a fork of it, the first once more
            runner.fork_request(src, dst)
            tokens[dst] = list(tokens[src])
            step(count)
            runner.cache.check_invariants()
        runner.free_request("a")               # the ways that came of it go on
        del tokens["a"]
        step(2)
        for r in tokens:
            runner.free_request(r)
        runner.cache.check_invariants()
        assert runner.cache.free_slots() == 5 and all(p.available == p.num_pages for p in runner.cache.pools)
