"""Engine.verify: trees of drafted tokens, some right and some wrong, in batches of unequal sequences; the tokens that come out
against single steps and against the plain implementation, and what the cache holds afterwards."""
import random

import pytest
import torch

import plain_qwen3 as P
from conftest import TINY, seeded_tokens, tolerance

pytestmark = pytest.mark.gpu

NAMES = ["A", "C", "D", "E"]        # plain tiles of 16 and 48, swizzled ones of 64 and 128, with and without a window


def grow(rng, good, vocab, nodes):
    """A tree that begins with good[0] and holds a stretch of `good` among wrong tokens, in any order parents allow."""
    tokens, parents, last, k = [good[0]], [-1], 0, 1
    while len(tokens) < nodes:
        if k < len(good) and rng.random() < 0.5:
            parents.append(last)
            tokens.append(good[k])
            last, k = len(tokens) - 1, k + 1
        else:
            parents.append(rng.randrange(len(tokens)))
            tokens.append(rng.randrange(vocab))
    return tokens, parents


def draft_all(eng, prompts, want, rng, nodes, configs=None, uniform=None):
    """Generates the tokens of `want` (a list a prompt) by verify alone, drafting from them; returns what came out and the steps."""
    from lumenllm_b200 import DraftEntry, SamplingConfig, StepEntry
    slots = [eng.alloc_slot() for _ in prompts]
    first = eng.run([(s, list(p)) for s, p in zip(slots, prompts)], configs or [SamplingConfig()] * len(prompts),
                    [uniform(b, 0) if uniform else 0.0 for b in range(len(prompts))])
    out, steps = [[t] for t in first], 0
    while any(len(o) < len(w) for o, w in zip(out, want)):
        live = [b for b in range(len(prompts)) if len(out[b]) < len(want[b])]
        drafts = []
        for b in live:
            n = rng.randint(1, nodes)
            ahead = [out[b][-1]] + list(want[b][len(out[b]):])
            drafts.append(DraftEntry(slots[b], *grow(rng, ahead, eng.vocab_size, n)))
        us = None if uniform is None else [[uniform(b, len(out[b]) + k) for k in range(nodes + 1)] for b in live]
        got = eng.verify(drafts, None if configs is None else [configs[b] for b in live], us)
        for b, g in zip(live, got):
            assert len(g) >= 1 and eng.length(slots[b]) == len(prompts[b]) + len(out[b]) - 1 + len(g)
            out[b] += g
        steps += 1
    eng.cache.check()
    return slots, out, steps


@pytest.fixture(scope="module")
def engines(tiny_models):
    from lumenllm_b200 import Engine
    cache = {}

    def get(name, dtype):
        if (name, dtype) not in cache:
            cache[name, dtype] = Engine.from_folder(tiny_models[name], dtype=dtype, max_tokens=4096)
        return cache[name, dtype]
    return get


@pytest.mark.parametrize("name", NAMES)
def test_drafts_give_the_tokens_of_single_steps(engines, tiny_models, name):
    """float32, greedy: whatever is drafted, the tokens are the plain implementation's, and after the last step the cache holds
    what a prompt of the same tokens leaves there (the next logits agree)."""
    from lumenllm_b200 import StepEntry
    eng = engines(name, "float32")
    cfg, w = P.load_model(tiny_models[name])
    prompts = seeded_tokens(TINY[name]["vocab_size"], [33, 70, 5], seed=3)
    want = [P.generate_greedy(cfg, w, p, 24)[0] for p in prompts]
    slots, out, steps = draft_all(eng, prompts, want, random.Random(1), nodes=20)
    for b in range(3):
        assert out[b][:24] == want[b]
    assert steps < 23                                   # single steps would have taken 23
    for b in range(3):
        seq = list(prompts[b]) + out[b]
        got = eng.step([StepEntry(slots[b], [out[b][-1]], [0])]).cpu()
        ref = P.forward_logits(cfg, w, seq)[-1:]
        assert float((got - ref).abs().max()) <= tolerance("float32", ref)
        eng.free_slot(slots[b])


@pytest.mark.parametrize("name", NAMES)
def test_bfloat16_drafts_pick_within_the_rounding_of_logits(engines, tiny_models, name):
    """bfloat16: every token that comes out is, by the plain implementation's logits after the tokens before it, within what
    rounding does to logits of the best one."""
    eng = engines(name, "bfloat16")
    cfg, w = P.load_model(tiny_models[name])
    prompts = seeded_tokens(TINY[name]["vocab_size"], [64, 130, 3, 40], seed=5)
    want = [P.generate_greedy(cfg, w, p, 20)[0] for p in prompts]
    slots, out, _ = draft_all(eng, prompts, want, random.Random(2), nodes=40)
    for b, p in enumerate(prompts):
        lg = P.forward_logits(cfg, w, list(p) + out[b])
        for k, tok in enumerate(out[b]):
            row = lg[len(p) - 1 + k]
            # both tokens' logits may be off by the bound that the engine's bfloat16 logits are held to
            assert float(row.max() - row[tok]) <= 2 * tolerance("bfloat16", row)
        eng.free_slot(slots[b])


def test_sampled_drafts_are_sampled_steps(engines):
    """With the numbers that single steps draw, sampling through trees gives the tokens of single steps (float32)."""
    from lumenllm_b200 import GenerateRequest, SamplingConfig
    from lumenllm_b200.sampling import uniform
    eng = engines("A", "float32")
    cfgs = [SamplingConfig(temperature=0.8, top_k=20, seed=11), SamplingConfig(temperature=1.1, top_p=0.9, seed=5), SamplingConfig()]
    prompts = seeded_tokens(TINY["A"]["vocab_size"], [20, 31, 7], seed=9)
    want = [o.tokens for o in eng.generate([GenerateRequest(p, 16, c) for p, c in zip(prompts, cfgs)], eos_token_ids=[])]
    slots, out, _ = draft_all(eng, prompts, want, random.Random(4), nodes=12, configs=cfgs,
                              uniform=lambda b, k: uniform(cfgs[b].seed or 0, 0, k))
    for b in range(3):
        assert out[b][:16] == want[b]
        eng.free_slot(slots[b])


def test_a_greedy_sequence_among_sampled_ones_needs_no_numbers(engines):
    from lumenllm_b200 import DraftEntry, SamplingConfig, StepEntry
    eng = engines("A", "float32")
    prompts = seeded_tokens(TINY["A"]["vocab_size"], [20, 31], seed=9)
    alone, cfgs = [], [SamplingConfig(), SamplingConfig(temperature=0.9, seed=2)]
    for rows in ([[0.1, 0.2], [0.3, 0.4]], [None, [0.3, 0.4]], [[], [0.3, 0.4]]):
        slots = [eng.alloc_slot() for _ in prompts]
        eng.step([StepEntry(s, p[:-1], []) for s, p in zip(slots, prompts)])
        alone.append(eng.verify([DraftEntry(s, [p[-1], 5], [-1, 0]) for s, p in zip(slots, prompts)], cfgs, rows))
        for s in slots:
            eng.free_slot(s)
    assert alone[0] == alone[1] == alone[2]


def test_drafts_between_ordinary_steps_and_a_full_cache(tiny_models):
    """verify, step and generate share the slots; a step of drafts for which there is no room is refused and changes nothing."""
    from lumenllm_b200 import DraftEntry, Engine, GenerateRequest, StepEntry, StepError
    eng = Engine.from_folder(tiny_models["D"], dtype="float32", max_tokens=192)
    prompt = seeded_tokens(TINY["D"]["vocab_size"], [100], seed=1)[0]
    want = eng.generate(GenerateRequest(prompt, 8), eos_token_ids=[]).tokens
    s = eng.alloc_slot()
    lg = eng.step([StepEntry(s, prompt, [99])])
    assert int(lg.argmax()) == want[0]
    before = eng.length(s)
    with pytest.raises(StepError, match="beyond the longest sequence"):
        eng.verify([DraftEntry(s, [want[0]] * 100, [-1] + [0] * 99)])
    assert eng.length(s) == before
    got = eng.verify([DraftEntry(s, [want[0], want[1], 3, want[2]], [-1, 0, 1, 1])])
    assert got == [want[1:4]] and eng.length(s) == before + 3
    lg = eng.step([StepEntry(s, [want[3]], [0])])
    assert int(lg.argmax()) == want[4]
    assert eng.verify([DraftEntry(s, [want[4]], [-1])]) == [[want[5]]]        # a tree of one: a decode step
    eng.free_slot(s)
    eng.cache.check()
    assert eng.generate(GenerateRequest(prompt, 8), eos_token_ids=[]).tokens == want


def test_models_with_state_take_no_drafts():
    from lumenllm_b200 import DraftEntry, Engine, StepError
    from rasezen_models import SMALL
    cfg = next(c for c in SMALL.values())
    eng = Engine.from_random(dict(cfg), dtype="float32", max_tokens=256)
    s = eng.alloc_slot()
    with pytest.raises(StepError, match="no drafts"):
        eng.verify([DraftEntry(s, [1], [-1])])


def test_drafts_that_crowd_the_cache(tiny_models):
    """Trees as large as the cache's room, mostly wrong: what they took is there again for other sequences, whose pages the
    page tables on the device follow, and the tokens stay the plain implementation's."""
    from lumenllm_b200 import DraftEntry, Engine, StepEntry, StepError
    eng = Engine.from_folder(tiny_models["D"], dtype="float32", max_tokens=512)
    cfg, w = P.load_model(tiny_models["D"])
    prompts = seeded_tokens(TINY["D"]["vocab_size"], [50, 64, 10], seed=7)
    want = [P.generate_greedy(cfg, w, p, 14)[0] for p in prompts]
    rng = random.Random(3)
    slots, out = [], []
    for p, t in zip(prompts, want):
        slots.append(eng.alloc_slot())
        eng.step([StepEntry(slots[-1], list(p), [len(p) - 1])])
        out.append([t[0]])
    while min(len(o) for o in out) < 12:
        for b in range(3):
            room = (eng.cache.free_tokens() // 64 + int(eng.cache.groups[0].end_page[slots[b]])) * 64 - eng.length(slots[b])
            tokens, parents = grow(rng, [out[b][-1]] + want[b][len(out[b]):], eng.vocab_size, min(room, 200))
            out[b] += eng.verify([DraftEntry(slots[b], tokens, parents)])[0]
            eng.cache.check()
        free = eng.cache.free_tokens()
        tables = [g.table.copy() for g in eng.cache.groups]
        with pytest.raises(StepError, match="full"):
            eng.verify([DraftEntry(s, [1] * 200, [-1] + [0] * 199) for s in slots])
        assert eng.cache.free_tokens() == free and all((g.table == t).all() for g, t in zip(eng.cache.groups, tables))
    for b in range(3):
        n = min(len(out[b]), 14)
        assert out[b][:n] == want[b][:n]
        assert eng.cache.groups[0].n_held[slots[b]] == -(-eng.length(slots[b]) // 64)
        eng.free_slot(slots[b])
    eng.cache.check()
