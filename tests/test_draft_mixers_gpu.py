"""Engine.verify through the mixers that take trees beside the grouped-query attention: whole-projection norms and head norms with
windows, capped scores, sinks, values of their own width, rotations in pairs, query temperatures by position and padded caches. Held to
the same engine's ordinary steps, which the tests of each model hold to plain implementations."""
import dataclasses
import random

import pytest
import torch

from conftest import seeded_tokens, tolerance
from rasezen_models import attention, config, dense, layer
from test_draft_engine_gpu import draft_all

pytestmark = pytest.mark.gpu

VOCAB, WIDTH = 131, 96
SIZES = {        # heads, kv heads, keys, values of two layers
    "odd": [(4, 2, 16, 24), (6, 3, 20, 12)],
    "swizzled": [(4, 2, 64, 64), (8, 1, 128, 128)],
    "mixed": [(4, 4, 64, 128), (4, 2, 128, 48)],
}
WIDE = {
    "plain": [{}, dict(window=30)],
    "sink": [dict(sink=True, window=50), dict(sink=True, value_norm=False, interleaved_rotation=True)],
}
HEAD = {
    "cap": [dict(softcap=2.0), dict(softcap=5.0, window=40, sink=True)],
    "temperature": [dict(query_temperature=(0.4, 16), interleaved_rotation=True, bias=True), dict(qk_norm="unit", window=33, sink=True)],
    "padded": [dict(padded_cache=True, sink=True), dict(padded_cache=True, softcap=3.0, window=70)],
}


def engine(kind, sizes, options, dtype, seed):
    """An attention-only model whose mixers are replaced by `kind` with the options, with weights that keep activations of order one."""
    from lumenllm_b200 import Engine, config_from_dict
    from lumenllm_b200.engine.model import expected_tensors
    layers = [layer(attention(H, G, d, dv, 1.5 * d ** -0.5, rot=d // 2 * 2 if d < 64 else 32), dense(80 + 16 * i))
              for i, (H, G, d, dv) in enumerate(SIZES[sizes])]
    spec = config_from_dict(config(VOCAB, WIDTH, 1e-6, layers)).model_spec()
    layers = tuple(dataclasses.replace(L, mixer=dataclasses.replace(L.mixer, kind=kind, params={**L.mixer.params, **opts}))
                   for L, opts in zip(spec.layers, options))
    spec = dataclasses.replace(spec, layers=layers, max_positions=2048)
    g = torch.Generator().manual_seed(seed)
    weights = {}
    for name, (shape, what) in expected_tensors(spec).items():
        x = torch.randn(shape, generator=g)
        if what == "norm":
            x = 1 + 0.1 * x
        elif name.endswith(".b") or name.endswith(".sink"):
            x = 0.2 * x
        elif name.endswith(".act"):
            x = torch.tensor([0.3, -0.2]) + 0.2 * x
        elif name != "embed":
            x = x * shape[-1] ** -0.5
        weights[name] = x.to(torch.bfloat16).cuda()
    return Engine(spec, weights, dtype, 4096, 8, 0)


CASES = [("wide_norm_attention", s, o) for s in SIZES for o in WIDE] + [("head_norm_attention", s, o) for s in SIZES for o in HEAD
                                                                         if not (o == "padded" and s != "swizzled")]


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("kind,sizes,options", CASES)
def test_drafts_pick_what_ordinary_steps_pick(kind, sizes, options, dtype):
    """Every token that comes out is, by the logits of an ordinary prompt step over the tokens before it, within rounding of the best one
    (both tokens' logits may be off by the engine's bound), and what the drafts leave in the cache gives the next token's logits."""
    from lumenllm_b200 import StepEntry
    eng = engine(kind, sizes, {**WIDE, **HEAD}[options], dtype, seed=17)
    assert eng.model.tree_safe
    prompts = seeded_tokens(VOCAB, [40, 75, 3], seed=21)
    want = []
    for p in prompts:
        s = eng.alloc_slot()
        seq = list(p)
        feed = list(p)
        for _ in range(20):
            seq.append(int(eng.step([StepEntry(s, feed, [len(feed) - 1])]).argmax()))
            feed = seq[-1:]
        want.append(seq[len(p):])
        eng.free_slot(s)
    slots, out, steps = draft_all(eng, prompts, want, random.Random(6), nodes=30)
    assert steps < 19 and sum(len(o) for o in out) >= 60
    for b, p in enumerate(prompts):
        seq = list(p) + out[b]
        s = eng.alloc_slot()
        ref = eng.step([StepEntry(s, seq, list(range(len(seq))))]).cpu()
        eng.free_slot(s)
        for k, tok in enumerate(out[b]):
            row = ref[len(p) - 1 + k]
            assert float(row.max() - row[tok]) <= 2 * tolerance(dtype, row)
        got = eng.step([StepEntry(slots[b], [out[b][-1]], [0])]).cpu()
        assert float((got - ref[-1:]).abs().max()) <= 2 * tolerance(dtype, ref[-1:])
        eng.free_slot(slots[b])
    eng.cache.check()


def test_a_padded_bfloat16_cache_of_other_widths_takes_no_trees():
    """Rows that are padded to the next multiple of 64 need an option that tree attention has not."""
    from lumenllm_b200 import DraftEntry, StepError
    eng = engine("head_norm_attention", "odd", HEAD["padded"], "bfloat16", seed=3)
    with pytest.raises(StepError, match="no drafts"):
        eng.verify([DraftEntry(eng.alloc_slot(), [1], [-1])])
    assert engine("head_norm_attention", "odd", HEAD["padded"], "float32", seed=3).model.tree_safe
