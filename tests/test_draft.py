"""What the operators for trees of drafted tokens refuse, before anything reaches a device, and the plain forms that the GPU
tests hold them to, against each other."""
import random

import pytest
import torch

import plain_draft as D
from lumenllm_b200.ops import kernels as K
from lumenllm_b200.ops.native import KernelError

F32, BF16, I32, I64 = torch.float32, torch.bfloat16, torch.int32, torch.int64


def i32(*shape):
    return torch.zeros(shape, dtype=I32)


def tree_args(**over):
    a = dict(q=torch.zeros(3, 4, 64, dtype=BF16), kcache=torch.zeros(5, 2, 64, 64, dtype=BF16),
             vcache=torch.zeros(5, 2, 64, 64, dtype=BF16), block_table=i32(1, 2), cu_q=i32(2), seq_start=i32(1), tok_seq=i32(3),
             tok_pos=i32(3), tree_mask=torch.zeros(3, 1, dtype=I64), window=0, scale=0.125)
    return {**a, **over}


@pytest.mark.parametrize("over,says", [
    (dict(q=torch.zeros(3, 4, 64, dtype=torch.float16)), "float32 or all bfloat16"),
    (dict(q=torch.zeros(3, 4, 64)), "float32 or all bfloat16"),
    (dict(q=torch.zeros(3, 4, 48, dtype=BF16)), "do not fit"),
    (dict(q=torch.zeros(3, 3, 64, dtype=BF16)), "do not fit"),
    (dict(vcache=torch.zeros(5, 1, 64, 64, dtype=BF16)), "do not fit"),
    (dict(vcache=torch.zeros(4, 2, 64, 64, dtype=BF16)), "do not fit"),
    (dict(kcache=torch.zeros(5, 2, 32, 64, dtype=BF16)), "do not fit"),
    (dict(kcache=torch.zeros(5, 64, 64, dtype=BF16)), "caches are"),
    (dict(vcache=torch.zeros(5, 2, 64, 513, dtype=BF16)), "1 to 512"),
    (dict(tree_mask=torch.zeros(3, 5, dtype=I64)), "tree_mask"),
    (dict(tree_mask=torch.zeros(3, dtype=I64)), "tree_mask"),
    (dict(tree_mask=torch.zeros(2, 1, dtype=I64)), "tree_mask"),
    (dict(tree_mask=torch.zeros(3, 1, dtype=I32)), "tree_mask"),
    (dict(window=-1), "window"),
    (dict(softcap=-1.0), "softcap"),
    (dict(softcap=float("nan")), "softcap"),
    (dict(cu_q=i32(3)), "block_table"),
    (dict(block_table=i32(1, 0)), "block_table"),
    (dict(block_table=i32(2, 2).t()), "block_table"),
    (dict(block_table=torch.zeros(1, 2, dtype=I64)), "block_table"),
    (dict(seq_start=i32(0)), "seq_start"),
    (dict(tok_seq=i32(2)), "tok_seq"),
    (dict(tok_pos=torch.zeros(3, dtype=I64)), "tok_pos"),
    (dict(q=torch.zeros(3, 64, 4, dtype=BF16).transpose(1, 2)), "contiguous"),
    (dict(layout=K.LAYOUT_SW128, kcache=torch.zeros(5, 2, 64, 48, dtype=BF16), q=torch.zeros(3, 4, 48, dtype=BF16)), "layout"),
    (dict(layout=7), "layout"),
    (dict(), "not on a CUDA device"),
])
def test_tree_attention_refuses(over, says):
    with pytest.raises(KernelError, match=says):
        K.attn_tree(**tree_args(**over))


@pytest.mark.parametrize("over,says", [
    (dict(slot_pages=i32(3, 2)), "slot_pages"),
    (dict(slot_pages=i32(4, 3).t()), "slot_pages"),
    (dict(slot_pages=torch.zeros(3, 4, dtype=I64)), "slot_pages"),
    (dict(width=0), "pages"),
    (dict(n_tokens=-1), "tokens"),
    (dict(mask_words=5), "mask words"),
    (dict(seq_qlen=i32(1)), "seq_qlen"),
    (dict(seq_slot=torch.zeros(2, dtype=I64)), "seq_slot"),
    (dict(seq_start=i32(4)[::2]), "contiguous"),
    (dict(parents=i32(4)), "parents"),
    (dict(), "not on a CUDA device"),
])
def test_step_tables_refuse(over, says):
    a = dict(seq_start=i32(2), seq_qlen=i32(2), slot_pages=i32(3, 4), seq_slot=i32(2), n_tokens=5, width=4, parents=i32(5))
    with pytest.raises(KernelError, match=says):
        K.step_tables(**{**a, **over})


@pytest.mark.parametrize("over,says", [
    (dict(max_path=0), "paths"),
    (dict(max_path=257), "paths"),
    (dict(tokens=i32(4)), "tokens"),
    (dict(parents=torch.zeros(5, dtype=I64)), "parents"),
    (dict(cu_q=i32(0)), "sequences"),
    (dict(), "not on a CUDA device"),
])
def test_acceptance_refuses(over, says):
    with pytest.raises(KernelError, match=says):
        K.tree_accept(**{**dict(picked=i32(5), tokens=i32(5), parents=i32(5), cu_q=i32(3), max_path=4), **over})


@pytest.mark.parametrize("over,says", [
    (dict(kcache=torch.zeros(2, 5, 2, 64, 64, dtype=torch.float16)), "float32 or bfloat16"),
    (dict(kcache=torch.zeros(2, 5, 2, 32, 64, dtype=BF16)), "keys are"),
    (dict(vcache=torch.zeros(2, 5, 1, 64, 64, dtype=BF16)), "do not fit"),
    (dict(vcache=torch.zeros(2, 5, 2, 64, 64)), "do not fit"),
    (dict(v_layout=1, vcache=torch.zeros(2, 5, 2, 64, 48, dtype=BF16)), "layout"),
    (dict(path=i32(3, 4)), "path"),
    (dict(path=i32(2, 300)), "path"),
    (dict(block_table=i32(1, 4)), "block_table"),
    (dict(seq_start=i32(1)), "seq_start"),
    (dict(), "not on a CUDA device"),
])
def test_cache_move_refuses(over, says):
    a = dict(kcache=torch.zeros(2, 5, 2, 64, 64, dtype=BF16), vcache=torch.zeros(2, 5, 2, 64, 64, dtype=BF16), block_table=i32(2, 4),
             seq_start=i32(2), path=i32(2, 4), count=i32(2))
    with pytest.raises(KernelError, match=says):
        K.cache_compact(**{**a, **over})


def test_plain_tree_attention_is_plain_attention_for_chains():
    """A chain of nodes is a causal prompt: the plain tree form and the suite's plain causal attention agree."""
    import plain_qwen3 as P
    c = D.Case([0, 70], [5, 9], 4, 2, 16, dtype=F32, seed=1)
    c.sets = [[set(range(i + 1)) for i in range(n)] for n in c.qlens]
    c.pos = [[s + i for i in range(n)] for s, n in zip(c.starts, c.qlens)]
    for window in (0, 6):
        ref, _ = c.reference(window=window)
        n0 = 0
        for b, (s, n) in enumerate(zip(c.starts, c.qlens)):
            full = torch.zeros(s + n, 4, 16)
            full[s:] = c.q[n0:n0 + n]
            want = P.causal_attention(full, c.k[b], c.v[b], window=window)[s:]
            # float32 sums of up to 79 weights near 1/79 of values below 5, and of 16 products
            assert float((ref[n0:n0 + n].float() - want).abs().max()) < 79 * 5 * 2.0 ** -23
            n0 += n


def test_plain_tables_of_a_small_tree():
    cu, seq, cpos, tpos, smap, table, mask = D.tables([62, 0], [4, 2], [[9, 8], [7, 6], [5, 4]], [2, 0], 8, 2,
                                                      parents=[-1, 0, 0, 2, -1, 0, 0, 0])
    assert cu.tolist() == [0, 4, 6] and seq.tolist() == [0, 0, 0, 0, 1, 1, 2, 2]
    assert cpos.tolist() == [62, 63, 64, 65, 0, 1, 0, 0] and tpos.tolist() == [62, 63, 63, 64, 0, 1, 0, 0]
    assert smap.tolist() == [5 * 64 + 62, 5 * 64 + 63, 4 * 64, 4 * 64 + 1, 9 * 64, 9 * 64 + 1, -1, -1]
    assert table.tolist() == [[5, 4], [9, 0], [0, 0]] and mask.flatten().tolist() == [1, 3, 5, 13, 1, 3, 0, 0]


def test_plain_walk():
    # node 0 picks 7: children 1 (token 5) and 2, 3 (token 7): the lower one, whose child 4 answers its pick 9
    count, path, said = D.accept([7, 1, 9, 9, 3], [0, 5, 7, 7, 9], [-1, 0, 0, 0, 2], [0, 5, 5], 4)
    assert count == [3, 0] and path == [[0, 2, 4, -1], [-1] * 4] and said == [[7, 9, 3, -1], [-1] * 4]


def test_segments_of_partial_results_fit_their_room():
    """The cut of a sequence (csrc/tree_plan.cuh) never needs more (token, segment) pairs than a call makes room for."""
    rng = random.Random(0)
    for _ in range(3000):
        width, G = rng.randint(1, 700), rng.choice([1, 2, 3, 4, 5, 8, 16, 40])
        q, np_ = rng.randint(1, 300), rng.randint(1, width)
        seg = min(np_, max(2, (q * G + 31) // 32))
        nseg = min(-(-np_ // seg), 64)
        assert nseg == 1 or (width > 2 and q * nseg <= q + -(-32 * width // G))


def drafting_engine(**over):
    """An Engine's bookkeeping without a device: enough for what verify refuses."""
    from lumenllm_b200.cache import CacheNeed, KVCache
    from lumenllm_b200.engine import Engine
    e = Engine.__new__(Engine)
    e.cache = KVCache({0: CacheNeed(1, 16)}, 640, 4, max_positions=512)
    e.model = type("M", (), {"tree_safe": True})()
    e.vocab_size, e.max_seq_len, e.max_step_tokens = 100, 300, 400
    for k, v in over.items():
        setattr(e, k, v)
    return e


@pytest.mark.parametrize("drafts,kw,says", [
    ([], {}, "at least one sequence"),
    ([(0, [1], [-1]), (0, [1], [-1])], {}, "twice"),
    ([(3, [1], [-1])], {}, "not live"),
    ([(0, [], [])], {}, "at least one token"),
    ([(0, [1, 100], [-1, 0])], {}, "vocabulary"),
    ([(0, [1] * 257, [-1] + [0] * 256)], {}, "up to 256"),
    ([(0, [1, 2], [-1])], {}, "parents"),
    ([(0, [1, 2], [0, 0])], {}, "parents"),
    ([(0, [1, 2], [-1, 1])], {}, "parents"),
    ([(0, [1, 2], [-1, -1])], {}, "parents"),
    ([(0, [1] * 250, [-1] + [0] * 249), (1, [1] * 200, [-1] + [0] * 199)], {}, "exceed a step"),
    ([(0, [1], [-1])], dict(configs=[]), "one sampling config"),
    ([(0, [1, 2], [-1, 0])], dict(configs=["hot"]), "uniform numbers"),
    ([(0, [1, 2], [-1, 0])], dict(configs=["hot"], uniforms=[[0.5]]), "2 tokens deep"),
    ([(0, [1, 2], [-1, 0])], dict(configs=["cold"], uniforms=[[0.5], [0.5]]), "one row of uniform numbers"),
    ([(0, [1, 2], [-1, 0]), (1, [1], [-1])], dict(configs=["cold", "hot"], uniforms=[[0.5, 0.5], None]), "0 uniform numbers"),
])
def test_verify_refuses(drafts, kw, says):
    from lumenllm_b200 import DraftEntry, SamplingConfig, StepError
    e = drafting_engine()
    assert [e.cache.alloc_slot() for _ in range(2)] == [0, 1]
    named = {"hot": SamplingConfig(temperature=0.7), "cold": SamplingConfig()}
    kw = {k: [named.get(x, x) if isinstance(x, str) else x for x in v] for k, v in kw.items()}
    with pytest.raises(StepError, match=says):
        e._validate_drafts([DraftEntry(*d) for d in drafts], kw.get("configs"), kw.get("uniforms"))
    assert e.cache.length(0) == 0 and e.cache.free_tokens() == 640        # nothing was taken


def test_verify_refuses_models_and_long_sequences():
    from lumenllm_b200 import DraftEntry, StepError
    e = drafting_engine()
    e.cache.alloc_slot()
    e.cache.commit(0, 298)
    with pytest.raises(StepError, match="context"):
        e._validate_drafts([DraftEntry(0, [1, 2, 3], [-1, 0, 0])], None, None)
    assert e._validate_drafts([DraftEntry(0, [1, 2], [-1, 0])], None, None) == [[0, 1]]
    e.model.tree_safe = False
    with pytest.raises(StepError, match="no drafts"):
        e._validate_drafts([DraftEntry(0, [1], [-1])], None, None)


def test_which_mixers_take_trees():
    from lumenllm_b200.parts import attention as A
    assert A.GQAttention.tree_safe
    safe = lambda cls, **kw: cls.tree_safe.fget(type("X", (), kw)())
    assert safe(A.WideNormAttention, taps=0, gated=False)
    assert not safe(A.WideNormAttention, taps=4, gated=False) and not safe(A.WideNormAttention, taps=0, gated=True)
    run = type("R", (), {"dtype": BF16})()
    base = dict(chunk=0, gated=False, keep_first=0, padded=False, runtime=run, d=96, dv=64)
    assert safe(A.HeadNormAttention, **base)
    for over in (dict(chunk=64), dict(gated=True), dict(keep_first=4), dict(padded=True)):
        assert not safe(A.HeadNormAttention, **{**base, **over})
    assert safe(A.HeadNormAttention, **{**base, "padded": True, "d": 128})
