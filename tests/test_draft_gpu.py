"""The operators for trees of drafted tokens on the device, against their plain 64-bit forms: sizes that cross page, tile and
segment edges, masks that leave a row empty, values that are no numbers in masked places, lengths beyond the room."""
import math
import random

import pytest
import torch

import plain_draft as D

pytestmark = pytest.mark.gpu

F32, BF16, I32, I64 = torch.float32, torch.bfloat16, torch.int32, torch.int64


def dev(x):
    return x.cuda()


def attend(c, window=0, softcap=0.0, sink=None, layout=None, scale=None, out=None, **over):
    """The library's attention of a Case; layout None: as the library keeps such pages."""
    from lumenllm_b200.cache.kv import tile_layout
    from lumenllm_b200.ops import kernels as K
    k_layout = tile_layout(c.dtype, c.d) if layout is None else layout
    v_layout = tile_layout(c.dtype, c.dv) if layout is None else layout
    kc = D.swizzled(c.kc) if k_layout else c.kc
    vc = D.swizzled(c.vc) if v_layout else c.vc
    a = {n: dev(x) for n, x in {**c.arrays(), **over}.items()}
    q = over.get("q", c.q)
    got = K.attn_tree(dev(q), dev(kc), dev(vc), a["block_table"], a["cu_q"], a["seq_start"], a["tok_seq"], a["tok_pos"], a["tree_mask"],
                      window, c.d ** -0.5 if scale is None else scale, layout=k_layout, v_layout=v_layout, softcap=softcap,
                      sink=False if sink is None else dev(sink), out=out)
    K.check_error_flags()
    return got.cpu()


def close(c, got, rounded=True, **opts):
    ref, size = c.reference(**opts)
    tol = c.bound(ref, size, softcap=opts.get("softcap", 0.0), scale=opts.get("scale"),
                  rounded_weights=rounded and c.dtype == BF16)
    off = (got.double() - ref).abs()
    assert not torch.isnan(got).any()
    assert bool((off <= tol).all()), f"off by {float((off / tol).max()):.2f} of what arithmetic allows"


SIZES = [  # starts, nodes, nq, nkv, d, dv
    ([0], [1], 1, 1, 64, 64),
    ([5, 0, 63, 64, 65], [1, 3, 1, 7, 20], 4, 2, 64, 64),
    ([300, 17, 1000], [9, 33, 64], 8, 2, 128, 128),
    ([700], [33], 32, 8, 128, 128),
    ([130, 250], [64, 128], 5, 1, 128, 128),
    ([4160], [2], 16, 1, 64, 64),
    ([100, 190], [40, 3], 6, 3, 48, 48),
    ([90], [12], 4, 4, 80, 80),
    ([65, 513], [11, 6], 4, 2, 192, 128),
    ([200], [30], 8, 1, 256, 256),
    ([77, 150], [5, 9], 20, 1, 64, 128),
    ([40], [200], 2, 2, 64, 64),
]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("starts,nodes,nq,nkv,d,dv", SIZES)
def test_tree_attention(starts, nodes, nq, nkv, d, dv, dtype):
    c = D.Case(starts, nodes, nq, nkv, d, dv, dtype, seed=len(starts) + d)
    close(c, attend(c))


@pytest.mark.parametrize("dtype,d,dv", [(F32, 37, 21), (BF16, 35, 50), (F32, 512, 512), (BF16, 320, 512), (F32, 1, 1), (F32, 130, 260)])
def test_tree_attention_of_odd_and_wide_heads(dtype, d, dv):
    c = D.Case([70, 3], [6, 18], 4, 2, d, dv, dtype, seed=d)
    close(c, attend(c, layout=0))


@pytest.mark.parametrize("dtype,d", [(BF16, 64), (BF16, 128), (F32, 64), (BF16, 80)])
@pytest.mark.parametrize("window,softcap,sink", [(1, 0.0, False), (7, 0.0, False), (64, 0.0, True), (100, 20.0, False), (500, 30.0, True),
                                                 (0, 5.0, True)])
def test_tree_attention_with_window_cap_and_sink(dtype, d, window, softcap, sink):
    c = D.Case([0, 10, 300, 63], [12, 40, 70, 9], 4, 2, d, dtype=dtype, seed=window + d, q_scale=3.0)
    s = torch.randn(4, generator=torch.Generator().manual_seed(1)) * 3 if sink else None
    close(c, attend(c, window, softcap, s), window=window, softcap=softcap, sink=s)


@pytest.mark.parametrize("dtype,d", [(BF16, 64), (BF16, 128), (BF16, 256), (F32, 64)])
def test_any_mask_and_rows_that_see_nothing(dtype, d):
    """Masks that are no tree's: later nodes, none at all, only others. Without cached tokens an empty mask leaves a row empty."""
    rng = random.Random(3)
    nodes = [10, 70, 4]
    sets = [[set(m for m in range(n) if rng.random() < 0.3) if i % 3 else set() for i in range(n)] for n in nodes]
    for starts in ([0, 0, 0], [0, 100, 3]):
        c = D.Case(starts, nodes, 4, 2, d, dtype=dtype, seed=5, sets=sets)
        got = attend(c)
        close(c, got)
        assert float(got[0].abs().max()) == 0.0          # node 0 of the first sequence sees nothing
        s = torch.tensor([-2.0, 0.0, 1.0, 30.0])
        close(c, attend(c, sink=s), sink=s)


@pytest.mark.parametrize("dtype,d", [(BF16, 64), (BF16, 128), (F32, 64), (BF16, 48)])
@pytest.mark.parametrize("what", [math.nan, math.inf, -math.inf])
def test_masked_numbers_never_reach_a_result(dtype, d, what):
    """A node and a cached token (out of the window) whose keys and values are no numbers: rows that do not see them are as
    before, those that do are not numbers either."""
    c = D.Case([200, 5], [30, 6], 4, 2, d, dtype=dtype, seed=9)
    window = 150
    clean, size = c.reference(window=window)
    hurt = {(0, 203), (0, 10), (1, 5)}                   # node 3 of the first, its token 10, node 0 of the second
    for b, j in hurt:
        c.k[b][j], c.v[b][j] = what, what
    c.fill()
    got = attend(c, window)
    n = 0
    for b, count in enumerate(c.qlens):
        for i in range(count):
            p = c.pos[b][i]
            sees = any(bb == b and ((j >= c.starts[b] and (j - c.starts[b]) in c.sets[b][i]) or (j < c.starts[b] and p - j < window))
                       for bb, j in hurt)
            if sees:
                assert not torch.isfinite(got[n]).any(), (b, i)
            else:
                # the bound without the hurt numbers: the clean case's
                fresh = D.Case([200, 5], [30, 6], 4, 2, d, dtype=dtype, seed=9)
                t = fresh.bound(clean[n], size[n], rounded_weights=dtype == BF16)
                assert bool(((got[n].double() - clean[n]).abs() <= t).all()), (b, i)
            n += 1


@pytest.mark.parametrize("dtype,d", [(BF16, 64), (BF16, 128), (BF16, 80), (F32, 64)])
@pytest.mark.parametrize("window", [0, 150])
def test_masked_numbers_do_not_move_a_bit(dtype, d, window):
    """Large numbers in places that a row does not see, and whatever calls before left in shared memory, under a cap on the scores."""
    case = lambda **kw: D.Case([200, 5], [30, 6], 4, 2, d, dtype=dtype, seed=9, **kw)
    c = case()
    want = attend(c, window, 20.0)
    hurt = {(0, 203), (0, 10), (1, 5)}
    for b, j in hurt:
        c.k[b][j], c.v[b][j] = 300.0, 1e4
    c.fill()
    attend(case(q_scale=1000.0), window, 20.0)
    got = attend(c, window, 20.0)
    n = 0
    for b, count in enumerate(c.qlens):
        for i in range(count):
            p = c.pos[b][i]
            sees = any(bb == b and ((j >= c.starts[b] and (j - c.starts[b]) in c.sets[b][i]) or
                                    (j < c.starts[b] and (not window or p - j < window))) for bb, j in hurt)
            assert sees or torch.equal(got[n], want[n]), (b, i)
            n += 1
    attend(case(q_scale=1000.0), window, 20.0)
    assert torch.equal(attend(case(), window, 20.0), want)


def test_values_alone_that_are_no_numbers():
    """Finite keys with infinite values: a row that sees the key is infinite there and right elsewhere."""
    for dtype, d in ((BF16, 64), (BF16, 128), (F32, 64)):
        c = D.Case([130], [20], 2, 1, d, dtype=dtype, seed=4)
        clean, size = c.reference()
        tol = c.bound(clean, size, rounded_weights=dtype == BF16)
        c.v[0][133, 0, 5], c.v[0][134, 0, 7] = math.inf, math.nan
        c.fill()
        got = attend(c)
        for i in range(20):
            for e, node in ((5, 3), (7, 4)):
                if node in c.sets[0][i]:
                    assert not torch.isfinite(got[i, :, e]).any()
                else:
                    assert bool(((got[i, :, e].double() - clean[i, :, e]).abs() <= tol[i, :, e]).all())
            rest = [e for e in range(d) if e not in (5, 7)]
            assert bool(((got[i].double() - clean[i]).abs() <= tol[i])[:, rest].all())


def test_rows_behind_the_last_sequence_and_wider_tables_change_nothing():
    for dtype, d in ((BF16, 128), (F32, 64)):
        c = D.Case([100, 700], [7, 20], 8, 2, d, dtype=dtype, seed=6)
        want = attend(c)
        a = c.arrays()
        more = 5
        pad = lambda x, v: torch.cat([x, torch.full((more, *x.shape[1:]), v, dtype=x.dtype)])
        wide = torch.full((4, c.width + 9), 12345, dtype=I32)        # entries beyond what is needed are not read
        wide[:2, :c.width] = a["block_table"]
        out = torch.full((27 + more, 8, d), 7.0, dtype=dtype, device="cuda")
        got = attend(c, out=out, q=pad(c.q, 3.0), block_table=wide, tok_seq=pad(a["tok_seq"], 2), tok_pos=pad(a["tok_pos"], 0),
                     tree_mask=pad(a["tree_mask"], -1))
        assert torch.equal(got[:27], want) and bool((got[27:] == 7.0).all())


def test_the_same_step_gives_the_same_bits_and_the_general_kernel_in_any_batch():
    """A step again: the same bits. A sequence alone: the same bits from the general kernel, whose cut of the keys is the
    sequence's own, and within what arithmetic allows from the tensor cores', whose cut is the step's."""
    for dtype, d in ((BF16, 128), (BF16, 64), (F32, 64), (BF16, 48)):
        c = D.Case([1500, 64, 0, 900], [16, 64, 3, 31], 8, 2, d, dtype=dtype, seed=8)
        whole = attend(c)
        assert torch.equal(attend(c), whole)
        ref, size = c.reference()
        tol = c.bound(ref, size, rounded_weights=dtype == BF16)
        n0 = 0
        a = c.arrays()
        for b, n in enumerate(c.qlens):
            alone = attend(c, q=c.q[n0:n0 + n], block_table=a["block_table"][b:b + 1], cu_q=torch.tensor([0, n], dtype=I32),
                           seq_start=a["seq_start"][b:b + 1], tok_seq=torch.zeros(n, dtype=I32), tok_pos=a["tok_pos"][n0:n0 + n],
                           tree_mask=a["tree_mask"][n0:n0 + n])
            if dtype == F32 or d == 48:
                assert torch.equal(alone, whole[n0:n0 + n])
            assert bool(((alone.double() - ref[n0:n0 + n]).abs() <= tol[n0:n0 + n]).all())
            n0 += n


def test_work_dealt_out_over_the_blocks():
    """Steps whose row blocks are cut by many blocks, by none, and by few: long beside empty sequences, more sequences than a
    block has threads."""
    for starts, nodes, nq, nkv, d in (([9000], [3], 2, 1, 64), ([5000, 0, 1, 3000], [1, 2, 200, 64], 4, 1, 128),
                                      ([17 * i % 130 for i in range(400)], [i % 4 for i in range(400)], 2, 2, 64),
                                      ([100] * 40, [60] * 40, 8, 8, 64), ([2500], [256], 16, 1, 256)):
        c = D.Case(starts, nodes, nq, nkv, d, seed=len(starts) + d)
        close(c, attend(c))


@pytest.mark.parametrize("nodes,nq,nkv,d", [(64, 16, 4, 64), (100, 8, 2, 64), (48, 8, 1, 128), (16, 32, 2, 64), (17, 32, 1, 64), (250, 6, 2, 64),
                                            (40, 16, 1, 256)])
def test_row_blocks_of_a_kv_head_side_by_side(nodes, nq, nkv, d):
    """Sequences of different lengths with as many row blocks each (2, 3, 4, 5, 6 and more, the last one not full), cut anywhere."""
    c = D.Case([1500, 30, 777, 2100, 0], [nodes] * 4 + [nodes - 1], nq, nkv, d, dtype=BF16, seed=nodes)
    got = attend(c)
    close(c, got)
    assert torch.equal(got, attend(c))
    c = D.Case([900, 64, 1300], [nodes] * 3, nq, nkv, d, dtype=BF16, seed=nodes + 1)
    close(c, attend(c, 300), window=300)


def test_lengths_and_pages_that_cannot_be_are_held_inside_the_arrays():
    """Lengths below 0 or beyond the page table, pages that are not there, cu_q beyond the tokens: no fault, and the
    sequences beside them are right."""
    for dtype, d in ((BF16, 128), (F32, 64)):
        c = D.Case([100, 200, 300], [7, 9, 5], 4, 2, d, dtype=dtype, seed=7)
        want = attend(c)
        c.kc[0], c.vc[0] = 0.0, 0.0                      # what a page that is not there reads
        a = c.arrays()
        table = a["block_table"].clone()
        table[1] = torch.tensor([-5, 10 ** 9, c.n_pages, -(1 << 31)] + [1 << 30] * (c.width - 4), dtype=I32)
        start = a["seq_start"].clone()
        start[1] = 10 ** 9
        ref, size = c.reference()
        tol = c.bound(ref, size, rounded_weights=dtype == BF16)
        right = lambda got: bool(((got.double() - ref).abs() <= tol)[[i for i in range(21) if not 7 <= i < 16]].all())
        assert right(want)
        assert right(attend(c, block_table=table, seq_start=start))
        start[1] = -(1 << 31)
        assert right(attend(c, block_table=table, seq_start=start, cu_q=torch.tensor([0, 7, 16, 1 << 30], dtype=I32)))


def test_long_caches_beyond_32_bits():
    """Tiles whose offset in the cache passes 2^32 bytes and 2^31 numbers."""
    from lumenllm_b200.ops import kernels as K
    for dtype, d in ((BF16, 128), (F32, 128)):
        c = D.Case([150], [6], 2, 1, d, dtype=dtype, seed=2)
        want = attend(c)
        pages = (1 << 31) // (64 * d) + 8
        kc = torch.empty((pages, 1, 64, d), dtype=dtype, device="cuda")
        vc = torch.empty((pages, 1, 64, d), dtype=dtype, device="cuda")
        layout = 1 if dtype == BF16 else 0
        table = c.table.clone()
        for w in range(c.width):
            to = pages - 1 - w
            src = int(c.table[0, w])
            kc[to], vc[to] = (dev(D.swizzled(x[src]) if layout else x[src]) for x in (c.kc, c.vc))
            table[0, w] = to
        a = {n: dev(x) for n, x in c.arrays().items()}
        got = K.attn_tree(dev(c.q), kc, vc, dev(table), a["cu_q"], a["seq_start"], a["tok_seq"], a["tok_pos"], a["tree_mask"], 0,
                          d ** -0.5, layout=layout)
        assert torch.equal(got.cpu(), want)
        before = kc[pages - 1].clone()
        K.cache_compact(kc, vc, dev(table), a["seq_start"], dev(torch.tensor([[0, 5]], dtype=I32)), dev(torch.tensor([2], dtype=I32)),
                        layout=layout)
        x = c.kc[int(c.table[0, 2])].clone()
        x[0, 151 % 64] = c.k[0][155, 0]
        x = D.swizzled(x) if layout else x
        rows = ~torch.isnan(x)                           # rows behind the end hold nothing
        assert torch.equal(kc[table[0, 2].item()].cpu()[rows], x[rows]) and torch.equal(kc[pages - 1], before)
        del kc, vc


@pytest.mark.parametrize("B,width,most,tree,words", [(1, 1, 1, True, 1), (3, 5, 9, True, 1), (40, 33, 64, True, 1), (7, 20, 256, True, 4),
                                                     (5, 1030, 200, True, 4), (300, 3, 5, False, 1), (2, 40, 900, False, 1)])
def test_step_tables(B, width, most, tree, words):
    from lumenllm_b200.ops import kernels as K
    rng = random.Random(B + width)
    starts = [rng.choice([0, 1, 63, 64, rng.randint(0, width * 64)]) for _ in range(B)]
    qlens = [rng.choice([0, 1, most, rng.randint(1, most)]) for _ in range(B)]
    slots = [rng.randint(-1, B + 1) for _ in range(B)]
    pages = [[rng.randint(1, 1 << 20) for _ in range(width + 2)] for _ in range(B + 1)]
    room = sum(min(q, max(0, width * 64 - s), 64 * words if tree else 1 << 30) for s, q in zip(starts, qlens))
    for N in {room, room + 5, max(0, room - 3), 0}:
        parents = [rng.choice([-1, 0, -7, 1 << 30, rng.randint(0, most)]) for _ in range(N)] if tree else None
        t = lambda x: torch.tensor(x, dtype=I32, device="cuda")
        got = K.step_tables(t(starts), t(qlens), t(pages), t(slots), N, width, parents=t(parents) if tree else None, mask_words=words)
        want = D.tables(starts, qlens, pages, slots, N, width, parents, words)
        for name, g, w in zip(got._fields, (got.cu_q, got.tok_seq, got.cache_pos, got.tok_pos, got.slot_map, got.block_table, got.tree_mask),
                              want):
            if w is None:
                assert g is None
            else:
                assert g.dtype == w.dtype and torch.equal(g.cpu(), w), name


def test_step_tables_of_lengths_that_cannot_be():
    from lumenllm_b200.ops import kernels as K
    t = lambda x: torch.tensor(x, dtype=I32, device="cuda")
    starts, qlens, slots = [-5, 10 ** 9, 100, -(1 << 31)], [3, 5, -2, (1 << 31) - 1], [0, 1, 7, -(1 << 31)]
    pages = [[3, 4, 5], [6, 7, 8]]
    wide = t([[3, 4, 5, 0, 0], [6, 7, 8, 0, 0]])[:, :3]           # rows of a wider table
    got = K.step_tables(t(starts), t(qlens), wide, t(slots), 200, 3, parents=t([0] * 200), mask_words=1)
    want = D.tables(starts, qlens, pages, slots, 200, 3, [0] * 200, 1)
    for g, w in zip((got.cu_q, got.tok_seq, got.cache_pos, got.tok_pos, got.slot_map, got.block_table, got.tree_mask), want):
        assert torch.equal(g.cpu(), w)


@pytest.mark.parametrize("B,most_nodes,most", [(1, 1, 1), (1, 8, 8), (33, 20, 3), (5, 256, 256), (6, 300, 40), (64, 64, 64)])
def test_acceptance(B, most_nodes, most):
    from lumenllm_b200.ops import kernels as K
    rng = random.Random(B + most_nodes)
    picked, tokens, parents, cu = [], [], [], [0]
    for b in range(B):
        n = rng.choice([0, 1, most_nodes, rng.randint(1, most_nodes)])
        parents += [rng.choice([i - 1, rng.randint(max(0, i - 4), i)]) if i and rng.random() < 0.95 else rng.choice([-1, -9, i, 1 << 30])
                    for i in range(n)]
        tokens += [rng.randint(0, 2) for _ in range(n)]       # few tokens: equal children are common
        picked += [rng.randint(0, 2) for _ in range(n)]
        cu.append(cu[-1] + n)
    t = lambda x: torch.tensor(x, dtype=I32, device="cuda")
    count, path, emitted = K.tree_accept(t(picked), t(tokens), t(parents), t(cu), most)
    want = D.accept(picked, tokens, parents, cu, most)
    for g, w in zip((count, path, emitted), want):
        assert g.tolist() == w


@pytest.mark.parametrize("dtype,d,dv,swizzle", [(BF16, 64, 64, True), (BF16, 128, 192, True), (BF16, 48, 48, False), (F32, 64, 64, False),
                                                (BF16, 33, 21, False), (F32, 7, 9, False), (BF16, 576, None, False)])
def test_cache_move(dtype, d, dv, swizzle):
    from lumenllm_b200.ops import kernels as K
    rng, g = random.Random(d), torch.Generator().manual_seed(d)
    layers, nkv, width, B, most = 3, 2, 3, 5, 40
    pages = B * width + 1
    kc = torch.randn(layers, pages, nkv, 64, d, generator=g).to(dtype)
    vc = torch.randn(layers, pages, nkv, 64, dv, generator=g).to(dtype) if dv else None
    table = torch.tensor(rng.sample(range(1, pages), B * width), dtype=I32).view(B, width)
    starts = [0, 60, 63, 64, 100]
    counts = [0, 1, most, 7, 12]
    path = torch.full((B, most), -1, dtype=I32)
    for b, n in enumerate(counts):
        # runs that stay, neighbours, and sources that earlier moves of the path have written over
        p = [0] + sorted(rng.sample(range(1, 80 if b != 2 else 50), n - 1)) if n else []
        path[b, :n] = torch.tensor(p, dtype=I32)
    path[3, :7] = torch.tensor([0, 1, 2, 4, 5, 6, 9])
    want = [kc.clone(), vc.clone() if dv else None]
    for x, src in zip(want, (kc, vc)):
        if x is None:
            continue
        for b, n in enumerate(counts):
            for k in range(1, n):
                i, j = starts[b] + int(path[b, k]), starts[b] + k
                x[:, table[b, j // 64], :, j % 64] = src[:, table[b, i // 64], :, i % 64]
    s = (lambda x: D.swizzled(x)) if swizzle else (lambda x: x)
    got = [dev(s(kc)), dev(s(vc)) if dv else None]
    K.cache_compact(got[0], got[1], dev(table), dev(torch.tensor(starts, dtype=I32)), dev(path), dev(torch.tensor(counts, dtype=I32)),
                    layout=1 if swizzle else 0)
    for x, w in zip(got, want):
        assert x is None or torch.equal(x.cpu(), s(w))


def test_paths_that_cannot_be_end_where_they_break():
    from lumenllm_b200.ops import kernels as K
    kc = torch.arange(1 * 6 * 1 * 64 * 4, dtype=F32).view(6, 1, 64, 4)
    table = torch.tensor([[1, 2], [3, 4], [5, 99], [-1, 1]], dtype=I32)
    starts, counts = [0, 100, 60, 0], [4, 5, 4, 3]
    path = torch.tensor([[0, 5, 5, 9, 0], [0, 3, 5, 1 << 30, 29], [0, 2, 6, 7, 9], [0, 2, 3, 4, 5]], dtype=I32)
    want = kc.clone()
    want[1, 0, 1] = kc[1, 0, 5]                  # then a number that does not rise
    want[4, 0, 37], want[4, 0, 38] = kc[4, 0, 39], kc[4, 0, 41]      # then one behind the table
    want[5, 0, 61] = kc[5, 0, 62]                # then a page that is not there; the last sequence's first page is none
    got = kc.cuda()
    K.cache_compact(got, None, table.cuda(), torch.tensor(starts, dtype=I32).cuda(), path.cuda(), torch.tensor(counts, dtype=I32).cuda())
    assert torch.equal(got.cpu(), want)


def test_the_operators_together_and_in_a_graph():
    """A step of drafted tokens as a user puts it together, twice with other lengths through one captured graph."""
    from lumenllm_b200.ops import kernels as K
    g = torch.Generator().manual_seed(0)
    B, nkv, nq, d, width, N = 3, 2, 4, 64, 6, 40
    slot_pages = (torch.randperm(5 * width, generator=g) + 1).to(I32).view(5, width).cuda()
    kc = torch.randn(2, 5 * width + 1, nkv, 64, d, generator=g).to(BF16).cuda()
    vc = torch.randn(2, 5 * width + 1, nkv, 64, d, generator=g).to(BF16).cuda()
    q = torch.randn(N, nq, d, generator=g).to(BF16).cuda()
    t = lambda x: torch.tensor(x, dtype=I32, device="cuda")
    rng = random.Random(1)
    tokens, picked = t([rng.randint(0, 2) for _ in range(N)]), t([rng.randint(0, 2) for _ in range(N)])

    def inputs(starts, qlens, slots):
        parents = [p for n in qlens for p in D.random_tree(rng, n)]
        return t(starts), t(qlens), t(slots), t(parents + [0] * (N - len(parents)))

    def step(start, qlen, slot, parents):
        s = K.step_tables(start, qlen, slot_pages, slot, N, width, parents=parents)
        out = torch.zeros_like(q)
        o = [K.attn_tree(q, kc[i], vc[i], s.block_table, s.cu_q, start, s.tok_seq, s.tok_pos, s.tree_mask, 0, d ** -0.5, layout=1,
                         out=torch.zeros_like(q)) for i in range(2)]
        count, path, said = K.tree_accept(picked, tokens, parents, s.cu_q, 16)
        K.cache_compact(kc, vc, s.block_table, start, path, count, layout=1)
        return [*o, count, path, said, s.cu_q, s.block_table, s.tok_pos, s.tree_mask]

    a, b = inputs([100, 0, 250], [16, 9, 15], [3, 0, 1]), inputs([10, 300, 64], [5, 30, 1], [2, 4, 0])
    k0, v0 = kc.clone(), vc.clone()
    want = []
    for x in (a, b):
        want.append([y.clone() for y in step(*x)] + [kc.clone(), vc.clone()])
    K.check_error_flags()
    kc.copy_(k0), vc.copy_(v0)
    held = [x.clone() for x in a]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):                # another stream than the tensors' own
        step(*held)
    torch.cuda.current_stream().wait_stream(side)
    kc.copy_(k0), vc.copy_(v0)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(*held)
    kc.copy_(k0), vc.copy_(v0)
    for x, w in zip((a, b), want):
        for h, y in zip(held, x):
            h.copy_(y)
        graph.replay()
        for g_, w_ in zip([*outs, kc, vc], w):
            assert torch.equal(g_, w_)
    K.check_error_flags()


def test_tree_attention_wherever_the_operands_lie():
    """Queries and outputs that begin anywhere, page tables with longer rows, negative and zero scales, a window beyond any position."""
    from lumenllm_b200.ops import kernels as K
    for dtype, d in ((BF16, 128), (BF16, 64), (F32, 64), (F32, 36)):
        c = D.Case([70, 200], [9, 33], 4, 2, d, dtype=dtype, seed=12)
        ref, size = c.reference()
        tol = c.bound(ref, size, rounded_weights=dtype == BF16)
        a = {n: dev(x) for n, x in c.arrays().items()}
        layout = 1 if dtype == BF16 else 0
        kc, vc = (dev(D.swizzled(x) if layout else x) for x in (c.kc, c.vc))
        wide = torch.full((2, c.width + 5), -1, dtype=I32, device="cuda")
        wide[:, :c.width] = a["block_table"]
        n = c.q.numel()
        for off, out_off in ((0, 0), (8, 0), (1, 0), (0, 8), (0, 1), (3, 5)):
            q = torch.empty((n + off,), dtype=dtype, device="cuda")[off:].view(c.q.shape).copy_(c.q)
            out = torch.empty((n + out_off,), dtype=dtype, device="cuda")[out_off:].view(c.q.shape)
            got = K.attn_tree(q, kc, vc, wide[:, :c.width], a["cu_q"], a["seq_start"], a["tok_seq"], a["tok_pos"], a["tree_mask"], 1 << 40,
                              d ** -0.5, layout=layout, out=out)
            assert got.data_ptr() == out.data_ptr() and bool(((got.cpu().double() - ref).abs() <= tol).all())
        for scale in (-0.25, 0.0):
            close(c, attend(c, scale=scale), scale=scale)
        close(c, attend(c, window=(1 << 31) - 1), window=(1 << 31) - 1)
    K.check_error_flags()


def test_more_nodes_than_masks_cover_and_lengths_that_contradict_one_another():
    from lumenllm_b200.ops import kernels as K
    for dtype, d in ((BF16, 64), (F32, 64)):
        # 300 nodes: the masks name the first 256, the others see those and are seen by nobody
        sets = [[set(m for m in range(0, min(i, 256), 7)) | ({i} if i < 256 else set()) for i in range(300)]]
        c = D.Case([40], [300], 2, 1, d, dtype=dtype, seed=3, words=4, sets=sets)
        close(c, attend(c))
        # sequences that claim the same tokens over and over: no fault, no wait that runs out
        c = D.Case([100] * 6, [5] * 6, 2, 1, d, dtype=dtype, seed=4)
        attend(c, cu_q=torch.tensor([0, 30, 0, 30, 0, 1 << 30, -5], dtype=I32))
        K.check_error_flags()


def test_two_streams_at_once():
    """Calls on two streams share nothing: the results are those of calls one behind the other."""
    from lumenllm_b200.ops import kernels as K
    cases = [D.Case([900, 50], [30, 7], 8, 2, 128, seed=s) for s in (1, 2)]
    want = [attend(c) for c in cases]
    held = []
    for c in cases:
        a = {n: dev(x) for n, x in c.arrays().items()}
        held.append((dev(c.q), dev(D.swizzled(c.kc)), dev(D.swizzled(c.vc)), a))
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            q, kc, vc, a = held[i]
            with torch.cuda.stream(s):
                got[i].append(K.attn_tree(q, kc, vc, a["block_table"], a["cu_q"], a["seq_start"], a["tok_seq"], a["tok_pos"],
                                          a["tree_mask"], 0, 128 ** -0.5, layout=1))
    torch.cuda.synchronize()
    for i, w in enumerate(want):
        assert all(torch.equal(x.cpu(), w) for x in got[i])
    K.check_error_flags()


def test_empty_steps():
    from lumenllm_b200.ops import kernels as K
    t = lambda *x: torch.tensor(x, dtype=I32, device="cuda")
    none = torch.empty((0,), dtype=I32, device="cuda")
    kc = torch.zeros((2, 1, 64, 64), dtype=BF16, device="cuda")
    got = K.step_tables(none, none, t(1, 2).view(1, 2), none, 3, 2, parents=t(0, 0, 0))
    assert got.cu_q.tolist() == [0] and got.tok_seq.tolist() == [0] * 3 and got.block_table.tolist() == [[0, 0]]
    q = torch.zeros((0, 2, 64), dtype=BF16, device="cuda")
    mask = torch.zeros((0, 1), dtype=I64, device="cuda")
    assert K.attn_tree(q, kc, kc, t(1, 1).view(1, 2), t(0, 0), t(5), none, none, mask, 0, 1.0, layout=1).shape == (0, 2, 64)
    out = torch.full((3, 2, 64), 2.0, dtype=BF16, device="cuda")
    q = torch.zeros((3, 2, 64), dtype=BF16, device="cuda")
    mask = torch.zeros((3, 1), dtype=I64, device="cuda")
    K.attn_tree(q, kc, kc, t(1, 1).view(1, 2), t(0, 0), t(5), t(0, 0, 0), t(0, 0, 0), mask, 0, 1.0, layout=1, out=out)      # nobody's tokens
    assert bool((out == 2.0).all())
    count, path, said = K.tree_accept(none, none, none, t(0), 4)
    assert count.shape == (0,) and path.shape == (0, 4) and said.shape == (0, 4)
    K.cache_compact(kc, kc, t(1, 1).view(1, 2), t(0), path, count, layout=1)


@pytest.mark.parametrize("args", [["--batch", "2", "--len", "200"], ["--batch", "1", "--len", "70", "--nodes", "130"],
                                  ["--batch", "2", "--len", "100", "--nodes", "5", "--head-dim", "80"]])
def test_the_micro_benchmark_runs_tree_attention(args, capsys):
    from lumenllm_b200 import kbench
    kbench.main(["attn_tree", *args, "--copies", "2", "--reps", "1"])
    line = capsys.readouterr().out.strip().splitlines()[-1]
    assert line.startswith("attn_tree:") and "us per launch" in line
