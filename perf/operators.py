"""The operators that check a tree of drafted tokens over the paged cache, as cases that a program can prepare,
run and time.

One step of a server that drafts: the tables of the step are built from the requests' lengths ("tables"), the
drafted tokens' queries attend to the cache and to their own ancestors ("attend"), the drafts that the model agrees
with are accepted ("accept"), and the accepted tokens' keys and values move to where the next step expects
them ("compact").

Sequence b has `start` cached tokens and brings `q` nodes of a tree, node i with a parent among the nodes
before it (-1: the last cached token). A cache page holds 64 tokens, [kv heads][64][dim]; bfloat16 pages whose dim is
a multiple of 64 are kept as [dim / 64][64][64] with the 16-byte chunk c of row r at c ^ (r & 7).
"""
import math
import random

import numpy as np
import torch

own = False

PAGE = 64
DTYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}


def listed():
    qwen = dict(op="attend", dtype="bfloat16", heads=32, kv=8, dim=128, window=0, softcap=0.0, sink=False)
    return [
        # one user's draft of a few tokens: nothing but latency
        dict(name="tables_1", op="tables", batch=1, low=1300, high=1300, nodes=9, width=32, tree=True),
        # a full server, every request with room for 131,072 tokens
        dict(name="tables_256", op="tables", batch=256, low=200, high=130000, nodes=64, width=2048, tree=True),
        # one user again, after a usual context: a short read of the cache
        dict(qwen, name="attend_1x8", batch=1, low=1300, high=1300, nodes=8),
        # the headline's batch with large trees, where products weigh as much as the cache's bytes
        dict(qwen, name="attend_8x64", batch=8, low=4000, high=6000, nodes=64),
        # a full server with small trees: the cache's bytes
        dict(qwen, name="attend_64x16", batch=64, low=1024, high=1700, nodes=16),
        # long contexts for two users: one sequence over many blocks
        dict(qwen, name="attend_2_long", batch=2, low=24000, high=30000, nodes=32),
        # heads of 64 under a window, with capped scores and a learned sink
        dict(qwen, name="attend_window", batch=16, low=700, high=5000, nodes=24, heads=16, kv=4, dim=64, window=1024,
             softcap=30.0, sink=True),
        # the true 32-bit path, which numerics are checked with
        dict(qwen, name="attend_float32", dtype="float32", batch=4, low=300, high=2000, nodes=13, heads=16, kv=4),
        # one user's walk, and a full server's
        dict(name="accept_1", op="accept", batch=1, nodes=8),
        dict(name="accept_256", op="accept", batch=256, nodes=64),
        # all layers of the 8B shape for the headline's batch; a full server's trees
        dict(name="compact_8", op="compact", dtype="bfloat16", batch=8, layers=36, kv=8, dim=128, nodes=16, most=5),
        dict(name="compact_64", op="compact", dtype="bfloat16", batch=64, layers=12, kv=8, dim=128, nodes=40, most=9),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["tables", "attend", "attend", "attend", "attend", "accept", "compact"])
    if op == "tables":
        width = _log(rng, 8, 2048)
        low = _log(rng, 1, width * PAGE // 2)
        return dict(op=op, batch=_log(rng, 1, 256), low=low, high=rng.randint(low, width * PAGE - 256), nodes=_log(rng, 1, 250),
                    width=width, tree=rng.random() < 0.8)
    if op == "accept":
        return dict(op=op, batch=_log(rng, 1, 256), nodes=_log(rng, 1, 64))
    if op == "compact":
        dtype = rng.choice(["bfloat16", "bfloat16", "float32"])
        return dict(op=op, dtype=dtype, batch=_log(rng, 1, 32), layers=_log(rng, 1, 12), kv=rng.choice([1, 2, 4, 8]),
                    dim=rng.choice([48, 64, 80, 128, 192, 256]), nodes=rng.randint(16, 64), most=rng.randint(1, 8))
    dtype = rng.choice(["bfloat16", "bfloat16", "bfloat16", "float32"])
    kv, group = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 4, 5, 8])
    dim = rng.choice([64, 128, 128, 256] if dtype == "bfloat16" and rng.random() < 0.8 else [48, 80, 112, 128])
    heads = kv * group
    nodes = _log(rng, 1, 100)
    most = 2.0e10 if dtype == "bfloat16" and dim % 64 == 0 else 1.0e9     # operations of a whole pass
    tokens = min(0.9e5 * 8 * 128 / (kv * dim), most / (4.0 * nodes * heads * dim))
    batch = _log(rng, 1, 64)
    high = max(2, min(32000, int(tokens / batch)))
    low = rng.choice([0, high // 4, high // 2, high - 1, _log(rng, 1, high)])
    return dict(op=op, dtype=dtype, batch=batch, low=low, high=high, nodes=nodes, heads=heads, kv=kv, dim=dim,
                window=rng.choice([0, 0, 0, _log(rng, 4, 2048)]), softcap=rng.choice([0.0, 0.0, 30.0]), sink=rng.random() < 0.3)


# ---------------------------------------------------------------- inputs

def _tree(rng, q):
    """Parents of q nodes: the first is the token that is certain, the others' parents lie close behind it or them."""
    return [-1] + [max(0, i - 1 - min(int(rng.expovariate(0.5)), i - 1)) for i in range(1, q)]


def _spread(rng, low, high, n):
    """n whole numbers that fill low..high evenly, in an order of the seed's."""
    out = [low + (high - low) * (2 * i + 1) // (2 * n) for i in range(n)]
    rng.shuffle(out)
    return out


def _ancestors(parents):
    anc, depth = [], []
    for i, p in enumerate(parents):
        anc.append((1 << i) | (anc[p] if p >= 0 else 0))
        depth.append(depth[p] + 1 if p >= 0 else 0)
    return anc, depth


def _int(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device="cuda")


def _words(anc, words):
    full = (1 << 64) - 1
    out = [[(a >> (64 * w)) & full for w in range(words)] for a in anc]
    return torch.from_numpy(np.array(out, dtype=np.uint64).reshape(-1, words).view(np.int64)).cuda()


def _swizzled(dtype, dim):
    return dtype == torch.bfloat16 and dim % 64 == 0


def _aligned(shape, dtype):
    """An empty tensor on a 1,024-byte boundary, as a cache has it."""
    size = torch.empty((), dtype=dtype).element_size() * int(np.prod(shape))
    raw = torch.empty((size + 1024,), dtype=torch.uint8, device="cuda")
    at = -raw.data_ptr() % 1024
    return raw[at:at + size].view(dtype).view(shape)


def _random_cache(shape, dtype, gen, mean=0.0):
    out = _aligned(shape, dtype)
    out.normal_(generator=gen)
    return out.add_(mean) if mean else out


def prepare(case, seed):
    rng, op = random.Random(seed), case["op"]
    gen = torch.Generator("cuda")
    gen.manual_seed(seed)
    s = {"case": case}
    B = case["batch"]
    if op in ("tables", "attend"):
        start = _spread(rng, case["low"], case["high"], B)
    if op == "tables":
        width, slots = case["width"], B + 3
        qlen = _spread(rng, 1, case["nodes"], B)
        s["parents"] = _int([p for q in qlen for p in _tree(rng, q)]) if case["tree"] else None
        pages = torch.randperm(slots * width, generator=gen, device="cuda").to(torch.int32)
        s["slot_pages"] = (pages + 1).view(slots, width)
        s["seq_slot"] = _int(rng.sample(range(slots), B))
        s["seq_start"], s["seq_qlen"] = _int(start), _int(qlen)
        s["n_tokens"], s["words"] = sum(qlen), -(-case["nodes"] // 64)
        return s
    if op == "accept":
        parents, tokens, picked, cu = [], [], [], [0]
        for q in _spread(rng, (case["nodes"] + 1) // 2, case["nodes"] + 1, B):
            tree = _tree(rng, q)
            tok = [rng.randrange(151936) for _ in range(q)]
            pick = [rng.randrange(151936) for _ in range(q)]
            for i, p in enumerate(tree):
                if p >= 0 and rng.random() < 0.6:        # a draft that the model agrees with
                    pick[p] = tok[i]
            parents += tree
            tokens += tok
            picked += pick
            cu.append(cu[-1] + q)
        return dict(s, parents=_int(parents), tokens=_int(tokens), picked=_int(picked), cu_q=_int(cu))
    dtype, kv, dim = DTYPES[case["dtype"]], case["kv"], case["dim"]
    if op == "compact":
        start = [rng.randint(1, 2 * PAGE) for _ in range(B)]
        width, most = -(-(2 * PAGE + case["nodes"]) // PAGE), case["most"]
        n = B * width + 1
        shape = (case["layers"], n, kv, PAGE, dim)
        s["k"], s["v"] = _random_cache(shape, dtype, gen), _random_cache(shape, dtype, gen)
        order = torch.randperm(n - 1, generator=gen, device="cuda").to(torch.int32) + 1
        s["block_table"], s["seq_start"] = order.view(B, width), _int(start)
        count = _spread(rng, 0, most + 1, B)
        # a tree whose first nodes are all children of the certain token: the accepted ones lie behind them
        path = [([0] + sorted(rng.sample(range(most, case["nodes"]), c - 1)) if c else []) + [-1] * (most - c) for c in count]
        return dict(s, path=_int(path), count=_int(count))
    q = _spread(rng, (case["nodes"] + 1) // 2, case["nodes"] + 1, B)
    lens = [a + b for a, b in zip(start, q)]
    width, words = max(-(-x // PAGE) for x in lens), -(-case["nodes"] // 64)
    n = sum(-(-x // PAGE) for x in lens) + 1
    s["k"] = _random_cache((n, kv, PAGE, dim), dtype, gen)
    s["v"] = _random_cache((n, kv, PAGE, dim), dtype, gen, 0.25)
    order = (torch.randperm(n - 1, generator=gen, device="cuda").to(torch.int32) + 1).tolist()
    table, anc, pos, cu, seq = [], [], [], [0], []
    for b in range(B):
        held = -(-lens[b] // PAGE)
        table.append(order[:held] + [0] * (width - held))
        order = order[held:]
        a, depth = _ancestors(_tree(rng, q[b]))
        anc += a
        pos += [start[b] + x for x in depth]
        cu.append(cu[-1] + q[b])
        seq += [b] * q[b]
    s["q"] = torch.randn((cu[-1], case["heads"], dim), generator=gen, device="cuda").mul_(2.0).to(dtype)
    s["sink"] = torch.randn((case["heads"],), generator=gen, device="cuda") if case["sink"] else None
    return dict(s, block_table=_int(table), cu_q=_int(cu), seq_start=_int(start), tok_seq=_int(seq), tok_pos=_int(pos),
                mask=_words(anc, words), scale=1.0 / math.sqrt(dim), nodes=case["nodes"], longest=max(lens))


# ---------------------------------------------------------------- plain forms

def _plain_tables(s):
    N, words, width = s["n_tokens"], s["words"], s["case"]["width"]
    start, table = s["seq_start"].long().clamp(0, width * PAGE), s["slot_pages"].long()
    B = start.shape[0]
    q = torch.minimum(s["seq_qlen"].long(), width * PAGE - start).clamp(min=0)
    cu = torch.cat([q.new_zeros(1), q.cumsum(0)]).clamp(max=N)
    n = torch.arange(N, device="cuda")
    seq = (n[:, None] >= cu[None, 1:]).sum(1)
    live = seq < B
    b = seq.clamp(max=B - 1)
    i = n - cu[b]
    pos = torch.where(live, start[b] + i, 0)
    held = torch.arange(width, device="cuda")[None] * PAGE < (start + q)[:, None]
    rows = torch.where(held, table[s["seq_slot"].long()], 0)
    block_table = torch.cat([rows, rows.new_zeros(1, width)])
    slot_map = torch.where(live, block_table[seq, pos // PAGE] * PAGE + pos % PAGE, -1)
    out = dict(cu_q=cu.int(), tok_seq=seq.int(), cache_pos=pos.int(), slot_map=slot_map, block_table=block_table.int())
    if s["parents"] is None:
        return dict(out, tok_pos=pos.int())
    M = words * 64
    up = torch.full((B + 1, M), -1, device="cuda")
    up[seq, i.clamp(0, M - 1)] = s["parents"].long()
    anc = torch.eye(M, dtype=torch.bool, device="cuda").expand(B + 1, M, M)
    for _ in range(max(1, (M - 1).bit_length())):
        there = up >= 0
        at = up.clamp(min=0)
        anc = anc | (torch.gather(anc, 1, at[:, :, None].expand(-1, -1, M)) & there[:, :, None])
        up = torch.where(there, torch.gather(up, 1, at), -1)
    mine = anc[seq, i.clamp(0, M - 1)]
    bits = (mine.view(N, words, 64).long() << torch.arange(64, device="cuda")).sum(2)
    return dict(out, tok_pos=(start[b] + mine.sum(1) - 1).int(), tree_mask=bits)


def _plain_rows(cache):
    """[..., pages, kv, 64, dim] with the rows' numbers in order."""
    dim = cache.shape[-1]
    if not _swizzled(cache.dtype, dim):
        return cache
    x = cache.view(*cache.shape[:-2], dim // 64, PAGE, 8, 8)
    chunk = torch.arange(8, device="cuda")[None, :] ^ (torch.arange(PAGE, device="cuda")[:, None] & 7)
    x = torch.gather(x, -2, chunk[:, :, None].expand(PAGE, 8, 8).expand_as(x))
    return x.transpose(-4, -3).reshape(cache.shape)


def _plain_attend(s):
    c, q, M = s["case"], s["q"], s["nodes"]
    N, heads, dim = q.shape
    B, kv = c["batch"], c["kv"]
    cu, start, seq = s["cu_q"].long(), s["seq_start"].long(), s["tok_seq"].long()
    i = torch.arange(N, device="cuda") - cu[seq]
    used = s["block_table"].long()
    L = used.shape[1] * PAGE
    keys, values = (_plain_rows(x[used]).float().transpose(2, 3).reshape(B, L, kv, dim) for x in (s["k"], s["v"]))
    # each row's place in [B, M]
    place = torch.zeros((B, M), dtype=torch.long, device="cuda")
    place[seq, i] = torch.arange(N, device="cuda")
    j = torch.arange(L, device="cuda")
    p = s["tok_pos"].long()[place]
    word = s["mask"][place]                                     # [B, M, words]
    node = j[None, :] - start[:, None]                          # [B, L]
    at = node.clamp(0, M - 1)
    bit = (torch.gather(word, 2, (at // 64)[:, None, :].expand(B, M, L)) >> (at % 64)[:, None, :]) & 1
    count = (cu[1:] - cu[:-1])[:, None]
    is_node = (node >= 0) & (node < count)
    seen = torch.where(is_node[:, None, :], bit == 1, (node < 0)[:, None, :])
    if c["window"]:
        key_pos = torch.where(is_node, torch.gather(p, 1, at), j[None, :])
        seen = seen & (p[:, :, None] - key_pos[:, None, :] < c["window"])
    queries = q.float()[place].view(B, M, kv, heads // kv, dim)
    x = torch.matmul(queries.permute(0, 2, 3, 1, 4).reshape(B, kv, -1, dim), keys.permute(0, 2, 3, 1))
    x = x.view(B, kv, heads // kv, M, L) * s["scale"]
    if c["softcap"]:
        x = c["softcap"] * torch.tanh(x / c["softcap"])
    x = torch.where(seen[:, None, None], x, -math.inf)
    top = x.amax(-1, keepdim=True)
    if s["sink"] is not None:
        sink = s["sink"].view(1, kv, heads // kv, 1, 1)
        top = torch.maximum(top, sink)
    top = torch.where(top == -math.inf, 0.0, top)
    e = torch.exp(x - top)
    total = e.sum(-1, keepdim=True)
    if s["sink"] is not None:
        total = total + torch.exp(sink - top)
    values = torch.where((j[None, :] < start[:, None] + count)[:, :, None, None], values, 0.0)
    o = torch.matmul(e.view(B, kv, -1, L), values.transpose(1, 2)).view(B, kv, heads // kv, M, dim)
    o = torch.where(total > 0, o / total, 0.0)
    return o.permute(0, 3, 1, 2, 4).reshape(B, M, heads, dim)[seq, i].to(q.dtype)


def _plain_accept(s):
    cu, up, tokens, picked, M = s["cu_q"].long(), s["parents"].long(), s["tokens"], s["picked"], s["case"]["nodes"]
    B, N = cu.shape[0] - 1, up.shape[0]
    n = torch.arange(N, device="cuda")
    seq = (n[:, None] >= cu[None, 1:]).sum(1)
    i = n - cu[seq]
    agreed = (up >= 0) & (tokens == picked[cu[seq] + up.clamp(min=0)])
    child = torch.full((B, M + 1), M, device="cuda")            # the lowest child that is agreed with
    child.view(-1).scatter_reduce_(0, seq * (M + 1) + torch.where(agreed, up, M), torch.where(agreed, i, M), "amin")
    cur = torch.where(cu[1:] > cu[:-1], 0, M)
    path = []
    for _ in range(M):
        path.append(cur)
        cur = torch.gather(child, 1, cur[:, None])[:, 0]
    path = torch.stack(path, 1)
    there = path < M
    emitted = torch.where(there, picked[(cu[:-1, None] + path).clamp(max=N - 1)], -1)
    return dict(count=there.sum(1).int(), path=torch.where(there, path, -1).int(), emitted=emitted)


def _plain_compact(s):
    count, path, start, table = s["count"].long(), s["path"].long(), s["seq_start"].long(), s["block_table"].long()
    most = path.shape[1]
    k = torch.arange(most, device="cuda").expand_as(path)
    moved = (k > 0) & (k < count[:, None])
    b, k = moved.nonzero(as_tuple=True)
    src, dst = start[b] + path[b, k], start[b] + k
    for cache in (s["k"], s["v"]):
        layers, pages, kv, _, dim = cache.shape
        blocks, width = (dim // 64, 64) if _swizzled(cache.dtype, dim) else (1, dim)
        x = cache.view(layers, pages, kv, blocks, PAGE, width)
        rows = x[:, table[b, src // PAGE], :, :, src % PAGE]
        if _swizzled(cache.dtype, dim):
            turn = (src ^ dst) & 7                              # where a row's 16-byte chunks lie depends on the row
            chunk = torch.arange(8, device="cuda")[None] ^ turn[:, None]
            rows = rows.view(*rows.shape[:-1], 8, 8)
            at = chunk.view(-1, 1, 1, 1, 8, 1).expand(rows.shape)
            rows = torch.gather(rows, -2, at).reshape(*rows.shape[:-2], 64)
        x[:, table[b, dst // PAGE], :, :, dst % PAGE] = rows
    return dict(k=s["k"], v=s["v"])


# ---------------------------------------------------------------- the calls

def run(s):
    c = s["case"]
    op = c["op"]
    if not own:
        return {"tables": _plain_tables, "attend": _plain_attend, "accept": _plain_accept, "compact": _plain_compact}[op](s)
    from lumenllm_b200.ops import kernels as K
    if op == "tables":
        t = K.step_tables(s["seq_start"], s["seq_qlen"], s["slot_pages"], s["seq_slot"], s["n_tokens"], c["width"],
                          parents=s["parents"], mask_words=s["words"])
        out = dict(cu_q=t.cu_q, tok_seq=t.tok_seq, cache_pos=t.cache_pos, slot_map=t.slot_map, block_table=t.block_table,
                   tok_pos=t.tok_pos)
        return dict(out, tree_mask=t.tree_mask) if s["parents"] is not None else out
    if op == "attend":
        layout = K.LAYOUT_SW128 if _swizzled(s["q"].dtype, c["dim"]) else K.LAYOUT_LINEAR
        return K.attn_tree(s["q"], s["k"], s["v"], s["block_table"], s["cu_q"], s["seq_start"], s["tok_seq"], s["tok_pos"],
                           s["mask"], c["window"], s["scale"], layout=layout, softcap=c["softcap"],
                           sink=s["sink"] if c["sink"] else False)
    if op == "accept":
        count, path, emitted = K.tree_accept(s["picked"], s["tokens"], s["parents"], s["cu_q"], c["nodes"])
        return dict(count=count, path=path, emitted=emitted)
    layout = K.LAYOUT_SW128 if _swizzled(s["k"].dtype, c["dim"]) else K.LAYOUT_LINEAR
    K.cache_compact(s["k"], s["v"], s["block_table"], s["seq_start"], s["path"], s["count"], layout=layout)
    return dict(k=s["k"], v=s["v"])


def work(case):
    op, B = case["op"], case["batch"]
    mid = (case["low"] + case["high"]) / 2 if "low" in case else 0
    if op == "tables":
        nodes = sum(_spread(random.Random(0), 1, case["nodes"], B))
        held = B * (mid + case["nodes"] / 2) / PAGE
        words = -(-case["nodes"] // 64) if case["tree"] else 0
        # the lengths, slots and pages once; the step's arrays, the whole table with its last row
        return {"bytes": int(12 * B + 4 * held + 4 * nodes * bool(words) + 4 * (B + 1) * (case["width"] + 1) + nodes * (20 + 8 * words)),
                "flops": 0}
    nodes = sum(_spread(random.Random(0), (case["nodes"] + 1) // 2, case["nodes"] + 1, B)) if op != "compact" else 0
    if op == "accept":
        return {"bytes": int(12 * nodes + 4 * B * (2 + 2 * case["nodes"])), "flops": 0}
    e = 2 if case["dtype"] == "bfloat16" else 4
    if op == "compact":
        moved = sum(max(0, c - 1) for c in _spread(random.Random(0), 0, case["most"] + 1, B))
        return {"bytes": int(4 * moved * case["layers"] * case["kv"] * case["dim"] * e), "flops": 0}
    seen = min(mid, case["window"]) if case["window"] else mid
    return {"bytes": int(2 * nodes * case["heads"] * case["dim"] * e + 2 * (B * seen + nodes) * case["kv"] * case["dim"] * e),
            "flops": int(4 * nodes * case["heads"] * case["dim"] * (seen + 4))}


# ---------------------------------------------------------------- 64 bits

def _exact_key(cache, page, row):
    """The numbers of one token's row for every kv head, float64 [kv, dim], page and row as tensors [L]."""
    kv, dim = cache.shape[1], cache.shape[3]
    flat = cache.reshape(cache.shape[0], kv, PAGE * dim)
    e = torch.arange(dim, device="cuda")
    r = row[:, None]
    if _swizzled(cache.dtype, dim):
        at = (e // 64) * (64 * PAGE) + r * 64 + (((e % 64) // 8) ^ (r % 8)) * 8 + e % 8
    else:
        at = r * dim + e
    return flat[page[:, None, None], torch.arange(kv, device="cuda")[None, :, None], at[:, None, :]].double()


def exact(case, seed):
    if case["op"] in ("tables", "accept"):       # whole numbers
        return None
    s = prepare(case, seed)
    if case["op"] == "compact":
        out = {}
        for name in ("k", "v"):
            cache, swizzled = s[name], _swizzled(s[name].dtype, case["dim"])
            e = torch.arange(case["dim"], device="cuda")

            def at(r):
                return (e // 64) * (64 * PAGE) + r * 64 + (((e % 64) // 8) ^ (r % 8)) * 8 + e % 8 if swizzled else r * case["dim"] + e

            flat = cache.double().flatten(3)
            for b, (begin, count) in enumerate(zip(s["seq_start"].tolist(), s["count"].tolist())):
                page, path = s["block_table"][b].tolist(), s["path"][b].tolist()
                for k in range(1, count):
                    i, j = begin + path[k], begin + k
                    flat[:, page[j // PAGE], :, at(j % PAGE)] = flat[:, page[i // PAGE], :, at(i % PAGE)]
            out[name] = flat.view(cache.shape)
        return out
    kv, dim, group = case["kv"], case["dim"], case["heads"] // case["kv"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    cu, start = s["cu_q"].tolist(), s["seq_start"].tolist()
    for b in range(case["batch"]):
        n0, n1, begin = cu[b], cu[b + 1], start[b]
        count = n1 - n0
        j = torch.arange(begin + count, device="cuda")
        page = s["block_table"][b].long()[j // PAGE]
        K, V = _exact_key(s["k"], page, j % PAGE), _exact_key(s["v"], page, j % PAGE)
        pos = s["tok_pos"][n0:n1].long()
        key_pos = torch.cat([j[:begin], pos])
        seen = torch.ones((count, begin + count), dtype=torch.bool, device="cuda")
        for m in range(count):
            seen[:, begin + m] = (s["mask"][n0:n1, m // 64] >> (m % 64)) & 1 == 1
        if case["window"]:
            seen &= pos[:, None] - key_pos[None] < case["window"]
        for h in range(case["heads"]):
            x = s["q"][n0:n1, h].double() @ K[:, h // group].T * s["scale"]
            if case["softcap"]:
                x = case["softcap"] * torch.tanh(x / case["softcap"])
            x = x.masked_fill(~seen, -math.inf)
            if s["sink"] is not None:
                x = torch.cat([x, s["sink"][h].double().expand(count, 1)], 1)
            a = torch.softmax(x, 1)[:, :begin + count]
            out[n0:n1, h] = a @ V[:, h // group]
    return out
