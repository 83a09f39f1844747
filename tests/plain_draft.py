"""Plain 64-bit forms of the operators that check trees of drafted tokens, and cases for them. Nothing of the library is
used here; shapes and meanings are those of ops.kernels.step_tables, attn_tree, tree_accept and cache_compact."""
import math
import random

import torch

I32, I64 = torch.int32, torch.int64
PAGE = 64


def random_tree(rng, q, roots=False):
    """Parents of q nodes in any order of depth; with `roots` more than one may hang on the cached tokens."""
    return [-1] + [rng.randint(-1 if roots else 0, i - 1) for i in range(1, q)]


def ancestors(parents):
    """Per node the set of its ancestors with itself; a parent that is no earlier node counts as none."""
    out = []
    for i, p in enumerate(parents):
        out.append({i} | (out[p] if 0 <= p < i else set()))
    return out


def mask_words(sets, words):
    rows = []
    for s in sets:
        v = [0] * words
        for m in s:
            if m < 64 * words:
                v[m // 64] |= 1 << (m % 64)
        rows.append([x - (1 << 64) if x >> 63 else x for x in v])
    return torch.tensor(rows, dtype=I64).view(-1, words)


def tables(starts, qlens, slot_pages, slots, N, width, parents=None, words=1):
    """step_tables with Python's whole numbers."""
    B, room = len(starts), width * PAGE
    cu, seq, cpos, tpos, smap, rows, masks = [0], [], [], [], [], [], []
    used = 0
    for b in range(B):
        s = min(max(starts[b], 0), room)
        q = min(max(qlens[b], 0), room - s, 64 * words if parents is not None else room)
        pages = slot_pages[slots[b]] if 0 <= slots[b] < len(slot_pages) else [0] * width
        held = -(-(s + q) // PAGE)
        rows.append([pages[w] if w < held else 0 for w in range(width)])
        q = min(q, N - used)
        sets = ancestors(parents[used:used + q]) if parents is not None else None
        for i in range(q):
            p = s + i
            seq.append(b)
            cpos.append(p)
            tpos.append(s + len(sets[i]) - 1 if sets else p)
            smap.append(pages[p // PAGE] * PAGE + p % PAGE)
            masks.append(sets[i] if sets else set())
        used += q
        cu.append(used)
    rows.append([0] * width)
    rest = N - used
    seq += [B] * rest
    cpos += [0] * rest
    tpos += [0] * rest
    smap += [-1] * rest
    masks += [set()] * rest
    t = lambda x, d=I32: torch.tensor(x, dtype=d)
    return (t(cu), t(seq), t(cpos), t(tpos), t(smap, I64), t(rows).view(B + 1, width),
            mask_words(masks, words) if parents is not None else None)


def accept(picked, tokens, parents, cu, most):
    """tree_accept, one node after the other."""
    counts, paths, said = [], [], []
    for n0, n1 in zip(cu[:-1], cu[1:]):
        path, cur = [], 0 if n1 > n0 else None
        while cur is not None and len(path) < most:
            path.append(cur)
            cur = next((i for i in range(cur + 1, min(n1 - n0, 256)) if parents[n0 + i] == cur and tokens[n0 + i] == picked[n0 + cur]), None)
        counts.append(len(path))
        paths.append(path + [-1] * (most - len(path)))
        said.append([picked[n0 + i] for i in path] + [-1] * (most - len(path)))
    return counts, paths, said


def attention(q, k, v, start, seen, pos, window, scale, softcap=0.0, sink=None):
    """One sequence: q [q, nq, d], k, v [start + q, nkv, .], seen: per node the set of nodes it sees, pos: the nodes'
    positions. Returns (out, weighted |v|) in float64; rows that see nothing are 0."""
    n, nq, _ = q.shape
    nkv = k.shape[1]
    out = torch.zeros(n, nq, v.shape[2], dtype=torch.float64)
    size = torch.zeros_like(out)
    for i in range(n):
        p = max(pos[i], start)
        js = [j for j in range(start) if not window or p - j < window]
        js += [start + m for m in sorted(seen[i]) if m < n and (not window or p - max(pos[m], start) < window)]
        if not js:
            continue
        for h in range(nq):
            x = (k[js, h // (nq // nkv)].double() @ q[i, h].double()) * scale
            if softcap:
                x = softcap * torch.tanh(x / softcap)
            if sink is not None:
                x = torch.cat([x, sink[h].double().view(1)])
            a = torch.softmax(x, 0)[:len(js)]
            vals = v[js, h // (nq // nkv)].double()
            out[i, h] = a @ vals
            size[i, h] = a @ vals.abs()
    return out, size


def swizzled(x):
    """[..., 64, d] rows in order -> the swizzled tile, as [..., 64, d] in storage order."""
    d = x.shape[-1]
    r, e = torch.meshgrid(torch.arange(PAGE), torch.arange(d), indexing="ij")
    at = (e // 64) * (PAGE * 64) + r * 64 + (((e % 64) // 8) ^ (r % 8)) * 8 + e % 8
    out = torch.empty_like(x).flatten(-2)
    out[..., at.flatten()] = x.flatten(-2)
    return out.view(x.shape)


class Case:
    """Sequences with cached tokens and nodes, their keys and values in a paged cache whose every other number is NaN."""

    def __init__(self, starts, qlens, nq, nkv, d, dv=None, dtype=torch.bfloat16, seed=0, words=None, sets=None, extra_width=0,
                 q_scale=1.0):
        rng, g = random.Random(seed), torch.Generator().manual_seed(seed)
        self.starts, self.qlens, self.nq, self.nkv, self.d, self.dv, self.dtype = starts, qlens, nq, nkv, d, dv or d, dtype
        self.parents = [random_tree(rng, n, roots=True) if n else [] for n in qlens]
        self.sets = sets if sets is not None else [ancestors(p) for p in self.parents]
        depth = [[len(s) - 1 for s in ancestors(p)] for p in self.parents]
        self.pos = [[s + x for x in row] for s, row in zip(starts, depth)]
        self.words = words or max(1, max(-(-n // 64) for n in qlens))
        self.width = max(1, max(-(-(s + n) // PAGE) for s, n in zip(starts, qlens))) + extra_width
        held = [-(-(s + n) // PAGE) for s, n in zip(starts, qlens)]
        self.n_pages = sum(held) + 3
        ids = rng.sample(range(1, self.n_pages), sum(held))
        self.table = torch.zeros(len(starts), self.width, dtype=I32)
        self.q = (torch.randn(sum(qlens), nq, d, generator=g) * q_scale).to(dtype)
        self.k, self.v = [], []
        self.kc = torch.full((self.n_pages, nkv, PAGE, d), math.nan, dtype=dtype)
        self.vc = torch.full((self.n_pages, nkv, PAGE, self.dv), math.nan, dtype=dtype)
        for b, (s, n) in enumerate(zip(starts, qlens)):
            self.k.append(torch.randn(s + n, nkv, d, generator=g).to(dtype))
            self.v.append((torch.randn(s + n, nkv, self.dv, generator=g) + 0.25).to(dtype))
            for w in range(held[b]):
                self.table[b, w] = ids.pop()
        self.fill()

    def fill(self):
        """Puts self.k and self.v into the pages."""
        for b, (s, n) in enumerate(zip(self.starts, self.qlens)):
            for w in range(-(-(s + n) // PAGE)):
                m = min(PAGE, s + n - PAGE * w)
                pg = int(self.table[b, w])
                self.kc[pg, :, :m] = self.k[b][PAGE * w:PAGE * w + m].transpose(0, 1)
                self.vc[pg, :, :m] = self.v[b][PAGE * w:PAGE * w + m].transpose(0, 1)

    def arrays(self):
        cu, seq, pos = [0], [], []
        for b, n in enumerate(self.qlens):
            cu.append(cu[-1] + n)
            seq += [b] * n
            pos += self.pos[b]
        t = lambda x: torch.tensor(x, dtype=I32)
        return dict(block_table=self.table, cu_q=t(cu), seq_start=t(self.starts), tok_seq=t(seq), tok_pos=t(pos),
                    tree_mask=mask_words([s for row in self.sets for s in row], self.words))

    def reference(self, window=0, softcap=0.0, sink=None, scale=None):
        outs, sizes, n0 = [], [], 0
        for b, n in enumerate(self.qlens):
            o, z = attention(self.q[n0:n0 + n], self.k[b], self.v[b], self.starts[b], self.sets[b], self.pos[b], window,
                             self.d ** -0.5 if scale is None else scale, softcap, sink)
            outs.append(o)
            sizes.append(z)
            n0 += n
        return torch.cat(outs), torch.cat(sizes)

    def bound(self, out, size, softcap=0.0, scale=None, rounded_weights=False):
        """How far a result may be off, number by number. A score is a float32 sum of d products: off by (d + 2) 2^-23 of the sum
        of their sizes at most (2^-23: sums that drop bits), its cap by softcap 2^-20; a weight by twice that beside the
        normalising sum's own error, and by 2^-21 for its exponential; n weights and products are added in float32. Results are
        rounded to the type, half a step; the tensor cores take weights of half a step of bfloat16 too."""
        scale = self.d ** -0.5 if scale is None else abs(scale)          # a score is off by its size, whatever its sign
        n = max(s + q for s, q in zip(self.starts, self.qlens))
        qk = float(self.q.float().abs().max()) * max(float(k.float().abs().max()) for k in self.k if k.numel()) * self.d
        qk = min(qk, float(self.q.double().norm(dim=-1).max()) * max(float(k.double().norm(dim=-1).max()) for k in self.k if k.numel()))
        score = (self.d + 2) * 2.0 ** -23 * qk * scale + softcap * 2.0 ** -20
        rel = 2 * score + 2.0 ** -20 + n * 2.0 ** -23
        tol = rel * size + 1e-30
        if self.dtype == torch.bfloat16:
            tol = tol + 2.0 ** -8 * out.abs()
        else:
            tol = tol + 2.0 ** -24 * out.abs()
        return tol + (2.0 ** -8 * size if rounded_weights else 0.0)
