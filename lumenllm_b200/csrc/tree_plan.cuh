// What the kernels of a tree of drafted tokens share: a sequence's lengths, made safe against whatever lies in the device's
// arrays, and the cut of its keys into segments.
//
// Sequence b has start cached tokens and brings q nodes, node i at index start + i of its cache. A row of the
// attention is a (node, query head) pair of one kv head: row f of a sequence is node f / G, head f % G of the group.
#pragma once
#include "common.cuh"

#define TREE_MAX_NODES 256        // nodes of a sequence that the masks and the walk cover
#define TREE_MAX_SEGS 64          // a sequence is never cut into more segments than this
#define TREE_MIN_SEG 2            // pages of the shortest segment
#define TREE_SEG_ROWS 32          // rows that have a page of a segment to themselves, at most
#define TREE_MMA_MIN_SEG 4        // both for the mma.sync kernel
#define TREE_MMA_SEG_ROWS 16

struct TreeSeq {
    int n0, q;        // its first token of the step, its nodes
    int start, end;   // its cached tokens, and the keys there are with the nodes'
};
// Lengths as the arrays say, held inside [0, N] tokens and the page table's room.
__device__ __forceinline__ TreeSeq tree_seq(const int* cu_q, const int* seq_start, int b, int N, int width) {
    TreeSeq s;
    s.n0 = min(max(cu_q[b], 0), N);
    s.q = max(0, min(cu_q[b + 1], N) - s.n0);
    const int room = width * LUMEN_PAGE;
    s.start = min(max(seq_start[b], 0), room);
    s.end = s.q > room - s.start ? room : s.start + s.q;
    return s;
}

// Pages [pg_lo, pg_lo + np) are those that some node of the sequence may see.
__host__ __device__ __forceinline__ void tree_pages(const TreeSeq& s, int window, int& pg_lo, int& np) {
    // no node stands before the cached tokens' end
    const int lo = window > 0 ? min(max(0, s.start - window + 1), s.end - 1) : 0;
    pg_lo = lo / LUMEN_PAGE;
    np = max((s.end - 1) / LUMEN_PAGE - pg_lo + 1, 1);
}
// The cut of them that does not depend on the step: nseg segments of per or per + 1 pages (the first rem have one more), of
// seg_min pages at least and one for every seg_rows rows. A segment's partial result is rows x dv float32, its keys and values
// are pages x 64 x (d + dv) numbers: with a page for 32 rows float32 partials come to a quarter of what the segment reads, beside a time
// that its arithmetic takes; with one for 16 rows bfloat16 ones to as much. Never on the neighbours in the batch or the page table's
// width.
struct TreePlan {
    int pg_lo, np, nseg, per, rem;
    __host__ __device__ __forceinline__ int first(int seg) const { return pg_lo + seg * per + min(seg, rem); }
    __host__ __device__ __forceinline__ int count(int seg) const { return per + (seg < rem ? 1 : 0); }
};
__host__ __device__ __forceinline__ TreePlan tree_plan(const TreeSeq& s, int window, int G, int seg_min, int seg_rows) {
    TreePlan p;
    tree_pages(s, window, p.pg_lo, p.np);
    const long long rows = (long long)s.q * G;
    const int seg = (int)min((long long)p.np, max((long long)seg_min, (rows + seg_rows - 1) / seg_rows));
    p.nseg = min((p.np + seg - 1) / seg, TREE_MAX_SEGS);
    p.per = p.np / p.nseg;
    p.rem = p.np - p.per * p.nseg;
    return p;
}
// Partial results of sequence b lie from this (token, segment) pair on, node i's segments at i * nseg: q * nseg is at most
// q + TREE_SEG_ROWS width / G whatever the lengths are (seg_min TREE_MIN_SEG or more, seg_rows TREE_SEG_ROWS or less).
__host__ __device__ __forceinline__ long long tree_part_room(int width, int G) { return ((long long)TREE_SEG_ROWS * width + G - 1) / G; }
__host__ __device__ __forceinline__ long long tree_part_base(int b, int n0, int width, int G) {
    return (long long)b * tree_part_room(width, G) + n0;
}
// Segments that the pages of a table of `width` pages may be cut into, and (token, segment) pairs of all sequences.
__host__ __device__ __forceinline__ int tree_max_segs(int width) { return min((width + TREE_MIN_SEG - 1) / TREE_MIN_SEG, TREE_MAX_SEGS); }
__host__ __device__ __forceinline__ long long tree_pairs(int B, int N, int width, int G) {
    return ((long long)B * tree_part_room(width, G) + N + 1) / 2 * 2;
}

// Unit u of a step whose sequences have ceil(q G / rows) tiles of rows each, in the order of the sequences: the sequence
// (B: there is no such unit) and the tile in it. Called by a whole warp.
__device__ __forceinline__ void tree_find(const int* cu_q, int B, int N, int G, int tile_rows, int u, int& b, int& tile) {
    const int lane = threadIdx.x & 31;
    for (int b0 = 0; b0 < B; b0 += 32) {
        const int i = b0 + lane;
        int t = 0;
        if (i < B) {
            const int n0 = min(max(cu_q[i], 0), N), q = max(0, min(cu_q[i + 1], N) - n0);
            t = (int)(((long long)q * G + tile_rows - 1) / tile_rows);
        }
        int sum = t;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum += v;
        }
        const unsigned hit = __ballot_sync(0xffffffffu, u < sum);
        if (hit) {
            const int at = __ffs(hit) - 1;
            b = b0 + at;
            tile = u - (__shfl_sync(0xffffffffu, sum, at) - __shfl_sync(0xffffffffu, t, at));
            return;
        }
        u -= __shfl_sync(0xffffffffu, sum, 31);
    }
    b = B;
    tile = 0;
}

// Which of the 64 keys jb .. jb + 63 a node at position p sees, as bits: cached ones by the window, the sequence's nodes by
// the node's mask (W words) and the window; pos: the nodes' positions (only read with a window).
__device__ __forceinline__ unsigned long long tree_seen(int jb, const TreeSeq& s, const unsigned long long* mask, int W, int p,
                                                        int window, const int* pos) {
    unsigned long long bits = 0;
    const int cached = s.start - jb;                      // keys of this page before the nodes
    if (cached > 0) {
        bits = cached >= 64 ? ~0ull : (1ull << cached) - 1;
        const long long lo = window > 0 ? (long long)p - window + 1 - jb : 0;        // keys before it are out of the window
        if (lo >= 64) bits = 0;
        else if (lo > 0) bits &= ~0ull << lo;
    }
    if (cached < 64) {
        const int m0 = -cached;                           // node at bit 0 of the page (negative: that many bits up)
        unsigned long long own = 0;
        if (m0 >= 0) {
            const int w = m0 >> 6, t = m0 & 63;
            if (w < W) own = mask[w] >> t;
            if (t && w + 1 < W) own |= mask[w + 1] << (64 - t);
        } else {
            own = mask[0] << -m0;
        }
        const int left = s.end - jb;                      // no key beyond the sequence's end
        if (left < 64) own &= left > 0 ? (1ull << left) - 1 : 0;
        if (window > 0 && p - s.start >= window) {        // else no node is that far before it
            unsigned long long todo = own;
            while (todo) {
                const int t = __ffsll((long long)todo) - 1;
                todo &= todo - 1;
                if (p - max(pos[m0 + t], s.start) >= window) own &= ~(1ull << t);
            }
        }
        bits |= own;
    }
    return bits;
}
