// What a step of drafted tokens needs beside its attention: the step's tables from the requests' lengths, the walk that
// accepts drafts, and the move of the accepted tokens' rows in the cache. Whole numbers and copies; what these kernels take
// is a launch and a few dependent reads, and for large tables and moves the bytes.
#include "tree_plan.cuh"

#define DT_THREADS 256
#define DT_TABLE 1024             // page table entries a block writes

// The nodes that sequence b brings: what its lengths say, held inside the page table's room and the masks' words.
__device__ __forceinline__ int dt_nodes(const int* seq_start, const int* seq_qlen, int b, int room, int most) {
    const int start = min(max(seq_start[b], 0), room);
    return min(min(max(seq_qlen[b], 0), room - start), most);
}

// Block (b, y): entries [1024 y, 1024 y + 1024) of row b of the page table, and (y = 0) sequence b's tokens; b = B stands for
// the table's last row, all zeros, and the tokens behind the last sequence. Every block adds up the lengths before its own
// sequence itself: no second launch and no wait between blocks. With a tree a thread has a node, and sets of
// ancestors double: after round r a node knows its 2^r nearest.
template <bool TREE>
__global__ void __launch_bounds__(DT_THREADS)
step_tables_kernel(const int* __restrict__ seq_start, const int* __restrict__ seq_qlen, const int* __restrict__ slot_pages,
                   long long slot_stride, int n_slots, const int* __restrict__ seq_slot, const int* __restrict__ parents, int B,
                   int N, int width, int words, int* __restrict__ cu_q, int* __restrict__ tok_seq, int* __restrict__ cache_pos,
                   int* __restrict__ tok_pos, long long* __restrict__ slot_map, int* __restrict__ block_table,
                   unsigned long long* __restrict__ tree_mask) {
    pdl_wait();
    pdl_trigger();
    __shared__ unsigned long long s_anc[TREE ? 4 * TREE_MAX_NODES : 1];
    __shared__ int s_up[TREE ? TREE_MAX_NODES : 1];
    __shared__ long long s_sum[DT_THREADS / 32];
    const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 31;
    const int room = width * LUMEN_PAGE, most = TREE ? 64 * words : room;
    int start = 0, q = 0, slot = -1;
    if (b < B) {
        start = min(max(seq_start[b], 0), room);
        q = dt_nodes(seq_start, seq_qlen, b, room, most);
        slot = seq_slot[b];
    }
    const int* row = (slot >= 0 && slot < n_slots) ? slot_pages + slot * slot_stride : nullptr;
    const int held = (start + q + LUMEN_PAGE - 1) / LUMEN_PAGE;
    for (int w = blockIdx.y * DT_TABLE + tid, end = min(width, (int)(blockIdx.y + 1) * DT_TABLE); w < end; w += DT_THREADS)
        block_table[(size_t)b * width + w] = (row && w < held) ? row[w] : 0;
    if (blockIdx.y) return;

    long long before = 0;
    for (int i = tid; i < b; i += DT_THREADS) before += dt_nodes(seq_start, seq_qlen, i, room, most);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) before += __shfl_xor_sync(0xffffffffu, before, o);
    if (lane == 0) s_sum[tid >> 5] = before;
    __syncthreads();
    before = 0;
#pragma unroll
    for (int i = 0; i < DT_THREADS / 32; ++i) before += s_sum[i];
    const int n0 = (int)min(before, (long long)N);
    if (tid == 0) cu_q[b] = n0;
    if (b == B) {
        for (int n = n0 + tid; n < N; n += DT_THREADS) {
            tok_seq[n] = B;
            cache_pos[n] = tok_pos[n] = 0;
            slot_map[n] = -1;
            if (TREE)
                for (int w = 0; w < words; ++w) tree_mask[(size_t)n * words + w] = 0;
        }
        return;
    }
    q = min(q, N - n0);
    if (TREE) {
        const int i = tid;
        unsigned long long anc[4] = {0, 0, 0, 0};
        int up = -1;
        if (i < q) {
            up = parents[n0 + i];
            if (up >= i || up < 0) up = -1;
#pragma unroll
            for (int w = 0; w < 4; ++w) anc[w] = (i >> 6) == w ? 1ull << (i & 63) : 0;
        }
        for (int span = 1; span < q; span <<= 1) {
            s_up[i] = up;
#pragma unroll
            for (int w = 0; w < 4; ++w)
                if (w < words) s_anc[w * TREE_MAX_NODES + i] = anc[w];
            if (__syncthreads_or(up >= 0) == 0) break;
            if (up >= 0) {
#pragma unroll
                for (int w = 0; w < 4; ++w)
                    if (w < words) anc[w] |= s_anc[w * TREE_MAX_NODES + up];
                up = s_up[up];
            }
            __syncthreads();
        }
        if (i < q) {
            int depth = -1;
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                depth += __popcll(anc[w]);
                if (w < words) tree_mask[(size_t)(n0 + i) * words + w] = anc[w];
            }
            tok_pos[n0 + i] = start + depth;
        }
    }
    for (int i = tid; i < q; i += DT_THREADS) {
        const int p = start + i;
        tok_seq[n0 + i] = b;
        cache_pos[n0 + i] = p;
        if (!TREE) tok_pos[n0 + i] = p;
        slot_map[n0 + i] = (long long)(row ? row[p / LUMEN_PAGE] : 0) * LUMEN_PAGE + p % LUMEN_PAGE;
    }
}

LUMEN_API int lumen_step_tables(const int* seq_start, const int* seq_qlen, const int* slot_pages, long long slot_stride, int n_slots,
                                const int* seq_slot, const int* parents, int B, int N, int width, int words, int* cu_q, int* tok_seq,
                                int* cache_pos, int* tok_pos, long long* slot_map, int* block_table, void* tree_mask,
                                cudaStream_t stream) {
    if (B < 0 || N < 0 || width < 1 || width > (1 << 24) || n_slots < 0 || (parents && (words < 1 || words > TREE_MAX_NODES / 64)))
        return LUMEN_ERR_BAD_ARGUMENT;
    const dim3 grid(B + 1, (width + DT_TABLE - 1) / DT_TABLE);
    cudaError_t e;
    if (parents)
        e = lumen_launch(step_tables_kernel<true>, grid, dim3(DT_THREADS), 0, stream, seq_start, seq_qlen, slot_pages, slot_stride, n_slots,
                         seq_slot, parents, B, N, width, words, cu_q, tok_seq, cache_pos, tok_pos, slot_map, block_table,
                         (unsigned long long*)tree_mask);
    else
        e = lumen_launch(step_tables_kernel<false>, grid, dim3(DT_THREADS), 0, stream, seq_start, seq_qlen, slot_pages, slot_stride, n_slots,
                         seq_slot, parents, B, N, width, words, cu_q, tok_seq, cache_pos, tok_pos, slot_map, block_table,
                         (unsigned long long*)tree_mask);
    if (e != cudaSuccess) return (int)e;
    LUMEN_LAUNCH_CHECK();
    return 0;
}

// The walk through a tree: from node 0, to the lowest child whose token is the one picked at the node, as long as there
// is one. A block has a sequence; every node that agrees with its parent's pick offers itself to the parent (the lowest
// index stays, whatever the order), then one thread walks: a read of shared memory a step.
__global__ void __launch_bounds__(128)
tree_accept_kernel(const int* __restrict__ picked, const int* __restrict__ tokens, const int* __restrict__ parents,
                   const int* __restrict__ cu_q, int N, int most, int* __restrict__ count, int* __restrict__ path,
                   int* __restrict__ emitted) {
    pdl_wait();
    pdl_trigger();
    __shared__ int s_child[TREE_MAX_NODES], s_path[TREE_MAX_NODES], s_pick[TREE_MAX_NODES], s_count;
    const int b = blockIdx.x, tid = threadIdx.x;
    const int n0 = min(max(cu_q[b], 0), N), q = min(max(0, min(cu_q[b + 1], N) - n0), TREE_MAX_NODES);
    for (int i = tid; i < q; i += 128) {
        s_child[i] = TREE_MAX_NODES;
        s_pick[i] = picked[n0 + i];
    }
    __syncthreads();
    for (int i = tid; i < q; i += 128) {
        const int up = parents[n0 + i];
        if (up >= 0 && up < i && tokens[n0 + i] == s_pick[up]) atomicMin(&s_child[up], i);
    }
    __syncthreads();
    if (tid == 0) {
        int cur = 0, n = 0;
        while (n < most && cur < q) {
            s_path[n++] = cur;
            cur = s_child[cur];
        }
        s_count = n;
        count[b] = n;
    }
    __syncthreads();
    for (int k = tid; k < most; k += 128) {
        const bool there = k < s_count;
        path[(size_t)b * most + k] = there ? s_path[k] : -1;
        emitted[(size_t)b * most + k] = there ? s_pick[s_path[k]] : -1;
    }
}

LUMEN_API int lumen_tree_accept(const int* picked, const int* tokens, const int* parents, const int* cu_q, int B, int N, int most,
                                int* count, int* path, int* emitted, cudaStream_t stream) {
    if (B <= 0) return 0;
    if (N < 0 || most < 1 || most > TREE_MAX_NODES) return LUMEN_ERR_BAD_ARGUMENT;
    const cudaError_t e = lumen_launch(tree_accept_kernel, dim3(B), dim3(128), 0, stream, picked, tokens, parents, cu_q, N, most, count,
                                       path, emitted);
    if (e != cudaSuccess) return (int)e;
    LUMEN_LAUNCH_CHECK();
    return 0;
}

// Moves rows inside the cache: the key and value at index start + path[k] of a sequence go to start + k, in every layer. A
// thread has the same U bytes of a row of one (layer, kv head) for all k and moves them in rising k, a batch of loads and
// then its stores: a path rises, so path[k] >= k, and no later move reads a row that an earlier one has written; other
// threads' bytes are never touched. It is bound by the latency of two dependent memory accesses for few rows and by the bytes
// for many.
struct CompactArgs {
    unsigned char* cache[2];
    int row_units[2], d[2], layout[2];       // U-byte pieces a row has, its numbers, its tile's layout
    const int* block_table;
    const int* seq_start;
    const int* path;
    const int* count;
    int bt_stride, width, most, layers, n_pages, nkv, es;
};
template <typename U>
__global__ void __launch_bounds__(128)
cache_compact_kernel(const CompactArgs a) {
    pdl_wait();
    pdl_trigger();
    __shared__ int s_from[TREE_MAX_NODES], s_to[TREE_MAX_NODES], s_n;       // rows: page * 64 + row in the page
    const int b = blockIdx.y, z = blockIdx.z, tid = threadIdx.x;
    const int n = min(min(max(a.count[b], 0), a.most), TREE_MAX_NODES);
    if (n < 2) return;
    const int room = a.width * LUMEN_PAGE, start = min(max(a.seq_start[b], 0), room);
    const int* path = a.path + (size_t)b * a.most;
    const int* bt = a.block_table + (size_t)b * a.bt_stride;
    if (tid == 0) s_n = n;
    __syncthreads();
    for (int k = 1 + tid; k < n; k += 128) {
        const int from = path[k], to = start + k;
        // the path ends where it does not rise, leaves the page table, or meets a page that there is not
        bool ok = from > path[k - 1] && from >= k && from < room - start;
        int pf = 0, pt = 0;
        if (ok) {
            pf = bt[(start + from) / LUMEN_PAGE];
            pt = bt[to / LUMEN_PAGE];
            ok = (unsigned)pf < (unsigned)a.n_pages && (unsigned)pt < (unsigned)a.n_pages;
        }
        if (!ok) atomicMin(&s_n, k);
        s_from[k] = pf * LUMEN_PAGE + (start + from) % LUMEN_PAGE;
        s_to[k] = pt * LUMEN_PAGE + to % LUMEN_PAGE;
    }
    __syncthreads();
    const int units = z ? a.row_units[1] : a.row_units[0], last = s_n;
    const long long idx = (long long)blockIdx.x * 128 + tid;
    if (idx >= (long long)a.layers * a.nkv * units) return;
    const int lh = (int)(idx / units), c = (int)(idx - (long long)lh * units), layer = lh / a.nkv, head = lh - layer * a.nkv;
    const int e = c * (int)(sizeof(U) / a.es), d = z ? a.d[1] : a.d[0], layout = z ? a.layout[1] : a.layout[0];
    unsigned char* base = (z ? a.cache[1] : a.cache[0]) + (size_t)layer * a.n_pages * a.nkv * LUMEN_PAGE * d * a.es;
    auto at = [&](int row) {
        const size_t tile = (size_t)(row / LUMEN_PAGE) * a.nkv + head;
        return reinterpret_cast<U*>(base + (tile * (size_t)(LUMEN_PAGE * d) + tile_offset(layout, row % LUMEN_PAGE, e, d)) * a.es);
    };
    constexpr int BATCH = 8;
    for (int k0 = 1; k0 < last; k0 += BATCH) {
        U v[BATCH];
#pragma unroll
        for (int i = 0; i < BATCH; ++i)
            if (k0 + i < last) v[i] = *at(s_from[k0 + i]);
#pragma unroll
        for (int i = 0; i < BATCH; ++i)
            if (k0 + i < last && s_from[k0 + i] != s_to[k0 + i]) *at(s_to[k0 + i]) = v[i];
    }
}

// keys [layers, n_pages, nkv, 64, d], values [layers, n_pages, nkv, 64, dv] (null: keys alone), es bytes a number.
LUMEN_API int lumen_cache_compact(void* kcache, void* vcache, const int* block_table, int bt_stride, int width, const int* seq_start,
                                  const int* path, int most, const int* count, int B, int layers, int n_pages, int nkv, int d, int dv,
                                  int layout, int v_layout, int es, cudaStream_t stream) {
    if (B <= 0 || layers <= 0) return 0;
    if (width < 1 || width > (1 << 24) || most < 1 || most > TREE_MAX_NODES || n_pages < 1 || n_pages > (1 << 24) || nkv < 1 || d < 1 ||
        (vcache && dv < 1) || (es != 2 && es != 4) || B > 65535)
        return LUMEN_ERR_BAD_ARGUMENT;
    if ((layout == LUMEN_LAYOUT_SW128 && (es != 2 || d % 64)) || (vcache && v_layout == LUMEN_LAYOUT_SW128 && (es != 2 || dv % 64)))
        return LUMEN_ERR_UNSUPPORTED;
    // the widest piece that divides the rows of both and their places
    const unsigned long long all = (unsigned long long)d * es | (unsigned long long)(uintptr_t)kcache |
                                   (vcache ? (unsigned long long)dv * es | (unsigned long long)(uintptr_t)vcache : 0ull);
    const int unit = all % 16 == 0 ? 16 : all % 4 == 0 ? 4 : 2;
    CompactArgs a = {{(unsigned char*)kcache, (unsigned char*)vcache}, {d * es / unit, dv * es / unit}, {d, dv}, {layout, v_layout},
                     block_table, seq_start, path, count, bt_stride, width, most, layers, n_pages, nkv, es};
    const int most_units = vcache && dv > d ? a.row_units[1] : a.row_units[0];
    const long long blocks = ((long long)layers * nkv * most_units + 127) / 128;
    if (blocks > 2147483647LL) return LUMEN_ERR_UNSUPPORTED;
    const dim3 grid((unsigned)blocks, B, vcache ? 2 : 1);
    cudaError_t e;
    if (unit == 16) e = lumen_launch(cache_compact_kernel<uint4>, grid, dim3(128), 0, stream, a);
    else if (unit == 4) e = lumen_launch(cache_compact_kernel<unsigned>, grid, dim3(128), 0, stream, a);
    else e = lumen_launch(cache_compact_kernel<unsigned short>, grid, dim3(128), 0, stream, a);
    if (e != cudaSuccess) return (int)e;
    LUMEN_LAUNCH_CHECK();
    return 0;
}
