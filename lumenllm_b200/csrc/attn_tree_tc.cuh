// Tree attention on the 5th-generation tensor cores: bfloat16, swizzled pages, keys and values of multiples of 64 up to 256.
//
// The work is blocks of 128 rows (node, query head) of one kv head, each with its pages. All of it, counted in pages, is dealt out
// evenly over as many blocks of threads as fit the device: a piece, one block's part of a row block, is a unit. Row blocks
// that one block has whole are finished there; of the others every piece leaves its unnormalised O, maximum and sum, which
// a second kernel joins in rising order of the pages. So where a sequence is cut depends on the whole step, and its last bits with
// it; the same step gives the same bits. (Cutting every sequence by its own length alone left the last of 1.3 rounds of equal
// units to a third of the blocks: 64 nodes for 8 sequences after 4,000 to 6,000 tokens took 82 us.)
//
// A unit is walked a page at a time as
// the prompts' kernel does: S = Q K^T into tensor memory (two buffers), the softmax by four warps with a row a thread, P as
// bfloat16 over the scores it came from, O += P V in tensor memory; K and V tiles by bulk copies through two rings of two
// stages. A block needs half of an SM, so that one's softmax runs under the other's products. Warp 0 finds the units, tells the
// others through shared memory and asks for the tiles, warp 1 fetches Q (while the last unit's rows are written) and issues the
// products, warps 2 to 5 are the softmax. Pages that hold
// nodes, or that a window cuts for some row, are masked: a row has one 64-bit word a page with the keys it sees.
//
// What bounds long steps. Of several row blocks a kv head (64 nodes for 8 sequences, 63 us): the chain of S, softmax and O a page,
// which the two blocks of an SM hide from one another in part; with all pages in L2 and the softmax left out it takes 54 us, with but one
// step of each product besides 40. Of one row block (16 nodes for 64 sequences, 78 us): HBM, 5.4 TB/s here; 73 without softmax and
// products, 67 with all pages in L2. S of two pages in one product with P in shared memory (tensor memory has no room for it then)
// took 73 and 81 us, that with two threads a row, half of the keys each, 86 and 98.
//
// Weights are rounded to bfloat16 because the product takes both operands in one type: half a step, 2^-8 of a weight, which
// the sum over the keys averages; the running sum takes them unrounded.
//
// A masked weight is 0, but 0 times a value that is no number would not be: in masked pages such values are replaced by
// zeros in the tile before the product reads it, and a row that does see one gets it added at the end.
//
// Every wait is bounded, also where warps wait for one another. When one runs out the block raises the error flag, lets the
// other roles run out, waits for its copies and products (warps 0 and 1 always do, before the roles meet), frees its tensor memory
// and returns.
#pragma once
#include "tmem_attn.cuh"

#define TT_THREADS 192
#define TT_STAGES 2
#define TT_RESCALE 8.0f
#define TT_BAR_WORDS 48           // 8-byte words of barriers, units and flags
// What a row block costs beside its pages, in pages: Q, the first page's latency and the rows' writing (64 nodes for 8 sequences, before the
// teams: 66 to 69 us; with 1 or 6 pages 70).
#define TT_COST 3
// A block's least share of the work, in pages: fewer make more pieces to join, more leave SMs idle in small steps (8 nodes after 1,300
// tokens: 13.1 us; with 2 pages 13.7, with 5 15.7).
#define TT_SHARE 3

// A place in the step's work: page `page` (counted from the first that the sequence's nodes see) of row block rb of sequence b.
// b = B: the end.
struct TreeCut {
    int b, rb, page;
};
// A row block that is cut, as each of its cuts leaves it for the second kernel: its sequence's first token, its first row, kv head and
// rows, the pieces it is in (0: this cut lies between row blocks), the number of this cut among its own and how many blocks apart they are.
struct TreeJoin {
    int n0, f0, kvh, nrows, pieces, order, step, unused;
};
struct TreeTc {
    TreeArgs a;
    float scale_log2;             // with CAP softcap * log2(e), what the tanh is multiplied by
    float cap_pre;                // with CAP scale / softcap
    TreeJoin* joins;              // [blocks] the row blocks that their work begins inside of
    int* err;
};
// A unit: rows f0 .. f0 + 127 of sequence b and kv head kvh over pages pg0 .. pg0 + npages - 1 (npages 0: there is no more). slot: where
// its partial result goes (0: it begins inside the row block, 1: it only ends inside), -1 for a whole row block.
struct TreeUnit {
    int npages, pg0, b, n0, q, start, end, f0, kvh, slot;
};
#define TT_UNIT_INTS 10

// A sequence's work: its row blocks (kv heads times tiles of 128 rows), the pages of each, and both together in pages.
struct TreeWork {
    int pg_lo, np, tiles, all;
};
__device__ __forceinline__ TreeWork tt_work(const TreeArgs& a, const TreeSeq& s, int G) {
    TreeWork w = {0, 0, 0, 0};
    if (s.q > 0) {
        tree_pages(s, a.window, w.pg_lo, w.np);
        w.tiles = (s.q * G + PT_ROWS - 1) / PT_ROWS;
        w.all = w.tiles * a.nkv * (w.np + TT_COST);
    }
    return w;
}
__device__ __forceinline__ TreeWork tt_work_of(const TreeArgs& a, int b, int G) {
    return b < a.B ? tt_work(a, tree_seq(a.cu_q, a.seq_start, b, a.N, a.width), G) : TreeWork{0, 0, 0, 0};
}

__device__ __forceinline__ bool mbar_test(uint64_t* bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n .reg .pred p;\n mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity)
        : "memory");
    return ok != 0;
}
// A whole warp's wait (one lane asks) and question.
__device__ __forceinline__ bool tt_warp_wait(uint64_t* bar, uint32_t parity) {
    int ok = 0;
    if ((threadIdx.x & 31) == 0) ok = mbar_wait(bar, parity);
    ok = __shfl_sync(0xffffffffu, ok, 0);
    __syncwarp();                     // the shuffle alone does not put the other lanes' reads behind what lane 0 has waited for
    return ok != 0;
}
__device__ __forceinline__ bool tt_warp_test(uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, mbar_test(bar, parity)); }
// One lane of a whole warp, the same one every time.
__device__ __forceinline__ bool tt_elect() {
    uint32_t p;
    asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}" : "=r"(p)::"memory");
    return p != 0;
}
__device__ __forceinline__ pt_f2 tt_mul2(pt_f2 a, pt_f2 b) {
    pt_f2 d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
// tanh of pre * a and pre * b, both at most 0.5 in size: x times a polynomial of degree 4 in x^2, the one that meets tanh(x) / x at the
// Chebyshev nodes of [0, 0.25] with its constant term set to 1 (off by 2.6e-8 of it at most, by 1.1e-7 in float32). Scores are rarely beyond half of their cap;
// this takes no special-function unit, whose three operations a score held the softmax before (a page of 64 keys took a block
// 3,400 cycles, with this 2,700; 21.8 against 25.2 us for 16 x 24 nodes under a window of 1,024, heads of 64).
__device__ __forceinline__ void tt_tanh_small(float& a, float& b, float pre) {
    const pt_f2 x = tt_mul2(pt_pair(a, b), pt_pair(pre, pre)), z = tt_mul2(x, x);
    pt_f2 h = pt_fma2(z, pt_pair(0.017131345346570015f, 0.017131345346570015f), pt_pair(-0.05298423767089844f, -0.05298423767089844f));
    h = pt_fma2(z, h, pt_pair(0.133247509598732f, 0.133247509598732f));
    h = pt_fma2(z, h, pt_pair(-0.3333306908607483f, -0.3333306908607483f));
    h = pt_fma2(z, h, pt_pair(1.0f, 1.0f));
    pt_unpair(tt_mul2(h, x), a, b);
}
__device__ __forceinline__ void tt_prefetch(const void* at) { asm volatile("prefetch.global.L1 [%0];" ::"l"(at)); }
// 32 bytes in one instruction; to has to lie on 32 bytes.
__device__ __forceinline__ void tt_store32(void* to, const uint32_t (&w)[8]) {
    asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(to), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]),
                 "r"(w[5]), "r"(w[6]), "r"(w[7])
                 : "memory");
}

// D: keys and values are D wide (64, 128), or (0) d and dv wide.
template <int D, bool CAP>
__global__ void __launch_bounds__(TT_THREADS, 2)
attn_tree_tc_kernel(const TreeTc t) {
    const TreeArgs& a = t.a;
    const int kw = D ? D : a.d, vw = D ? D : a.dv;
    const int K_BYTES = LUMEN_PAGE * kw * 2, V_BYTES = LUMEN_PAGE * vw * 2;
    const int STAGE_BYTES = K_BYTES + V_BYTES;
    const int NCOLS = vw <= 128 ? 256 : 512;            // S0 | S1 | O
    constexpr uint32_t O_COL = 128;
    extern __shared__ __align__(1024) unsigned char smem[];
    if (smem_u32(smem) & 1023u) {                       // operand tiles start on 1,024 bytes
        pdl_wait();
        if (threadIdx.x == 0) {
            t.joins[blockIdx.x] = TreeJoin{0, 0, 0, 0, 0, 0, 1, 0};      // the second kernel finds no pieces
            atomicExch(t.err, 1);
        }
        return;
    }
    unsigned char* sQ = smem;
    unsigned char* sKV = sQ + PT_ROWS * kw * 2;         // [stage][K tile, V tile]
    uint64_t* bars = reinterpret_cast<uint64_t*>(sKV + TT_STAGES * STAGE_BYTES);
    uint64_t* k_full = bars;                   // [stages] the K tile has landed
    uint64_t* k_empty = bars + TT_STAGES;      // [stages] the S product has read it
    uint64_t* v_full = bars + 2 * TT_STAGES;   // [stages] the V tile has landed
    uint64_t* v_empty = bars + 3 * TT_STAGES;  // [stages] the O product has read it
    uint64_t* s_full = bars + 4 * TT_STAGES;   // [2] S is in tensor memory
    uint64_t* p_ready = s_full + 2;            // [2] P is in tensor memory, O corrected, V without what is no number
    uint64_t* pv_done = p_ready + 2;           // [2] the PV product of that page has finished
    uint64_t* u_full = pv_done + 2;            // [2] a unit is told
    uint64_t* u_empty = u_full + 2;            // [2] it has been worked off
    uint64_t* together = u_empty + 2;          // the softmax warps wait for one another
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(together + 1);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    int* s_bad = reinterpret_cast<int*>(tmem_slot + 2);        // [2] unit number + 1 where a masked page holds a value that is no number
    volatile int* s_unit = s_bad + 2;          // [2][TT_UNIT_INTS]
    TreeCut* s_cut = reinterpret_cast<TreeCut*>(s_bad + 2 + 2 * TT_UNIT_INTS);      // [2] where this block's work begins and ends
    volatile int* s_sum = reinterpret_cast<volatile int*>(s_cut + 2);               // [warps]
    volatile int* s_tiles = s_sum + TT_THREADS / 32;                                // [warps][2] least and most row blocks of a kv head
    volatile int* s_first = s_tiles + 2 * (TT_THREADS / 32);                        // [7] the first unit's sequence

    const int G = a.nq / a.nkv, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int i = 0; i < TT_STAGES; ++i) {
            mbar_init(&k_full[i], 1); mbar_init(&k_empty[i], 1);
            mbar_init(&v_full[i], 1); mbar_init(&v_empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&s_full[i], 1); mbar_init(&p_ready[i], 4); mbar_init(&pv_done[i], 1);
            mbar_init(&u_full[i], 1); mbar_init(&u_empty[i], 5);
        }
        mbar_init(together, 4);
        *abort_flag = 0;
        s_bad[0] = s_bad[1] = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                     "r"(NCOLS)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    pt_fence_before();
    __syncthreads();
    pt_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    pdl_wait();      // nothing of this kernel touches global memory before this
    pdl_trigger();
    // Row blocks of a kv head read the same pages. Where every sequence has as many of them, 2 to 4 neighbouring blocks are a team that
    // walks the same pages at the same time, each for a row block of its own: the pages come from HBM once (64 nodes for 8 sequences:
    // 171 MB of HBM reads and 63 us, without teams 255 and 66 to 69).
    //
    // Every block adds up the step's work, a thread the work of `run` neighbouring sequences; the threads whose sequences hold the
    // ends of the block's share find the places there. A cut is not made within two pages of a row block's ends.
    const int run = (a.B + TT_THREADS - 1) / TT_THREADS;
    int team = 1, in_team = 0;
    {
        TreeWork w = tt_work_of(a, threadIdx.x * run, G);
        const TreeWork w0 = w;
        long long all = w.all;
        int least = w.tiles ? w.tiles : 1 << 30, most = w.tiles;
        for (int i = 1; i < run; ++i) {
            const TreeWork x = tt_work_of(a, threadIdx.x * run + i, G);
            all += x.all;
            if (x.tiles) least = min(least, x.tiles);
            most = max(most, x.tiles);
        }
        least = __reduce_min_sync(0xffffffffu, least);
        most = __reduce_max_sync(0xffffffffu, most);
        // what the host has room for fits 32 bits; lengths that come to more contradict the number of tokens, and nothing is done
        int mine = all < (1 << 30) ? (int)all : 1 << 30;
        unsigned sum = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const unsigned v = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum = min(sum + v, 1u << 30);
        }
        if (lane == 31) { s_sum[warp] = (int)sum; s_tiles[2 * warp] = least; s_tiles[2 * warp + 1] = most; }
        __syncthreads();
        unsigned total = 0;
#pragma unroll
        for (int i = 0; i < TT_THREADS / 32; ++i) total = min(total + (unsigned)s_sum[i], 1u << 30);
        if (total >= 1u << 30) total = 0;
        int before = (int)sum - mine;                   // the work ahead of this thread's
#pragma unroll
        for (int i = 0; i < TT_THREADS / 32; ++i)
            if (i < warp) before += s_sum[i];
#pragma unroll
        for (int i = 0; i < TT_THREADS / 32; ++i) {
            least = min(least, s_tiles[2 * i]);
            most = max(most, s_tiles[2 * i + 1]);
        }
        // (with few blocks those that make no whole team would be missed, and the pages stay in L2 anyway)
        if (least == most && most > 1 && gridDim.x >= 64) team = most % 4 == 0 ? 4 : most % 3 == 0 ? 3 : most % 2 == 0 ? 2 : 1;
        int teams = gridDim.x, number = blockIdx.x;      // of a team's line of work, which has every team-th row block
        if (team > 1) {
            teams /= team;
            number /= team;
            in_team = blockIdx.x - number * team;
            total /= team;
            before /= team;
            mine /= team;
        }
        auto line = [&](int x) { return team > 1 ? x / team : x; };
        const int share = max((int)((total + teams - 1) / teams), TT_SHARE);
#pragma unroll 1
        for (int end = 0; end < 2; ++end) {
            int x = number < teams ? (number + end) * share : (int)total;
            TreeCut cut = {a.B, 0, 0};
            if (x >= (int)total ? threadIdx.x != 0 : x < before || x >= before + mine) continue;
            if (x < (int)total) {
                x -= before;
                cut.b = threadIdx.x * run;
                w = w0;
                while (x >= line(w.all)) {
                    x -= line(w.all);
                    w = tt_work_of(a, ++cut.b, G);
                }
                cut.rb = x / (w.np + TT_COST);
                cut.page = max(0, x - cut.rb * (w.np + TT_COST) - TT_COST);
                if (cut.page < 2) cut.page = 0;
                else if (w.np - cut.page < 2) {
                    cut.page = 0;
                    if (++cut.rb == line(w.tiles) * a.nkv) {
                        cut.rb = 0;
                        do w = tt_work_of(a, ++cut.b, G);
                        while (cut.b < a.B && w.all == 0);
                    }
                }
            }
            s_cut[end] = cut;
            if (end == 1) continue;
            TreeJoin join = {0, 0, 0, 0, 0, 0, team, 0};
            if (cut.b < a.B) {
                // what warp 0 needs for the block's first keys, and the second kernel to put the row block together
                const TreeSeq s = tree_seq(a.cu_q, a.seq_start, cut.b, a.N, a.width);
                s_first[0] = s.n0; s_first[1] = s.q; s_first[2] = s.start; s_first[3] = s.end;
                s_first[4] = w.pg_lo; s_first[5] = w.np; s_first[6] = w.tiles;
                tt_prefetch(a.block_table + (size_t)cut.b * a.bt_stride + w.pg_lo + cut.page);
                if (cut.page > 0) {
                    join.n0 = s.n0;
                    const int tiles = line(w.tiles);
                    join.kvh = cut.rb / tiles;
                    join.f0 = ((cut.rb - join.kvh * tiles) * team + in_team) * PT_ROWS;
                    join.nrows = min(PT_ROWS, s.q * G - join.f0);
                    join.order = (cut.page - 2) / share;          // the cuts before it and behind it lie `share` pages apart
                    join.pieces = 2 + join.order + (w.np - 2 - cut.page) / share;
                }
            }
            t.joins[blockIdx.x] = join;
        }
    }
    __syncthreads();
    const __nv_bfloat16* kcache = (const __nv_bfloat16*)a.kcache;
    const __nv_bfloat16* vcache = (const __nv_bfloat16*)a.vcache;

    // Counters of every role: k units and c pages since the block began; page c is in stage c % 2 of its ring and in
    // score buffer c & 1.
    auto unit_at = [&](int slot) {
        volatile int* from = s_unit + slot * TT_UNIT_INTS;
        TreeUnit x;
        x.npages = from[0]; x.pg0 = from[1]; x.b = from[2]; x.n0 = from[3]; x.q = from[4]; x.start = from[5]; x.end = from[6];
        x.f0 = from[7]; x.kvh = from[8]; x.slot = from[9];
        return x;
    };

    if (warp == 0) {
        uint32_t ck = 0, cv = 0;                        // K and V tiles asked for
        bool ok = true;
        TreeCut at = s_cut[0];
        const TreeCut to = s_cut[1];
        int b0 = at.b, held = 1;                        // lane i holds sequence b0 + i, `held` of them; at first the one that is known
        TreeSeq sq_l = {s_first[0], s_first[1], s_first[2], s_first[3]};
        TreeWork w_l = {s_first[4], s_first[5], s_first[6], 0};
        for (int k = 0; ok; ++k) {
            // the next piece of the block's work
            TreeUnit x = {0, 0, 0, 0, 0, 0, 0, 0, 0, -1};
            while (at.b < a.B) {
                if (at.b >= b0 + held) {
                    b0 = at.b;
                    held = 32;
                    sq_l = b0 + lane < a.B ? tree_seq(a.cu_q, a.seq_start, b0 + lane, a.N, a.width) : TreeSeq{0, 0, 0, 0};
                    w_l = tt_work(a, sq_l, G);
                }
                const int src = at.b - b0, np = __shfl_sync(0xffffffffu, w_l.np, src), all_tiles = __shfl_sync(0xffffffffu, w_l.tiles, src);
                const int tiles = team > 1 ? all_tiles / team : all_tiles;
                if (at.rb >= tiles * a.nkv) { ++at.b; at.rb = at.page = 0; continue; }
                const bool ends = at.b == to.b && at.rb == to.rb;
                const int last = ends ? to.page : np;
                if (at.b > to.b || (at.b == to.b && at.rb > to.rb) || (ends && at.page >= last)) break;
                x.b = at.b;
                x.n0 = __shfl_sync(0xffffffffu, sq_l.n0, src);
                x.q = __shfl_sync(0xffffffffu, sq_l.q, src);
                x.start = __shfl_sync(0xffffffffu, sq_l.start, src);
                x.end = __shfl_sync(0xffffffffu, sq_l.end, src);
                x.pg0 = __shfl_sync(0xffffffffu, w_l.pg_lo, src) + at.page;
                x.npages = last - at.page;
                x.kvh = at.rb / tiles;
                x.f0 = ((at.rb - x.kvh * tiles) * team + in_team) * PT_ROWS;
                x.slot = at.page > 0 ? 0 : last < np ? 1 : -1;
                ++at.rb;
                at.page = 0;
                break;
            }
            // page numbers 32 at a time: the first are under way while the others are told of the unit
            const int* bt = a.block_table + (size_t)x.b * a.bt_stride + x.pg0;
            int ids = lane < x.npages ? bt[lane] : 0, before = 0;
            if ((unsigned)ids >= (unsigned)a.n_pages) ids = 0;
            const int slot = k & 1;
            if (!(ok = tt_warp_wait(&u_empty[slot], ((k >> 1) & 1) ^ 1))) break;
            if (lane == 0) {
                volatile int* told = s_unit + slot * TT_UNIT_INTS;
                told[0] = x.npages; told[1] = x.pg0; told[2] = x.b; told[3] = x.n0; told[4] = x.q; told[5] = x.start; told[6] = x.end;
                told[7] = x.f0; told[8] = x.kvh; told[9] = x.slot;
                pt_mbar_arrive(&u_full[slot]);
            }
            if (x.npages == 0) break;
            const uint32_t first = cv, end = cv + x.npages;
            uint32_t spin = 0;
            while (cv < end) {
                // whichever slot is free: K tiles run ahead of V tiles, their slots come free earlier
                if (ck < end && tt_warp_test(&k_empty[ck % TT_STAGES], ((ck / TT_STAGES) & 1) ^ 1)) {
                    const uint32_t i = ck - first, st = ck % TT_STAGES;
                    if (i > 0 && (i & 31) == 0) {
                        before = ids;
                        ids = (int)(i + lane) < x.npages ? bt[i + lane] : 0;
                        if ((unsigned)ids >= (unsigned)a.n_pages) ids = 0;
                    }
                    const size_t tile = (size_t)__shfl_sync(0xffffffffu, ids, i & 31) * a.nkv + x.kvh;
                    if (lane == 0) {
                        mbar_expect_tx(&k_full[st], K_BYTES);
                        bulk_load(sKV + st * STAGE_BYTES, kcache + tile * (size_t)(LUMEN_PAGE * kw), K_BYTES, &k_full[st]);
                    }
                    ++ck;
                    spin = 0;
                }
                if (cv < ck && tt_warp_test(&v_empty[cv % TT_STAGES], ((cv / TT_STAGES) & 1) ^ 1)) {
                    const uint32_t i = cv - first, st = cv % TT_STAGES;
                    const int from = (i >> 5) == ((ck - first - 1) >> 5) ? ids : before;
                    const size_t tile = (size_t)__shfl_sync(0xffffffffu, from, i & 31) * a.nkv + x.kvh;
                    if (lane == 0) {
                        mbar_expect_tx(&v_full[st], V_BYTES);
                        bulk_load(sKV + st * STAGE_BYTES + K_BYTES, vcache + tile * (size_t)(LUMEN_PAGE * vw), V_BYTES, &v_full[st]);
                    }
                    ++cv;
                    spin = 0;
                }
                if (++spin > LUMEN_SPIN_LIMIT || __any_sync(0xffffffffu, *abort_flag != 0)) { ok = false; break; }
            }
        }
        if (lane == 0) {
            if (!ok) {
                *abort_flag = 1;
                atomicExch(t.err, 1);
            }
            // the last copies have landed before the block ends, also where it is another role that gives up on them
            for (uint32_t i = ck > TT_STAGES ? ck - TT_STAGES : 0; i < ck; ++i) mbar_wait(&k_full[i % TT_STAGES], (i / TT_STAGES) & 1);
            for (uint32_t i = cv > TT_STAGES ? cv - TT_STAGES : 0; i < cv; ++i) mbar_wait(&v_full[i % TT_STAGES], (i / TT_STAGES) & 1);
        }
    } else if (warp == 1) {
        // The whole warp runs through this, so that what a product is told is the same in all lanes and known to be (with one
        // thread alone S takes 770 cycles to issue instead of 640, O 490 instead of 280); one elected lane issues.
        constexpr uint32_t idesc_qk = pt_idesc(LUMEN_PAGE, 0);
        const uint32_t idesc_pv = pt_idesc(vw, 1);
        const int k_steps = kw / 16;
        const uint32_t q_at = smem_u32(sQ), kv_at = smem_u32(sKV);
        bool ok = true;
        uint32_t cs = 0, cv = 0;                        // pages whose S, whose O product has been issued
        // Q of a unit into [kw/64][row][64], 16-byte chunk c of a row at c ^ (row & 7): a node's G rows lie together in memory. Rows that
        // the sequence has not keep what was there: they are nobody's.
        auto ask_q = [&](const TreeUnit& x) {
            const int nrows = min(PT_ROWS, x.q * G - x.f0), pieces = kw >> 3, tok0 = x.f0 / G, skip = x.f0 - tok0 * G;
            const int toks = (skip + nrows + G - 1) / G;
            const __nv_bfloat16* src = (const __nv_bfloat16*)a.q + ((size_t)(x.n0 + tok0) * a.nq + x.kvh * G) * kw;
            for (int i = lane; i < G * pieces; i += 32) {
                const int h = i / pieces, c = i - h * pieces;
                const uint32_t to = q_at + (c >> 3) * (PT_ROWS * 128);
                const __nv_bfloat16* from = src + 8 * i;
                int row = h - skip;
#pragma unroll 4
                for (int tok = 0; tok < toks; ++tok, row += G, from += (size_t)a.nq * kw)
                    if (row >= 0 && row < nrows)
                        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to + row * 128 + (((c & 7) ^ (row & 7)) << 4)), "l"(from)
                                     : "memory");
            }
        };
        bool asked = false;                             // whether the next unit's Q is under way
        for (int k = 0; ok; ++k) {
            const int slot = k & 1;
            if (!(ok = tt_warp_wait(&u_full[slot], (k >> 1) & 1))) break;
            const TreeUnit x = unit_at(slot);
            const uint32_t first = cv, end = cv + x.npages;
            if (x.npages == 0) break;
            if (!asked) {
                // the last unit's S products have read their Q
                if (cs > 0 && !(ok = tt_warp_wait(&s_full[(cs - 1) & 1], ((cs - 1) >> 1) & 1))) break;
                ask_q(x);
            }
            asked = false;
            asm volatile("cp.async.wait_all;" ::: "memory");
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");       // the tensor cores read it
            __syncwarp();
            uint32_t spin = 0;
            while (cv < end) {
                // S of the next page as soon as its keys are there (its buffer's last weights went into a product that was
                // issued before), else O of this page: neither waits for what the other lacks
                if (cs < end && cs < cv + 2 && tt_warp_test(&k_full[cs % TT_STAGES], (cs / TT_STAGES) & 1)) {
                    pt_fence_after();
                    const uint32_t st = cs % TT_STAGES, kt = kv_at + st * STAGE_BYTES, to = tmem_base + (cs & 1) * LUMEN_PAGE;
                    if (tt_elect()) {
#pragma unroll(D ? D / 16 : 1)
                        for (int ks = 0; ks < k_steps; ++ks) {
                            const uint32_t aoff = (ks >> 2) * (PT_ROWS * 128) + (ks & 3) * 32;
                            const uint32_t boff = (ks >> 2) * (LUMEN_PAGE * 128) + (ks & 3) * 32;
                            pt_mma(to, pt_desc(q_at + aoff, 16), pt_desc(kt + boff, 16), idesc_qk, ks > 0 ? 1u : 0u);
                        }
                        pt_commit(&s_full[cs & 1]);
                        pt_commit(&k_empty[st]);
                    }
                    __syncwarp();
                    ++cs;
                    spin = 0;
                } else if (cv < cs && tt_warp_test(&p_ready[cv & 1], (cv >> 1) & 1) && tt_warp_test(&v_full[cv % TT_STAGES], (cv / TT_STAGES) & 1)) {
                    pt_fence_after();
                    const uint32_t st = cv % TT_STAGES, vt = kv_at + st * STAGE_BYTES + K_BYTES;
                    const uint32_t pt = tmem_base + (cv & 1) * LUMEN_PAGE;       // P lies over the first 32 columns of its scores
                    if (tt_elect()) {
#pragma unroll
                        for (int kk = 0; kk < LUMEN_PAGE / 16; ++kk)
                            pt_mma_ts(tmem_base + O_COL, pt + kk * 8,
                                      pt_desc(vt + kk * (16 * 128), LUMEN_PAGE * 128), idesc_pv, (cv > first || kk > 0) ? 1u : 0u);
                        pt_commit(&v_empty[st]);
                        pt_commit(&pv_done[cv & 1]);
                    }
                    __syncwarp();
                    ++cv;
                    spin = 0;
                } else if (!asked && cs == end && tt_warp_test(&s_full[(cs - 1) & 1], ((cs - 1) >> 1) & 1) &&
                           tt_warp_test(&u_full[slot ^ 1], ((k + 1) >> 1) & 1)) {
                    // all S products are done, the last weights are not yet: time for the next unit's Q
                    const TreeUnit next = unit_at(slot ^ 1);
                    if (next.npages > 0) ask_q(next);
                    asked = true;
                    spin = 0;
                } else if (++spin > LUMEN_SPIN_LIMIT || __any_sync(0xffffffffu, *abort_flag != 0)) {
                    ok = false;
                    break;
                }
            }
            if (ok && lane == 0) pt_mbar_arrive(&u_empty[slot]);
        }
        // its copies and products in flight end before the tensor memory is given back, whichever role gives up
        asm volatile("cp.async.wait_all;" ::: "memory");
        if (lane == 0) {
            if (!ok) {
                *abort_flag = 1;
                atomicExch(t.err, 1);
            }
            if (cs > 0) mbar_wait(&s_full[(cs - 1) & 1], ((cs - 1) >> 1) & 1);
            if (cv > 0) mbar_wait(&pv_done[(cv - 1) & 1], ((cv - 1) >> 1) & 1);
        }
        __syncwarp();
    } else {
        const int r = (warp & 3) * 32 + lane;            // this thread's row of a unit
        const uint32_t lane_addr = tmem_base + ((uint32_t)((warp & 3) * 32) << 16);
        int meetings = 0;
        auto meet = [&]() {                              // all four warps
            __syncwarp();
            if (lane == 0) pt_mbar_arrive(together);
            return tt_warp_wait(together, meetings++ & 1);
        };
        TreeUnit x;
        auto read_unit = [&](int k) {
            if (!tt_warp_wait(&u_full[k & 1], (k >> 1) & 1)) return false;
            volatile int* from = s_unit + (k & 1) * TT_UNIT_INTS;
            x.npages = from[0]; x.pg0 = from[1]; x.b = from[2]; x.n0 = from[3]; x.q = from[4]; x.start = from[5]; x.end = from[6];
            x.f0 = from[7]; x.kvh = from[8]; x.slot = from[9];
            return true;
        };
        int c = 0;
        bool ok = read_unit(0);
        for (int k = 0; ok && x.npages > 0; ++k) {
            const TreeSeq sq = {x.n0, x.q, x.start, x.end};
            const int nrows = min(PT_ROWS, sq.q * G - x.f0), f = x.f0 + min(r, nrows - 1), node = f / G, head = x.kvh * G + f % G;
            const bool row_ok = r < nrows;
            const int n = sq.n0 + node, pg0 = x.pg0, npages = x.npages;
            const unsigned long long* mask = a.mask + (size_t)n * a.W;
            int prow = 0, lo_last = 0;                   // this row's position, the last of all rows' window edges
            if (a.window > 0) {
                prow = max(a.tok_pos[n], sq.start);
                int top = sq.start;
                for (int i = lane; i < PT_ROWS; i += 32)
                    if (i < nrows) top = max(top, a.tok_pos[sq.n0 + (x.f0 + i) / G]);
                lo_last = max(0, __reduce_max_sync(0xffffffffu, top) - a.window + 1);
            }
            auto masked = [&](int jb) { return jb + LUMEN_PAGE > sq.start || jb < lo_last; };      // the same for every row
            if ((pg0 + npages) * LUMEN_PAGE > sq.start) tt_prefetch(mask);
            bool any_masked = false;
            float m_ref = -INFINITY, l = 0.0f;
            for (int it = 0; it < npages; ++it, ++c) {
                if (__any_sync(0xffffffffu, *abort_flag != 0)) { ok = false; break; }
                if (!tt_warp_wait(&s_full[c & 1], (c >> 1) & 1)) { ok = false; break; }
                pt_fence_after();
                float s[64];
                pt_ld64(lane_addr + (c & 1) * LUMEN_PAGE, s);
                const int jb = (pg0 + it) * LUMEN_PAGE;
                const bool part = masked(jb);
                uint32_t s0 = ~0u, s1 = ~0u;             // the keys that this row sees
                if (part) {
                    const unsigned long long seen = row_ok ? tree_seen(jb, sq, mask, a.W, prow, a.window, a.tok_pos + sq.n0) : 0ull;
                    s0 = (uint32_t)seen;
                    s1 = (uint32_t)(seen >> 32);
                }
                if (CAP) {       // capped scores: tanh here, times softcap * log2(e) (scale_log2) below
                    if (part) {
#pragma unroll
                        for (int j = 0; j < 32; ++j) {
                            s[j] = (s0 >> j) & 1 ? s[j] : 0.0f;
                            s[32 + j] = (s1 >> j) & 1 ? s[32 + j] : 0.0f;
                        }
                    }
                    // a row takes the one or the other by the scores of its own that it sees, whatever its neighbours have
                    float big[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int j = 0; j < 64; j += 8)
#pragma unroll
                        for (int h = 0; h < 4; ++h) big[h] = pt_max3(big[h], fabsf(s[j + 2 * h]), fabsf(s[j + 2 * h + 1]));
                    if (!row_ok || fmaxf(fmaxf(big[0], big[1]), fmaxf(big[2], big[3])) * t.cap_pre <= 0.5f) {
#pragma unroll
                        for (int j = 0; j < 64; j += 2) tt_tanh_small(s[j], s[j + 1], t.cap_pre);
                    } else {
#pragma unroll
                        for (int j = 0; j < 64; ++j) s[j] = pt_tanh(s[j] * t.cap_pre);
                    }
                    __syncwarp();
                }
                if (part) {
                    any_masked = true;
#pragma unroll
                    for (int j = 0; j < 32; ++j) {
                        s[j] = (s0 >> j) & 1 ? s[j] : -INFINITY;
                        s[32 + j] = (s1 >> j) & 1 ? s[32 + j] : -INFINITY;
                    }
                    // values that are no numbers: 16 bytes a thread at a time, neighbours' side by side
                    const int st = c % TT_STAGES;
                    if (!tt_warp_wait(&v_full[st], (c / TT_STAGES) & 1)) { ok = false; break; }
                    uint4* tile = reinterpret_cast<uint4*>(sKV + st * STAGE_BYTES + K_BYTES);
                    bool bad = false, wrote = false;
#pragma unroll 4
                    for (int i = threadIdx.x - 64; i < V_BYTES / 16; i += 128) {
                        uint4 v = tile[i];
                        uint32_t* p = reinterpret_cast<uint32_t*>(&v);
                        bool here = false;
#pragma unroll
                        for (int h = 0; h < 4; ++h) {                // exponents of all ones
                            if ((p[h] & 0x7f80u) == 0x7f80u) { p[h] &= 0xffff0000u; here = true; }
                            if ((p[h] & 0x7f800000u) == 0x7f800000u) { p[h] &= 0x0000ffffu; here = true; }
                        }
                        if (here) {
                            tile[i] = v;
                            wrote = true;
                            bad |= jb + ((i >> 3) & (LUMEN_PAGE - 1)) < sq.end;
                        }
                    }
                    if (bad) s_bad[k & 1] = k + 1;               // every writer writes the same
                    if (wrote) asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    __syncwarp();
                }
                // row maximum of the raw scores, four independent chains (the scale is positive)
                float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int j = 0; j < 64; j += 8) {
                    mx4[0] = pt_max3(mx4[0], s[j], s[j + 1]);
                    mx4[1] = pt_max3(mx4[1], s[j + 2], s[j + 3]);
                    mx4[2] = pt_max3(mx4[2], s[j + 4], s[j + 5]);
                    mx4[3] = pt_max3(mx4[3], s[j + 6], s[j + 7]);
                }
                const float mx = row_ok ? fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3])) * t.scale_log2 : -INFINITY;
                // reference for the exponentials: moved only when the maximum has grown a lot
                float corr = 1.0f;
                if (mx > m_ref + TT_RESCALE || m_ref == -INFINITY) {
                    const float nref = fmaxf(mx, m_ref);
                    if (nref != -INFINITY) {
                        corr = (m_ref == -INFINITY) ? 0.0f : pt_ex2(m_ref - nref);
                        m_ref = nref;
                    }
                }
                const float nbase = (m_ref == -INFINITY) ? 0.0f : -m_ref;
                pt_f2 rs[4] = {0ull, 0ull, 0ull, 0ull};
                const pt_f2 scale2 = pt_pair(t.scale_log2, t.scale_log2), nbase2 = pt_pair(nbase, nbase);
#pragma unroll
                for (int j = 0; j < 64; j += 8) {
#pragma unroll
                    for (int h = 0; h < 4; ++h) {
                        float& x0 = s[j + 2 * h];
                        float& x1 = s[j + 2 * h + 1];
                        pt_unpair(pt_fma2(pt_pair(x0, x1), scale2, nbase2), x0, x1);
                        x0 = pt_ex2(x0);
                        x1 = pt_ex2(x1);
                        rs[h] = pt_add2(rs[h], pt_pair(x0, x1));
                    }
                }
                float l_even, l_odd;
                pt_unpair(pt_add2(pt_add2(rs[0], rs[1]), pt_add2(rs[2], rs[3])), l_even, l_odd);
                l = l * corr + (l_even + l_odd);
                // O is rescaled rarely; only then must the PV product of the page before be done
                if (it > 0 && __any_sync(0xffffffffu, corr != 1.0f)) {
                    if (!tt_warp_wait(&pv_done[(c - 1) & 1], ((c - 1) >> 1) & 1)) { ok = false; break; }
                    pt_fence_after();
#pragma unroll 1
                    for (int c0 = 0; c0 < vw; c0 += 32) {
                        float ov[32];
                        pt_ld32(lane_addr + O_COL + c0, ov);
#pragma unroll
                        for (int j = 0; j < 32; ++j) ov[j] *= corr;
                        pt_st32(lane_addr + O_COL + c0, ov);
                    }
                }
                uint32_t pk[32];
#pragma unroll
                for (int i = 0; i < 32; ++i) pk[i] = pack_bf16(s[2 * i], s[2 * i + 1]);
                pt_st32u(lane_addr + (c & 1) * LUMEN_PAGE, pk);
                asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                pt_fence_before();
                __syncwarp();
                if (lane == 0) pt_mbar_arrive(&p_ready[c & 1]);
            }
            if (!ok) break;
            if (!(ok = tt_warp_wait(&pv_done[(c - 1) & 1], ((c - 1) >> 1) & 1))) break;
            pt_fence_after();
            if (any_masked && !(ok = meet())) break;         // every warp's s_bad
            const bool whole = x.slot < 0, any_bad = any_masked && *(volatile int*)(s_bad + (k & 1)) == k + 1;
            float mul = 1.0f;
            __nv_bfloat16* dst = (__nv_bfloat16*)a.out + ((size_t)n * a.nq + head) * vw;
            float* part = nullptr;
            if (whole) {
                // in units of log 2, beside the sink's term
                if (m_ref == -INFINITY) mul = l == 0.0f ? 0.0f : l;      // no weight at all, or a score that is no number
                else if (!a.sink) mul = 1.0f / l;
                else {
                    const float sk = a.sink[head] * 1.4426950408889634f, top = fmaxf(m_ref, sk), fr = exp2f(m_ref - top);
                    mul = fr / (l * fr + exp2f(sk - top));
                }
            } else {
                const size_t at = (size_t)(2 * blockIdx.x + x.slot) * PT_ROWS + r;
                part = a.part_o + at * vw;
                if (row_ok) a.part_ml[at] = make_float2(m_ref, l);
            }
#pragma unroll 1
            for (int c0 = 0; c0 < vw; c0 += 32) {
                float ov[32];
                __syncwarp();
                pt_ld32(lane_addr + O_COL + c0, ov);
                if (any_bad && row_ok) {
                    // values that are no numbers, where the row sees them: they were zeros in the product
                    for (int it = 0; it < npages; ++it) {
                        const int jb = (pg0 + it) * LUMEN_PAGE;
                        if (!masked(jb)) continue;
                        unsigned long long seen = tree_seen(jb, sq, mask, a.W, prow, a.window, a.tok_pos + sq.n0);
                        const int page = a.block_table[(size_t)x.b * a.bt_stride + pg0 + it];
                        const __nv_bfloat16* vt = vcache + ((size_t)((unsigned)page < (unsigned)a.n_pages ? page : 0) * a.nkv + x.kvh) *
                                                               (size_t)(LUMEN_PAGE * vw);
                        while (seen) {
                            const int key = __ffsll((long long)seen) - 1;
                            seen &= seen - 1;
                            for (int j = 0; j < 32; ++j) {
                                const float y = __bfloat162float(vt[tile_offset(LUMEN_LAYOUT_SW128, key, c0 + j, vw)]);
                                if (!(fabsf(y) <= 3.402823466e38f)) ov[j] += y;
                            }
                        }
                    }
                }
                if (row_ok && whole) {
#pragma unroll
                    for (int j = 0; j < 32; j += 16) {
                        uint32_t w[8];
#pragma unroll
                        for (int i = 0; i < 8; ++i) w[i] = pack_bf16(ov[j + 2 * i] * mul, ov[j + 2 * i + 1] * mul);
                        tt_store32(dst + c0 + j, w);
                    }
                } else if (row_ok) {
#pragma unroll
                    for (int j = 0; j < 32; j += 8) {
                        uint32_t w[8];
#pragma unroll
                        for (int i = 0; i < 8; ++i) w[i] = __float_as_uint(ov[j + i]);
                        tt_store32(part + c0 + j, w);
                    }
                }
            }
            pt_fence_before();                           // O has been read: the next unit's products may write it
            __syncwarp();
            if (lane == 0) pt_mbar_arrive(&u_empty[k & 1]);
            if (!(ok = read_unit(k + 1))) break;
        }
        if (!ok) {
            *abort_flag = 1;
            if (lane == 0) atomicExch(t.err, 1);
        }
    }

    pt_fence_before();
    __syncthreads();
    if (warp == 1) {
        pt_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(NCOLS) : "memory");
    }
}

// Joins the pieces of the row blocks that were cut, in the order of their pages; the blocks of all of its
// cuts share a row block's rows, a thread has four columns of a row at a time. What it takes is the latency of its loads, one behind
// the other: those of TJ_BATCH pieces are under way together, and few registers let all blocks be resident at once.
#define TJ_BATCH 4
#define TJ_SLICES 4               // blocks a cut (16 nodes for 64 sequences: 78 us; with 2 blocks 84, with 8 80)
__global__ void __launch_bounds__(256, 4)
attn_tree_tc_join_kernel(const TreeTc t) {
    pdl_wait();
    pdl_trigger();
    const TreeArgs& a = t.a;
    const int i = blockIdx.x + 1, G = a.nq / a.nkv, quads = a.dv >> 2;
    const TreeJoin join = t.joins[i];
    if (join.pieces == 0) return;
    const int cut0 = i - join.order * join.step;        // the block behind the first cut; piece 0 is in slot 1 of the one before it
    for (int idx = (join.order * TJ_SLICES + blockIdx.y) * 256 + threadIdx.x; idx < join.nrows * quads; idx += (join.pieces - 1) * TJ_SLICES * 256) {
        const int row = idx / quads, e = (idx - row * quads) * 4;
        float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        float l = 0.0f, top = -INFINITY;
        for (int s0 = 0; s0 < join.pieces; s0 += TJ_BATCH) {
            float2 x[TJ_BATCH];
            float4 v[TJ_BATCH];
#pragma unroll
            for (int s = 0; s < TJ_BATCH; ++s) {
                x[s] = make_float2(-INFINITY, 0.0f);
                v[s] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                if (s0 + s < join.pieces) {
                    // the pieces behind: slot 0 of the block behind the first cut and of those that follow
                    const int block = cut0 + (s0 + s - 1) * join.step;
                    const size_t from = (size_t)(2 * block + (s0 + s == 0 ? 1 : 0)) * PT_ROWS + row;
                    x[s] = a.part_ml[from];
                    v[s] = *reinterpret_cast<const float4*>(a.part_o + from * a.dv + e);
                }
            }
            float mn = top;
#pragma unroll
            for (int s = 0; s < TJ_BATCH; ++s) mn = fmaxf(mn, x[s].x);
            // weights in units of log 2; without a maximum there is no weight, or a score that is no number
            const float c = top == -INFINITY ? (l == 0.0f ? 0.0f : 1.0f) : exp2f(top - mn);
            o.x *= c; o.y *= c; o.z *= c; o.w *= c;
            l *= c;
            top = mn;
#pragma unroll
            for (int s = 0; s < TJ_BATCH; ++s) {
                if (x[s].x == -INFINITY && x[s].y == 0.0f) continue;
                const float f = x[s].x == -INFINITY ? 1.0f : exp2f(x[s].x - mn);
                o.x = fmaf(f, v[s].x, o.x); o.y = fmaf(f, v[s].y, o.y);
                o.z = fmaf(f, v[s].z, o.z); o.w = fmaf(f, v[s].w, o.w);
                l = fmaf(f, x[s].y, l);
            }
        }
        const int f = join.f0 + row, node = f / G, head = join.kvh * G + f - node * G;
        const float inv = ta_close(top * 0.6931471805599453f, l, a.sink, head);
        *reinterpret_cast<uint2*>((__nv_bfloat16*)a.out + ((size_t)(join.n0 + node) * a.nq + head) * a.dv + e) =
            make_uint2(pack_bf16(o.x * inv, o.y * inv), pack_bf16(o.z * inv, o.w * inv));
    }
}

// What a call's blocks need: shared memory, blocks that are resident at once (and no more than the work can come to, whatever the
// lengths are), and float32 numbers of scratch: two partial results a block and what to join.
static int tt_smem(int d, int dv) {
    const int smem = PT_ROWS * d * 2 + TT_STAGES * LUMEN_PAGE * (d + dv) * 2 + TT_BAR_WORDS * 8;
    return dv > 128 && smem < 116 * 1024 ? 116 * 1024 : smem;        // values beyond 128: all of the SM's tensor memory for one block
}
static int tt_blocks(int B, int N, int width, int nq, int nkv, int d, int dv) {
    const long long most = 148 * (tt_smem(d, dv) <= 113 * 1024 ? 2 : 1);
    const long long work = ((long long)N * (nq / nkv) / PT_ROWS + B) * nkv * ((long long)width + TT_COST);
    const long long n = (work + TT_SHARE - 1) / TT_SHARE;
    return (int)(n < most ? n : most);
}
static long long tt_floats(int blocks, int dv) { return (long long)blocks * (2 * PT_ROWS * (dv + 2) + 8); }

template <int D, bool CAP>
static cudaError_t tt_go(const TreeTc& t, int blocks, cudaStream_t stream) {
    const TreeArgs& a = t.a;
    const int smem = tt_smem(a.d, a.dv);
    auto k = attn_tree_tc_kernel<D, CAP>;
    cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e == cudaSuccess) e = lumen_launch(k, dim3(blocks), dim3(TT_THREADS), smem, stream, t);
    if (e == cudaSuccess && blocks > 1)
        e = lumen_launch(attn_tree_tc_join_kernel, dim3(blocks - 1, TJ_SLICES), dim3(256), 0, stream, t);
    return e;
}

// Whether the kernel takes these arguments (beside the operands' places, which bulk copies and its wide stores need).
static bool tt_takes(int is_bf16, int B, int N, int width, int nq, int nkv, int d, int dv, int layout, int v_layout, float scale) {
    // the work and a sequence's rows are counted in 30 bits
    const long long work = ((long long)N * (nq / nkv) / PT_ROWS + B) * nkv * ((long long)width + TT_COST);
    return work < (1 << 30) && (long long)N * (nq / nkv) < (1 << 30) && is_bf16 && layout == LUMEN_LAYOUT_SW128 && v_layout == LUMEN_LAYOUT_SW128 && d <= 256 && dv <= 256 && scale > 0.0f;
}
static bool tt_aligned(const void* q, const void* kcache, const void* vcache, const void* out) {
    return !(((uintptr_t)q | (uintptr_t)kcache | (uintptr_t)vcache) & 15) && !((uintptr_t)out & 31);
}
static cudaError_t tt_launch(TreeArgs a, float* scratch, int* err, cudaStream_t stream) {
    const int blocks = tt_blocks(a.B, a.N, a.width, a.nq, a.nkv, a.d, a.dv);
    const size_t rows = (size_t)blocks * 2 * PT_ROWS;
    a.part_o = scratch;
    a.part_ml = (float2*)(scratch + rows * a.dv);
    const bool cap = a.softcap > 0.0f;
    const TreeTc t = {a, (cap ? a.softcap : a.scale) * 1.4426950408889634f, cap ? a.scale / a.softcap : 0.0f,
                      (TreeJoin*)(scratch + rows * (a.dv + 2)), err};
#define TT_GO(D) (cap ? tt_go<D, true>(t, blocks, stream) : tt_go<D, false>(t, blocks, stream))
    if (a.d == 128 && a.dv == 128) return TT_GO(128);
    if (a.d == 64 && a.dv == 64) return TT_GO(64);
    return TT_GO(0);
#undef TT_GO
}
