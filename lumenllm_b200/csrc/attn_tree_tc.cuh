// Tree attention on the 5th-generation tensor cores: bfloat16, swizzled pages, keys and values of multiples of 64 up to 256.
//
// A unit of work is 128 rows (node, query head) of one kv head and one segment of the keys. It is walked a page at a time as
// the prompts' kernel does: S = Q K^T into tensor memory (two buffers), the softmax by four warps with a row a thread, P as
// bfloat16 over the scores it came from, O += P V in tensor memory; K and V tiles by bulk copies through two rings of two
// stages. A block needs half of an SM, so that one's softmax runs under the other's products, and stays: as many blocks as fit the
// device take the units in turn, so that no block is launched for a segment that a short sequence has not, and the next
// unit's keys are under way while the last one's rows are written. Warp 0 finds the units, tells the others through
// shared memory and asks for the tiles, warp 1 issues the products, warps 2 to 5 are the softmax and gather Q. Pages that hold
// nodes, or that a window cuts for some row, are masked: a row has one 64-bit word a page with the keys it sees.
//
// Weights are rounded to bfloat16 because the product takes both operands in one type: half a step, 2^-8 of a weight, which
// the sum over the keys averages; the running sum takes them unrounded.
//
// A masked weight is 0, but 0 times a value that is no number would not be: in masked pages such values are replaced by
// zeros in the tile before the product reads it, and a row that does see one gets it added at the end.
//
// Every wait is bounded, also where warps wait for one another. When one runs out the block raises the error flag, lets the
// other roles run out, waits for its copies, frees its tensor memory and returns.
#pragma once
#include "tmem_attn.cuh"

#define TT_THREADS 192
#define TT_STAGES 2
#define TT_RESCALE 8.0f

struct TreeTc {
    TreeArgs a;
    float scale_log2;             // with CAP softcap * log2(e), what the tanh is multiplied by
    float cap_pre;                // with CAP scale / softcap
    int* err;
};

// A unit: rows f0 .. f0 + 127 of sequence b and kv head kvh over pages pg0 .. pg0 + npages - 1 (npages 0: there is no more).
struct TreeUnit {
    int npages, pg0, b, n0, q, start, end, f0, kvh, seg, nseg;
};
#define TT_UNIT_INTS 11

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
    return __shfl_sync(0xffffffffu, ok, 0) != 0;
}
__device__ __forceinline__ bool tt_warp_test(uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, mbar_test(bar, parity)); }
// One lane of a whole warp, the same one every time.
__device__ __forceinline__ bool tt_elect() {
    uint32_t p;
    asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}" : "=r"(p)::"memory");
    return p != 0;
}

// The units in order, found by a whole warp: lane i holds sequence b0 + i. Sequences in order; of one, segments, then kv
// heads, then row tiles, so that tiles which read the same keys run side by side.
struct TreeFinder {
    int b0, base, count, sum, tiles;
    TreeSeq sq;
    TreePlan plan;
    __device__ __forceinline__ void chunk(const TreeArgs& a, int G, int lane) {
        const int b = b0 + lane;
        count = tiles = 0;
        sq = TreeSeq{0, 0, 0, 0};
        plan = TreePlan{0, 0, 1, 0, 0};
        if (b < a.B) {
            sq = tree_seq(a.cu_q, a.seq_start, b, a.N, a.width);
            if (sq.q > 0) {
                plan = tree_plan(sq, a.window, G);
                tiles = (int)(((long long)sq.q * G + PT_ROWS - 1) / PT_ROWS);
                count = tiles * plan.nseg * a.nkv;
            }
        }
        sum = count;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum += v;
        }
    }
    __device__ __forceinline__ TreeUnit at(const TreeArgs& a, int G, int lane, int u) {
        TreeUnit t = {0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0};
        for (;;) {
            const int total = __shfl_sync(0xffffffffu, sum, 31);
            if (u < base + total) break;
            base += total;
            b0 += 32;
            if (b0 >= a.B) return t;
            chunk(a, G, lane);
        }
        const int src = __ffs(__ballot_sync(0xffffffffu, u < base + sum)) - 1;
        const int x = u - base - __shfl_sync(0xffffffffu, sum - count, src), nt = __shfl_sync(0xffffffffu, tiles, src);
        const int per = __shfl_sync(0xffffffffu, plan.per, src), rem = __shfl_sync(0xffffffffu, plan.rem, src);
        t.b = b0 + src;
        t.n0 = __shfl_sync(0xffffffffu, sq.n0, src);
        t.q = __shfl_sync(0xffffffffu, sq.q, src);
        t.start = __shfl_sync(0xffffffffu, sq.start, src);
        t.end = __shfl_sync(0xffffffffu, sq.end, src);
        t.nseg = __shfl_sync(0xffffffffu, plan.nseg, src);
        t.f0 = (x % nt) * PT_ROWS;
        t.kvh = (x / nt) % a.nkv;
        t.seg = x / nt / a.nkv;
        t.pg0 = __shfl_sync(0xffffffffu, plan.pg_lo, src) + t.seg * per + min(t.seg, rem);
        t.npages = per + (t.seg < rem ? 1 : 0);
        return t;
    }
};

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
        if (threadIdx.x == 0) atomicExch(t.err, 1);
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
    uint64_t* q_ready = u_empty + 2;           // Q of the next unit is in place
    uint64_t* together = q_ready + 1;          // the softmax warps wait for one another
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(together + 1);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    int* s_bad = reinterpret_cast<int*>(tmem_slot + 2);        // [2] unit number + 1 where a visible place of a masked page holds no number
    volatile int* s_unit = s_bad + 2;          // [2][TT_UNIT_INTS]

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
        mbar_init(q_ready, 4);
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
    const __nv_bfloat16* kcache = (const __nv_bfloat16*)a.kcache;
    const __nv_bfloat16* vcache = (const __nv_bfloat16*)a.vcache;

    // Counters of every role: k units and c pages since the block began; page c is in stage c % 2 of its ring and in
    // score buffer c & 1.
    if (warp == 0) {
        TreeFinder find;
        find.b0 = find.base = 0;
        find.chunk(a, G, lane);
        uint32_t ck = 0, cv = 0;                        // K and V tiles asked for
        bool ok = true;
        for (int k = 0, u = blockIdx.x; ok; ++k, u += gridDim.x) {
            const TreeUnit x = find.at(a, G, lane, u);
            const int slot = k & 1;
            if (!(ok = tt_warp_wait(&u_empty[slot], ((k >> 1) & 1) ^ 1))) break;
            if (lane == 0) {
                volatile int* to = s_unit + slot * TT_UNIT_INTS;
                to[0] = x.npages; to[1] = x.pg0; to[2] = x.b; to[3] = x.n0; to[4] = x.q; to[5] = x.start; to[6] = x.end;
                to[7] = x.f0; to[8] = x.kvh; to[9] = x.seg; to[10] = x.nseg;
                pt_mbar_arrive(&u_full[slot]);
            }
            if (x.npages == 0) break;
            const int* bt = a.block_table + (size_t)x.b * a.bt_stride + x.pg0;
            const uint32_t first = cv, end = cv + x.npages;
            int ids = 0, before = 0;                    // page numbers 32 at a time, and the ones before them
            uint32_t spin = 0;
            while (cv < end) {
                // whichever slot is free: K tiles run ahead of V tiles, their slots come free earlier
                if (ck < end && tt_warp_test(&k_empty[ck % TT_STAGES], ((ck / TT_STAGES) & 1) ^ 1)) {
                    const uint32_t i = ck - first, st = ck % TT_STAGES;
                    if ((i & 31) == 0) {
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
        if (lane == 0 && !ok) {
            *abort_flag = 1;
            atomicExch(t.err, 1);
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
        for (int k = 0; ok; ++k) {
            const int slot = k & 1;
            if (!(ok = tt_warp_wait(&u_full[slot], (k >> 1) & 1))) break;
            const uint32_t npages = __shfl_sync(0xffffffffu, s_unit[slot * TT_UNIT_INTS], 0), first = cv, end = cv + npages;
            if (npages == 0) break;
            if (!(ok = tt_warp_wait(q_ready, k & 1))) break;
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
                } else if (++spin > LUMEN_SPIN_LIMIT || __any_sync(0xffffffffu, *abort_flag != 0)) {
                    ok = false;
                    break;
                }
            }
            if (ok && lane == 0) pt_mbar_arrive(&u_empty[slot]);
        }
        if (!ok && lane == 0) { *abort_flag = 1; atomicExch(t.err, 1); }
    } else {
        const int r = (warp & 3) * 32 + lane;            // this thread's row of a unit
        const uint32_t lane_addr = tmem_base + ((uint32_t)((warp & 3) * 32) << 16);
        const __nv_bfloat16* q = (const __nv_bfloat16*)a.q;
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
            x.f0 = from[7]; x.kvh = from[8]; x.seg = from[9]; x.nseg = from[10];
            return true;
        };
        // Q: 128 rows into [kw/64][row][64], 16-byte chunk c of a row at c ^ (row & 7); rows beyond the sequence's are zeros.
        // The products that read the last unit's Q are done: this warp has seen their last scores.
        auto gather_q = [&]() {
            const int nrows = min(PT_ROWS, x.q * G - x.f0), qpieces = kw >> 3;
            constexpr int QL = 8;                        // loads a thread has under way
            for (int base = threadIdx.x - 64; base < PT_ROWS * qpieces; base += QL * 128) {
                uint4 v[QL];
#pragma unroll
                for (int i = 0; i < QL; ++i) {
                    const int idx = base + i * 128, qr = idx / qpieces, c = idx - qr * qpieces, f = x.f0 + qr;
                    v[i] = make_uint4(0u, 0u, 0u, 0u);
                    if (qr < nrows) v[i] = *reinterpret_cast<const uint4*>(q + ((size_t)(x.n0 + f / G) * a.nq + x.kvh * G + f % G) * kw + 8 * c);
                }
#pragma unroll
                for (int i = 0; i < QL; ++i) {
                    const int idx = base + i * 128, qr = idx / qpieces, c = idx - qr * qpieces;
                    if (idx < PT_ROWS * qpieces)
                        *reinterpret_cast<uint4*>(sQ + (c >> 3) * (PT_ROWS * 128) + qr * 128 + (((c & 7) ^ (qr & 7)) << 4)) = v[i];
                }
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");   // Q is read by the tensor cores
            __syncwarp();
            if (lane == 0) pt_mbar_arrive(q_ready);
        };
        int c = 0;
        bool ok = read_unit(0);
        if (ok && x.npages > 0) gather_q();
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
            bool any_masked = false;
            float m_ref = -INFINITY, l = 0.0f;
            for (int it = 0; it < npages; ++it, ++c) {
                if (__any_sync(0xffffffffu, *abort_flag != 0)) { ok = false; break; }
                if (!tt_warp_wait(&s_full[c & 1], (c >> 1) & 1)) { ok = false; break; }
                pt_fence_after();
                float s[64];
                pt_ld64(lane_addr + (c & 1) * LUMEN_PAGE, s);
                if (CAP) {       // capped scores: tanh here, times softcap * log2(e) (scale_log2) below
#pragma unroll
                    for (int j = 0; j < 64; ++j) s[j] = pt_tanh(s[j] * t.cap_pre);
                }
                const int jb = (pg0 + it) * LUMEN_PAGE;
                if (masked(jb)) {
                    any_masked = true;
                    const unsigned long long seen = row_ok ? tree_seen(jb, sq, mask, a.W, prow, a.window, a.tok_pos + sq.n0) : 0ull;
                    const uint32_t s0 = (uint32_t)seen, s1 = (uint32_t)(seen >> 32);
#pragma unroll
                    for (int j = 0; j < 32; ++j) {
                        s[j] = (s0 >> j) & 1 ? s[j] : -INFINITY;
                        s[32 + j] = (s1 >> j) & 1 ? s[32 + j] : -INFINITY;
                    }
                    // this thread's half of a value row, in every block of 64 numbers
                    const int st = c % TT_STAGES, vr = (threadIdx.x - 64) >> 1, half = threadIdx.x & 1;
                    if (!tt_warp_wait(&v_full[st], (c / TT_STAGES) & 1)) { ok = false; break; }
                    unsigned char* row = sKV + st * STAGE_BYTES + K_BYTES + vr * 128 + half * 64;
                    bool bad = false;
                    for (int blk = 0; blk < vw >> 6; ++blk) {
                        uint4* y = reinterpret_cast<uint4*>(row + blk * (LUMEN_PAGE * 128));
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            uint4 v = y[i];
                            uint32_t* p = reinterpret_cast<uint32_t*>(&v);
                            bool here = false;
#pragma unroll
                            for (int h = 0; h < 4; ++h) {            // exponents of all ones
                                if ((p[h] & 0x7f80u) == 0x7f80u) { p[h] &= 0xffff0000u; here = true; }
                                if ((p[h] & 0x7f800000u) == 0x7f800000u) { p[h] &= 0x0000ffffu; here = true; }
                            }
                            if (here) y[i] = v;
                            bad |= here;
                        }
                    }
                    if (bad && jb + vr < sq.end) s_bad[k & 1] = k + 1;         // every writer writes the same
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
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
                const float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3])) * t.scale_log2;
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
            // the next unit's Q while the last product runs
            const TreeUnit now = x;
            if (!(ok = read_unit(k + 1))) break;
            if (x.npages > 0) gather_q();
            if (!(ok = tt_warp_wait(&pv_done[(c - 1) & 1], ((c - 1) >> 1) & 1))) break;
            pt_fence_after();
            if (any_masked && !(ok = meet())) break;         // every warp's s_bad
            const bool whole = now.nseg == 1, any_bad = any_masked && *(volatile int*)(s_bad + (k & 1)) == k + 1;
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
                const long long at = (tree_part_base(now.b, sq.n0, a.width, G) + (long long)node * now.nseg + now.seg) * a.nq + head;
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
                        const int page = a.block_table[(size_t)now.b * a.bt_stride + pg0 + it];
                        const __nv_bfloat16* vt = vcache + ((size_t)((unsigned)page < (unsigned)a.n_pages ? page : 0) * a.nkv + now.kvh) *
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
                    for (int j = 0; j < 32; j += 8) {
                        uint4 v;
                        v.x = pack_bf16(ov[j] * mul, ov[j + 1] * mul);
                        v.y = pack_bf16(ov[j + 2] * mul, ov[j + 3] * mul);
                        v.z = pack_bf16(ov[j + 4] * mul, ov[j + 5] * mul);
                        v.w = pack_bf16(ov[j + 6] * mul, ov[j + 7] * mul);
                        *reinterpret_cast<uint4*>(dst + c0 + j) = v;
                    }
                } else if (row_ok) {
#pragma unroll
                    for (int j = 0; j < 32; j += 4)
                        *reinterpret_cast<float4*>(part + c0 + j) = make_float4(ov[j], ov[j + 1], ov[j + 2], ov[j + 3]);
                }
            }
            pt_fence_before();                           // O has been read: the next unit's products may write it
            __syncwarp();
            if (lane == 0) pt_mbar_arrive(&u_empty[k & 1]);
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

template <int D, bool CAP>
static cudaError_t tt_go(const TreeTc& t, int max_segs, cudaStream_t stream) {
    const TreeArgs& a = t.a;
    int smem = PT_ROWS * a.d * 2 + TT_STAGES * LUMEN_PAGE * (a.d + a.dv) * 2 + 384;
    if (a.dv > 128 && smem < 116 * 1024) smem = 116 * 1024;      // such a block has the SM's tensor memory to itself
    auto k = attn_tree_tc_kernel<D, CAP>;
    cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    // no more units than these come of the tokens and the page table, whatever the lengths are
    const long long units = ((long long)a.N * (a.nq / a.nkv) / PT_ROWS + a.B) * a.nkv * max_segs;
    const long long most = 148 * (smem <= 113 * 1024 ? 2 : 1);      // blocks that are resident at once
    return lumen_launch(k, dim3((unsigned)(units < most ? units : most)), dim3(TT_THREADS), smem, stream, t);
}

// Whether the kernel takes these arguments: 16-byte aligned operands are what bulk copies and its vector loads need.
static bool tt_takes(const TreeArgs& a, int is_bf16) {
    return is_bf16 && a.layout == LUMEN_LAYOUT_SW128 && a.v_layout == LUMEN_LAYOUT_SW128 && a.d <= 256 && a.dv <= 256 && a.scale > 0.0f &&
           !(((uintptr_t)a.q | (uintptr_t)a.kcache | (uintptr_t)a.vcache | (uintptr_t)a.out | (uintptr_t)a.part_o) & 15);
}
static cudaError_t tt_launch(const TreeArgs& a, int max_segs, int* err, cudaStream_t stream) {
    const bool cap = a.softcap > 0.0f;
    const TreeTc t = {a, (cap ? a.softcap : a.scale) * 1.4426950408889634f, cap ? a.scale / a.softcap : 0.0f, err};
    if (a.d == 128 && a.dv == 128) return cap ? tt_go<128, true>(t, max_segs, stream) : tt_go<128, false>(t, max_segs, stream);
    if (a.d == 64 && a.dv == 64) return cap ? tt_go<64, true>(t, max_segs, stream) : tt_go<64, false>(t, max_segs, stream);
    return cap ? tt_go<0, true>(t, max_segs, stream) : tt_go<0, false>(t, max_segs, stream);
}
