// Tree attention on the 5th-generation tensor cores: bfloat16, swizzled pages, keys and values of multiples of 64 up to 256.
//
// A block takes 128 rows (node, query head) of one kv head and one segment of the keys, and walks it a page at a time as the
// prompts' kernel does: S = Q K^T into tensor memory (two buffers), the softmax by four warps with a row a thread, P as
// bfloat16 over the scores it came from, O += P V in tensor memory; K and V tiles by bulk copies through two rings of two
// stages, a block needing half of an SM so that one's softmax runs under the other's products. Pages that hold
// nodes, or that a window cuts for some row, are masked: a row has one 64-bit word a page with the keys it sees.
//
// Weights are rounded to bfloat16 because the product takes both operands in one type: half a step, 2^-8 of a weight, which
// the sum over the keys averages; the running sum takes them unrounded.
//
// A masked weight is 0, but 0 times a value that is no number would not be: in masked pages such values are replaced by
// zeros in the tile before the product reads it, and a row that does see one gets it added at the end.
#pragma once
#include "tmem_attn.cuh"

#define TT_THREADS 192
#define TT_STAGES 2
#define TT_RESCALE 8.0f
#define TT_PAGE_IDS 128           // page numbers of a segment kept in shared memory

struct TreeTc {
    TreeArgs a;
    float scale_log2;             // with CAP softcap * log2(e), what the tanh is multiplied by
    float cap_pre;                // with CAP scale / softcap
    int* err;
};

// D: keys and values are D wide (64, 128), or (0) d and dv wide.
template <int D, bool CAP>
__global__ void __launch_bounds__(TT_THREADS, 2)
attn_tree_tc_kernel(const TreeTc t) {
    pdl_wait();      // nothing of this kernel touches global memory before this
    pdl_trigger();
    const TreeArgs& a = t.a;
    const int kw = D ? D : a.d, vw = D ? D : a.dv;
    const int K_BYTES = LUMEN_PAGE * kw * 2, V_BYTES = LUMEN_PAGE * vw * 2;
    const int STAGE_BYTES = K_BYTES + V_BYTES;
    const int NCOLS = vw <= 128 ? 256 : 512;            // S0 | S1 | O
    constexpr uint32_t O_COL = 128;
    extern __shared__ __align__(1024) unsigned char smem[];
    if (smem_u32(smem) & 1023u) {                       // operand tiles start on 1,024 bytes
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
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(pv_done + 2);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    int* s_unit = reinterpret_cast<int*>(tmem_slot + 2);       // [2]
    int* s_lo = s_unit + 2;                    // the last of the rows' window edges
    int* s_bad = s_lo + 1;                     // a visible place of a masked page holds a value that is no number
    int* s_pos = s_bad + 1;                    // [256] the nodes' positions
    int* s_page = s_pos + TREE_MAX_NODES;      // [128]

    const int G = a.nq / a.nkv, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int kvh = blockIdx.x % a.nkv, seg = blockIdx.y;
    if (warp == 0) {
        int b, tile;
        tree_find(a.cu_q, a.B, a.N, G, PT_ROWS, blockIdx.x / a.nkv, b, tile);
        if (lane == 0) { s_unit[0] = b; s_unit[1] = tile; *s_lo = 0; *s_bad = 0; }
    }
    __syncthreads();
    const int b = s_unit[0];
    if (b >= a.B) return;
    const TreeSeq sq = tree_seq(a.cu_q, a.seq_start, b, a.N, a.width);
    const TreePlan plan = tree_plan(sq, a.window, G);
    if (seg >= plan.nseg) return;
    const int f0 = s_unit[1] * PT_ROWS, nrows = min(PT_ROWS, sq.q * G - f0);
    const int pg0 = plan.first(seg), npages = plan.count(seg);
    const int* bt = a.block_table + (size_t)b * a.bt_stride;
    auto page_at = [&](int i) {
        const int page = bt[pg0 + i];
        return (unsigned)page < (unsigned)a.n_pages ? page : 0;
    };
    if (threadIdx.x < TT_PAGE_IDS && threadIdx.x < npages) s_page[threadIdx.x] = page_at(threadIdx.x);
    for (int i = threadIdx.x; i < min(sq.q, TREE_MAX_NODES); i += TT_THREADS) s_pos[i] = a.tok_pos[sq.n0 + i];
    __syncthreads();
    auto tile_of = [&](int i) { return (size_t)(i < TT_PAGE_IDS ? s_page[i] : page_at(i)) * a.nkv + kvh; };
    const __nv_bfloat16* kcache = (const __nv_bfloat16*)a.kcache;
    const __nv_bfloat16* vcache = (const __nv_bfloat16*)a.vcache;
    auto load_k = [&](int i) {
        const int st = i % TT_STAGES;
        mbar_expect_tx(&k_full[st], K_BYTES);
        bulk_load(sKV + st * STAGE_BYTES, kcache + tile_of(i) * (size_t)(LUMEN_PAGE * kw), K_BYTES, &k_full[st]);
    };
    auto load_v = [&](int i) {
        const int st = i % TT_STAGES;
        mbar_expect_tx(&v_full[st], V_BYTES);
        bulk_load(sKV + st * STAGE_BYTES + K_BYTES, vcache + tile_of(i) * (size_t)(LUMEN_PAGE * vw), V_BYTES, &v_full[st]);
    };

    if (threadIdx.x == 0) {
        for (int i = 0; i < TT_STAGES; ++i) {
            mbar_init(&k_full[i], 1); mbar_init(&k_empty[i], 1);
            mbar_init(&v_full[i], 1); mbar_init(&v_empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) { mbar_init(&s_full[i], 1); mbar_init(&p_ready[i], 4); mbar_init(&pv_done[i], 1); }
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        for (int i = 0; i < TT_STAGES && i < npages; ++i) { load_k(i); load_v(i); }      // under way while Q is gathered
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                     "r"(NCOLS)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    // Q: 128 rows into [kw/64][row][64], 16-byte chunk c of a row at c ^ (row & 7); rows beyond the sequence's are zeros
    const int qpieces = kw >> 3;
    const __nv_bfloat16* q = (const __nv_bfloat16*)a.q;
    constexpr int QL = D ? (PT_ROWS * D / 8 + TT_THREADS - 1) / TT_THREADS : 8;      // loads a thread has under way
    for (int base = threadIdx.x; base < PT_ROWS * qpieces; base += QL * TT_THREADS) {
        uint4 v[QL];
#pragma unroll
        for (int i = 0; i < QL; ++i) {
            const int idx = base + i * TT_THREADS, r = idx / qpieces, c = idx - r * qpieces, f = f0 + r;
            v[i] = make_uint4(0u, 0u, 0u, 0u);
            if (r < nrows) v[i] = *reinterpret_cast<const uint4*>(q + ((size_t)(sq.n0 + f / G) * a.nq + kvh * G + f % G) * kw + 8 * c);
        }
#pragma unroll
        for (int i = 0; i < QL; ++i) {
            const int idx = base + i * TT_THREADS, r = idx / qpieces, c = idx - r * qpieces;
            if (idx < PT_ROWS * qpieces)
                *reinterpret_cast<uint4*>(sQ + (c >> 3) * (PT_ROWS * 128) + r * 128 + (((c & 7) ^ (r & 7)) << 4)) = v[i];
        }
    }
    // this thread's row, where it has one
    const int r = (warp & 3) * 32 + lane, f = f0 + min(r, nrows - 1), node = f / G, head = kvh * G + f % G;
    const bool row_ok = r < nrows;
    const int n = sq.n0 + node;
    int prow = 0, lorow = 0;
    if (warp >= 2 && a.window > 0) {
        prow = max(a.tok_pos[n], sq.start);
        lorow = max(0, prow - a.window + 1);
        if (row_ok) atomicMax(s_lo, lorow);
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");   // Q is read by the tensor cores
    pt_fence_before();
    __syncthreads();
    pt_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    const int lo_last = *s_lo;

    if (warp == 0) {
        if (lane == 0) {
            // K runs a page ahead of V: its slot comes free earlier
            for (int i = TT_STAGES; i <= npages && !*abort_flag; ++i) {
                if (i < npages) {
                    if (!mbar_wait(&k_empty[i % TT_STAGES], ((i / TT_STAGES) & 1) ^ 1)) { *abort_flag = 1; atomicExch(t.err, 1); break; }
                    load_k(i);
                }
                const int j = i - 1;
                if (j >= TT_STAGES) {
                    if (!mbar_wait(&v_empty[j % TT_STAGES], ((j / TT_STAGES) & 1) ^ 1)) { *abort_flag = 1; atomicExch(t.err, 1); break; }
                    load_v(j);
                }
            }
        }
    } else if (warp == 1) {
        if (lane == 0) {
            constexpr uint32_t idesc_qk = pt_idesc(LUMEN_PAGE, 0);
            const uint32_t idesc_pv = pt_idesc(vw, 1);
            const int k_steps = kw / 16;
            auto issue_qk = [&](int it) {       // S[it & 1] = Q K(it)^T
                const int st = it % TT_STAGES;
                const uint32_t kt = smem_u32(sKV + st * STAGE_BYTES);
#pragma unroll(D ? D / 16 : 1)
                for (int ks = 0; ks < k_steps; ++ks) {
                    const uint32_t aoff = (ks >> 2) * (PT_ROWS * 128) + (ks & 3) * 32;
                    const uint32_t boff = (ks >> 2) * (LUMEN_PAGE * 128) + (ks & 3) * 32;
                    pt_mma(tmem_base + (it & 1) * LUMEN_PAGE, pt_desc(smem_u32(sQ) + aoff, 16),
                           pt_desc(kt + boff, 16), idesc_qk, ks > 0 ? 1u : 0u);
                }
                pt_commit(&k_empty[st]);
                pt_commit(&s_full[it & 1]);
            };
            bool ok = mbar_wait(&k_full[0], 0);
            if (ok) {
                pt_fence_after();
                issue_qk(0);
            }
            for (int it = 0; ok && it < npages && !*abort_flag; ++it) {
                if (it + 1 < npages) {
                    const int st1 = (it + 1) % TT_STAGES;
                    if (!mbar_wait(&k_full[st1], ((it + 1) / TT_STAGES) & 1)) { ok = false; break; }
                    pt_fence_after();
                    issue_qk(it + 1);
                }
                const int st = it % TT_STAGES;
                if (!mbar_wait(&v_full[st], (it / TT_STAGES) & 1)) { ok = false; break; }
                if (!mbar_wait(&p_ready[it & 1], (it >> 1) & 1)) { ok = false; break; }
                pt_fence_after();
                const uint32_t vt = smem_u32(sKV + st * STAGE_BYTES + K_BYTES);
                const uint32_t pt = tmem_base + (it & 1) * LUMEN_PAGE;       // P lies over the first 32 columns of its scores
#pragma unroll
                for (int kk = 0; kk < LUMEN_PAGE / 16; ++kk)
                    pt_mma_ts(tmem_base + O_COL, pt + kk * 8,
                              pt_desc(vt + kk * (16 * 128), LUMEN_PAGE * 128), idesc_pv, (it > 0 || kk > 0) ? 1u : 0u);
                pt_commit(&v_empty[st]);
                pt_commit(&pv_done[it & 1]);
            }
            if (!ok) { *abort_flag = 1; atomicExch(t.err, 1); }
        }
    } else {
        const unsigned long long* mask = a.mask + (size_t)n * a.W;
        const uint32_t lane_addr = tmem_base + ((uint32_t)((warp & 3) * 32) << 16);
        float m_ref = -INFINITY, l = 0.0f;
        bool ok = true;
        auto masked = [&](int jb) { return jb + LUMEN_PAGE > sq.start || jb < lo_last; };      // the same for every row
        for (int it = 0; it < npages; ++it) {
            if (__any_sync(0xffffffffu, *abort_flag != 0)) { ok = false; break; }
            bool w = mbar_wait(&s_full[it & 1], (it >> 1) & 1);
            if (!__all_sync(0xffffffffu, w)) { ok = false; break; }
            pt_fence_after();
            float s[64];
            pt_ld64(lane_addr + (it & 1) * LUMEN_PAGE, s);
            if (CAP) {       // capped scores: tanh here, times softcap * log2(e) (scale_log2) below
#pragma unroll
                for (int j = 0; j < 64; ++j) s[j] = pt_tanh(s[j] * t.cap_pre);
            }
            const int jb = (pg0 + it) * LUMEN_PAGE;
            if (masked(jb)) {
                const unsigned long long seen = row_ok ? tree_seen(jb, sq, mask, a.W, prow, a.window, s_pos) : 0ull;
                const uint32_t s0 = (uint32_t)seen, s1 = (uint32_t)(seen >> 32);
#pragma unroll
                for (int j = 0; j < 32; ++j) {
                    s[j] = (s0 >> j) & 1 ? s[j] : -INFINITY;
                    s[32 + j] = (s1 >> j) & 1 ? s[32 + j] : -INFINITY;
                }
                // this thread's half of a value row, in every block of 64 numbers
                const int st = it % TT_STAGES, vr = (threadIdx.x - 64) >> 1, half = threadIdx.x & 1;
                w = mbar_wait(&v_full[st], (it / TT_STAGES) & 1);
                if (!__all_sync(0xffffffffu, w)) { ok = false; break; }
                unsigned char* row = sKV + st * STAGE_BYTES + K_BYTES + vr * 128 + half * 64;
                bool bad = false;
                for (int blk = 0; blk < vw >> 6; ++blk) {
                    uint4* x = reinterpret_cast<uint4*>(row + blk * (LUMEN_PAGE * 128));
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        uint4 v = x[c];
                        uint32_t* u = reinterpret_cast<uint32_t*>(&v);
                        bool here = false;
#pragma unroll
                        for (int i = 0; i < 4; ++i) {            // exponents of all ones
                            if ((u[i] & 0x7f80u) == 0x7f80u) { u[i] &= 0xffff0000u; here = true; }
                            if ((u[i] & 0x7f800000u) == 0x7f800000u) { u[i] &= 0x0000ffffu; here = true; }
                        }
                        if (here) x[c] = v;
                        bad |= here;
                    }
                }
                if (bad && jb + vr < sq.end) *s_bad = 1;         // every writer writes the same
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
                    float& x = s[j + 2 * h];
                    float& y = s[j + 2 * h + 1];
                    pt_unpair(pt_fma2(pt_pair(x, y), scale2, nbase2), x, y);
                    x = pt_ex2(x);
                    y = pt_ex2(y);
                    rs[h] = pt_add2(rs[h], pt_pair(x, y));
                }
            }
            float l_even, l_odd;
            pt_unpair(pt_add2(pt_add2(rs[0], rs[1]), pt_add2(rs[2], rs[3])), l_even, l_odd);
            l = l * corr + (l_even + l_odd);
            // O is rescaled rarely; only then must the PV product of the page before be done
            if (it > 0 && __any_sync(0xffffffffu, corr != 1.0f)) {
                w = mbar_wait(&pv_done[(it - 1) & 1], ((it - 1) >> 1) & 1);
                if (!__all_sync(0xffffffffu, w)) { ok = false; break; }
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
            for (int c = 0; c < 32; ++c) pk[c] = pack_bf16(s[2 * c], s[2 * c + 1]);
            pt_st32u(lane_addr + (it & 1) * LUMEN_PAGE, pk);
            asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
            pt_fence_before();
            __syncwarp();
            if (lane == 0) pt_mbar_arrive(&p_ready[it & 1]);
        }
        if (ok) {
            const bool w = mbar_wait(&pv_done[(npages - 1) & 1], ((npages - 1) >> 1) & 1);
            ok = __all_sync(0xffffffffu, w);
        }
        if (!ok) {
            *abort_flag = 1;
            if (lane == 0) atomicExch(t.err, 1);
        }
        asm volatile("bar.sync 1, 128;" ::: "memory");       // every warp's s_bad
        if (ok) {
            pt_fence_after();
            const bool whole = plan.nseg == 1, any_bad = *(volatile int*)s_bad != 0;
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
                const long long at = (tree_part_base(b, sq.n0, a.width, G) + (long long)node * plan.nseg + seg) * a.nq + head;
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
                        unsigned long long seen = tree_seen(jb, sq, mask, a.W, prow, a.window, s_pos);
                        const __nv_bfloat16* vt = vcache + tile_of(it) * (size_t)(LUMEN_PAGE * vw);
                        while (seen) {
                            const int key = __ffsll((long long)seen) - 1;
                            seen &= seen - 1;
                            for (int j = 0; j < 32; ++j) {
                                const float x = __bfloat162float(vt[tile_offset(LUMEN_LAYOUT_SW128, key, c0 + j, vw)]);
                                if (!(fabsf(x) <= 3.402823466e38f)) ov[j] += x;
                            }
                        }
                    }
                }
                if (!row_ok) continue;
                if (whole) {
#pragma unroll
                    for (int j = 0; j < 32; j += 8) {
                        uint4 v;
                        v.x = pack_bf16(ov[j] * mul, ov[j + 1] * mul);
                        v.y = pack_bf16(ov[j + 2] * mul, ov[j + 3] * mul);
                        v.z = pack_bf16(ov[j + 4] * mul, ov[j + 5] * mul);
                        v.w = pack_bf16(ov[j + 6] * mul, ov[j + 7] * mul);
                        *reinterpret_cast<uint4*>(dst + c0 + j) = v;
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < 32; j += 4)
                        *reinterpret_cast<float4*>(part + c0 + j) = make_float4(ov[j], ov[j + 1], ov[j + 2], ov[j + 3]);
                }
            }
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
    int smem = PT_ROWS * a.d * 2 + TT_STAGES * LUMEN_PAGE * (a.d + a.dv) * 2 + 256 + 4 * (TREE_MAX_NODES + TT_PAGE_IDS);
    if (a.dv > 128 && smem < 116 * 1024) smem = 116 * 1024;      // such a block has the SM's tensor memory to itself
    auto k = attn_tree_tc_kernel<D, CAP>;
    cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    const long long tiles = (long long)a.N * (a.nq / a.nkv) / PT_ROWS + a.B;
    return lumen_launch(k, dim3((unsigned)(tiles * a.nkv), max_segs), dim3(TT_THREADS), smem, stream, t);
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
