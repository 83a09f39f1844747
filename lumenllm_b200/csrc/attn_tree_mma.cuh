// Tree attention for bfloat16 tiles in plain rows (head sizes that are multiples of 8 but not of 64, up to 256) on mma.sync: a block has 64
// rows (node, query head) of one kv head, sixteen a warp, and a segment of the keys. Pages arrive by asynchronous copies, one ahead;
// scores, weights and outputs stay in registers (m16n8k16: what a product leaves of the scores is laid out as the
// next one takes its weights). Rows of shared memory are an odd number of 16 bytes long, so eight rows' pieces lie in different banks.
// It is bound by the latency of a page where a step has few rows (a warp without rows sits out) and by the cache's bytes where
// it has many sequences. 8 x 24 nodes after 1,500 to 2,500 tokens, 32 heads of 80 over 8: 50 us (the float32 kernel 235); 32 x 8 nodes, 16
// heads of 48 over 4: 39 (180). Three blocks of 128 columns an SM instead of two (168 registers instead of 249) took 57 to 50.
#pragma once
#include "tmem_attn.cuh"

#define TM_THREADS 128
#define TM_ROWS 64

// 16-byte pieces of a page's rows to shared memory, rows from `valid` on zeros
__device__ __forceinline__ void tm_stage(unsigned char* dst, int stride, const __nv_bfloat16* tile, int cols, int valid) {
    const int pieces = cols >> 3, step_r = TM_THREADS / pieces, step_c = TM_THREADS - step_r * pieces;
    int r = threadIdx.x / pieces, c = threadIdx.x - r * pieces;
    for (int idx = threadIdx.x; idx < LUMEN_PAGE * pieces; idx += TM_THREADS) {
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst) + r * stride + 16 * c),
                     "l"(tile + (r < valid ? r * cols + 8 * c : 0)), "r"(r < valid ? 16 : 0)
                     : "memory");
        r += step_r;
        c += step_c;
        if (c >= pieces) { c -= pieces; ++r; }
    }
}

// VT: values of up to 8 VT columns.
template <int VT>
__global__ void __launch_bounds__(TM_THREADS, VT == 16 ? 3 : 0)
attn_tree_mma_kernel(const TreeArgs a) {
    pdl_wait();      // nothing of this kernel touches global memory before this
    pdl_trigger();
    extern __shared__ __align__(16) unsigned char tm_smem[];
    __shared__ int s_unit[2], s_tok[TM_ROWS], s_head[TM_ROWS];
    const int G = a.nq / a.nkv, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int kvh = blockIdx.x % a.nkv, seg = blockIdx.y;
    if (tid < 32) {
        int b, tile;
        tree_find(a.cu_q, a.B, a.N, G, TM_ROWS, blockIdx.x / a.nkv, b, tile);
        if (tid == 0) { s_unit[0] = b; s_unit[1] = tile; }
    }
    __syncthreads();
    const int b = s_unit[0];
    if (b >= a.B) return;
    const TreeSeq sq = tree_seq(a.cu_q, a.seq_start, b, a.N, a.width);
    const TreePlan plan = tree_plan(sq, a.window, G, a.seg_min, a.seg_rows);
    if (seg >= plan.nseg) return;
    const int f0 = s_unit[1] * TM_ROWS, nrows = min(TM_ROWS, sq.q * G - f0);
    const int ksteps = (a.d + 15) >> 4, vsteps = (a.dv + 15) >> 4;
    const int k_row = 32 * ksteps + 16, v_row = 32 * vsteps + 16;             // bytes
    const int stage = LUMEN_PAGE * (k_row + v_row);
    unsigned char* sq_ = tm_smem;                       // [64][k_row]
    unsigned char* kv = sq_ + TM_ROWS * k_row;          // [2][64][k_row], [64][v_row]
    const int* bt = a.block_table + (size_t)b * a.bt_stride;
    const int pg0 = plan.first(seg), npages = plan.count(seg);
    const __nv_bfloat16* kcache = (const __nv_bfloat16*)a.kcache;
    const __nv_bfloat16* vcache = (const __nv_bfloat16*)a.vcache;
    auto tile_of = [&](int i) {
        const int page = bt[pg0 + i];
        return ((size_t)((unsigned)page < (unsigned)a.n_pages ? page : 0) * a.nkv + kvh) * (size_t)LUMEN_PAGE;
    };
    auto ask = [&](int i) {
        unsigned char* to = kv + (i & 1) * stage;
        const size_t tile = tile_of(i);
        const int valid = min(LUMEN_PAGE, sq.end - (pg0 + i) * LUMEN_PAGE);
        tm_stage(to, k_row, kcache + tile * a.d, a.d, valid);
        tm_stage(to + LUMEN_PAGE * k_row, v_row, vcache + tile * a.dv, a.dv, valid);
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    ask(0);
    {
        // Q: two threads a row; zeros for rows and columns that there are not, in the pages' places too
        const int r = tid >> 1, f = f0 + min(r, nrows - 1), node = f / G, head = kvh * G + f - node * G;
        if ((tid & 1) == 0) { s_tok[r] = sq.n0 + node; s_head[r] = head; }
        const __nv_bfloat16* src = (const __nv_bfloat16*)a.q + ((size_t)(sq.n0 + node) * a.nq + head) * a.d;
        for (int c = tid & 1; c < 2 * ksteps; c += 2)
            *reinterpret_cast<uint4*>(sq_ + r * k_row + 16 * c) = r < nrows && 8 * c < a.d ? *reinterpret_cast<const uint4*>(src + 8 * c)
                                                                                           : make_uint4(0u, 0u, 0u, 0u);
        unsigned char* row = kv + (tid & 1) * stage;
        if (a.d & 8) *reinterpret_cast<uint4*>(row + r * k_row + 2 * a.d) = make_uint4(0u, 0u, 0u, 0u);
        if (a.dv & 8) *reinterpret_cast<uint4*>(row + LUMEN_PAGE * k_row + r * v_row + 2 * a.dv) = make_uint4(0u, 0u, 0u, 0u);
    }
    __syncthreads();
    const bool idle = 16 * warp >= nrows;               // a warp without rows only copies
    const int ra = 16 * warp + g, rb = ra + 8;          // this lane's rows
    const int tok_a = s_tok[ra], tok_b = s_tok[rb];
    const unsigned long long* mask_a = a.mask + (size_t)tok_a * a.W;
    const unsigned long long* mask_b = a.mask + (size_t)tok_b * a.W;
    const int pos_a = max(a.tok_pos[tok_a], sq.start), pos_b = max(a.tok_pos[tok_b], sq.start);
    const bool cap = a.softcap > 0.0f;
    const float mul = (cap ? a.softcap : a.scale) * 1.4426950408889634f, pre = cap ? a.scale / a.softcap : 0.0f;
    float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.0f, l1 = 0.0f;
    float o[VT][4];
#pragma unroll
    for (int i = 0; i < VT; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;
    bool any_bad = false;
    auto all_seen = [&](int jb) { return jb + LUMEN_PAGE <= sq.start && a.window == 0; };

    for (int i = 0; i < npages; ++i) {
        if (i + 1 < npages) ask(i + 1);
        else asm volatile("cp.async.commit_group;" ::: "memory");
        asm volatile("cp.async.wait_group 1;" ::: "memory");
        __syncthreads();                                // the page is there
        unsigned char* kt = kv + (i & 1) * stage;
        unsigned char* vt = kt + LUMEN_PAGE * k_row;
        const int jb = (pg0 + i) * LUMEN_PAGE;
        const bool all = all_seen(jb);
        if (!all) {
            // values that are no numbers, on a page that some row does not see whole, become zeros; rows that see them get them at the end
            bool bad = false;
            const int pieces = a.dv >> 3;
            for (int idx = tid; idx < LUMEN_PAGE * pieces; idx += TM_THREADS) {
                const int r = idx / pieces;
                uint4* at = reinterpret_cast<uint4*>(vt + r * v_row + 16 * (idx - r * pieces));
                uint4 v = *at;
                uint32_t* p = reinterpret_cast<uint32_t*>(&v);
                bool here = false;
#pragma unroll
                for (int h = 0; h < 4; ++h) {           // exponents of all ones
                    if ((p[h] & 0x7f80u) == 0x7f80u) { p[h] &= 0xffff0000u; here = true; }
                    if ((p[h] & 0x7f800000u) == 0x7f800000u) { p[h] &= 0x0000ffffu; here = true; }
                }
                if (here) *at = v;
                bad |= here;
            }
            any_bad |= __syncthreads_or(bad) != 0;
        }
        if (!idle) {
            float s[8][4];
#pragma unroll
            for (int j = 0; j < 8; ++j) s[j][0] = s[j][1] = s[j][2] = s[j][3] = 0.0f;
            const uint32_t q_at = smem_u32(sq_) + (16 * warp + (lane & 15)) * k_row + 16 * (lane >> 4);
            const uint32_t k_at = smem_u32(kt) + ((lane & 7) + ((lane >> 4) << 3)) * k_row + 16 * ((lane >> 3) & 1);
#pragma unroll 2
            for (int ks = 0; ks < ksteps; ++ks) {
                uint32_t qa[4];
                ldsm_x4(qa, q_at + 32 * ks);
#pragma unroll
                for (int j = 0; j < 8; j += 2) {
                    uint32_t r[4];
                    ldsm_x4(r, k_at + 8 * j * k_row + 32 * ks);
                    mma_bf16(s[j], qa, r[0], r[1]);
                    mma_bf16(s[j + 1], qa, r[2], r[3]);
                }
            }
            if (cap) {
#pragma unroll
                for (int j = 0; j < 8; ++j)
#pragma unroll
                    for (int x = 0; x < 4; ++x) s[j][x] = pt_tanh(s[j][x] * pre);
            }
            if (!all) {
                const unsigned long long sa = ra < nrows ? tree_seen(jb, sq, mask_a, a.W, pos_a, a.window, a.tok_pos + sq.n0) : 0ull;
                const unsigned long long sb = rb < nrows ? tree_seen(jb, sq, mask_b, a.W, pos_b, a.window, a.tok_pos + sq.n0) : 0ull;
#pragma unroll
                for (int j = 0; j < 8; ++j)
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        if (!((sa >> (8 * j + 2 * t + x)) & 1)) s[j][x] = -INFINITY;
                        if (!((sb >> (8 * j + 2 * t + x)) & 1)) s[j][2 + x] = -INFINITY;
                    }
                __syncwarp();
            }
            float x0 = -INFINITY, x1 = -INFINITY;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
#pragma unroll
                for (int x = 0; x < 4; ++x) s[j][x] *= mul;                  // in units of log 2
                x0 = pt_max3(x0, s[j][0], s[j][1]);
                x1 = pt_max3(x1, s[j][2], s[j][3]);
            }
            x0 = fmaxf(x0, __shfl_xor_sync(0xffffffffu, x0, 1));
            x0 = fmaxf(x0, __shfl_xor_sync(0xffffffffu, x0, 2));
            x1 = fmaxf(x1, __shfl_xor_sync(0xffffffffu, x1, 1));
            x1 = fmaxf(x1, __shfl_xor_sync(0xffffffffu, x1, 2));
            const float n0 = fmaxf(m0, x0), n1 = fmaxf(m1, x1);
            const float b0 = n0 == -INFINITY ? 0.0f : n0, b1 = n1 == -INFINITY ? 0.0f : n1;
            const float c0 = m0 == -INFINITY ? 0.0f : pt_ex2(m0 - b0), c1 = m1 == -INFINITY ? 0.0f : pt_ex2(m1 - b1);
            float u0 = 0.0f, u1 = 0.0f;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                s[j][0] = pt_ex2(s[j][0] - b0);
                s[j][1] = pt_ex2(s[j][1] - b0);
                s[j][2] = pt_ex2(s[j][2] - b1);
                s[j][3] = pt_ex2(s[j][3] - b1);
                u0 += s[j][0] + s[j][1];
                u1 += s[j][2] + s[j][3];
            }
            l0 = l0 * c0 + u0;                          // a lane's own keys: put together at the end
            l1 = l1 * c1 + u1;
            m0 = n0;
            m1 = n1;
#pragma unroll
            for (int v = 0; v < VT; ++v) { o[v][0] *= c0; o[v][1] *= c0; o[v][2] *= c1; o[v][3] *= c1; }
            const uint32_t v_at = smem_u32(vt) + (lane & 15) * v_row + 16 * (lane >> 4);
#pragma unroll
            for (int kk = 0; kk < 4; ++kk) {
                // weights are rounded to bfloat16, the values' type: 2^-8 of a weight, averaged by the sum; l has them unrounded
                uint32_t pa[4];
                pa[0] = pack_bf16(s[2 * kk][0], s[2 * kk][1]);
                pa[1] = pack_bf16(s[2 * kk][2], s[2 * kk][3]);
                pa[2] = pack_bf16(s[2 * kk + 1][0], s[2 * kk + 1][1]);
                pa[3] = pack_bf16(s[2 * kk + 1][2], s[2 * kk + 1][3]);
#pragma unroll
                for (int v = 0; v < VT / 2; ++v) {
                    if (v >= vsteps) break;
                    uint32_t r[4];
                    ldsm_x4_t(r, v_at + 16 * kk * v_row + 32 * v);
                    mma_bf16(o[2 * v], pa, r[0], r[1]);
                    mma_bf16(o[2 * v + 1], pa, r[2], r[3]);
                }
            }
        }
        __syncthreads();                                // the page has been read
    }
    if (idle) return;
    l0 += __shfl_xor_sync(0xffffffffu, l0, 1);
    l0 += __shfl_xor_sync(0xffffffffu, l0, 2);
    l1 += __shfl_xor_sync(0xffffffffu, l1, 1);
    l1 += __shfl_xor_sync(0xffffffffu, l1, 2);
    const bool whole = plan.nseg == 1;
    const long long pair0 = tree_part_base(b, sq.n0, a.width, G);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int row = h ? rb : ra;
        if (row >= nrows) continue;
        const int tok = h ? tok_b : tok_a, head = s_head[row];
        const float m = (h ? m1 : m0) * 0.6931471805599453f, l = h ? l1 : l0;
        const long long at = (pair0 + (long long)(tok - sq.n0) * plan.nseg + seg) * a.nq + head;
        const float inv = whole ? ta_close(m, l, a.sink, head) : 1.0f;
        if (!whole && t == 0) a.part_ml[at] = make_float2(m, l);
#pragma unroll
        for (int v = 0; v < VT; ++v) {
            const int e = 8 * v + 2 * t;
            if (e >= a.dv) break;
            float y[2] = {o[v][2 * h], o[v][2 * h + 1]};
            if (any_bad)
                for (int i = 0; i < npages; ++i) {
                    const int jb = (pg0 + i) * LUMEN_PAGE;
                    if (all_seen(jb)) continue;
                    unsigned long long seen = tree_seen(jb, sq, h ? mask_b : mask_a, a.W, h ? pos_b : pos_a, a.window, a.tok_pos + sq.n0);
                    const __nv_bfloat16* tile = vcache + tile_of(i) * a.dv + e;
                    while (seen) {
                        const int key = __ffsll((long long)seen) - 1;
                        seen &= seen - 1;
                        for (int x = 0; x < 2; ++x) {
                            const float z = __bfloat162float(tile[key * a.dv + x]);
                            if (!(fabsf(z) <= 3.402823466e38f)) y[x] += z;
                        }
                    }
                }
            if (whole) {
                __nv_bfloat16* dst = (__nv_bfloat16*)a.out + ((size_t)tok * a.nq + head) * a.dv + e;
                dst[0] = __float2bfloat16_rn(y[0] * inv);
                dst[1] = __float2bfloat16_rn(y[1] * inv);
            } else {
                *reinterpret_cast<float2*>(a.part_o + at * a.dv + e) = make_float2(y[0], y[1]);
            }
        }
    }
}

// Whether it takes these: rows of whole 16 bytes in plain tiles.
static bool tm_takes(const TreeArgs& a, int is_bf16) {
    return is_bf16 && a.layout == LUMEN_LAYOUT_LINEAR && a.v_layout == LUMEN_LAYOUT_LINEAR && a.d % 8 == 0 && a.dv % 8 == 0 && a.d <= 256 &&
           a.dv <= 256 && a.scale > 0.0f && !(((uintptr_t)a.q | (uintptr_t)a.kcache | (uintptr_t)a.vcache) & 15);
}
template <int VT>
static cudaError_t tm_run(const TreeArgs& a, const int* tok_seq, int max_segs, cudaStream_t stream) {
    const int k_row = 32 * ((a.d + 15) / 16) + 16, v_row = 32 * ((a.dv + 15) / 16) + 16;
    const int smem = TM_ROWS * k_row + 2 * LUMEN_PAGE * (k_row + v_row);
    auto k = attn_tree_mma_kernel<VT>;
    cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    const long long tiles = (long long)a.N * (a.nq / a.nkv) / TM_ROWS + a.B;
    e = lumen_launch(k, dim3((unsigned)(tiles * a.nkv), max_segs), dim3(TM_THREADS), smem, stream, a);
    if (e != cudaSuccess || max_segs == 1) return e;
    return lumen_launch(attn_tree_join_kernel<__nv_bfloat16>, dim3(a.N, ((a.dv + 3) / 4 * a.nq + 127) / 128), dim3(128), 0, stream, a, tok_seq);
}
static cudaError_t tm_go(const TreeArgs& a, const int* tok_seq, int max_segs, cudaStream_t stream) {
    if (a.dv <= 64) return tm_run<8>(a, tok_seq, max_segs, stream);
    return a.dv <= 128 ? tm_run<16>(a, tok_seq, max_segs, stream) : tm_run<32>(a, tok_seq, max_segs, stream);
}
