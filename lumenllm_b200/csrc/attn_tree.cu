// Attention of a tree of drafted tokens over the paged cache: node i of a sequence sees the cached keys and the nodes that its
// mask names (its ancestors and itself),
//   o_i = sum_j a_ij v_j / (sum_j a_ij + exp(sink)),   a_ij = exp(f(scale q_i . k_j)),   f(x) = x or c tanh(x / c),
// where with a window w only keys within w positions before the node's own position count (a node's position is its depth
// behind the cached tokens, not its index in the cache). A row that sees no key is 0. Keys and values of masked places never
// reach a result, whatever they hold.
//
// Three kernels. Swizzled bfloat16 pages go to the 5th-generation tensor cores (attn_tree_tc.cuh), bfloat16 pages in plain rows to
// mma.sync (attn_tree_mma.cuh); this file has the general kernel (float32 and bfloat16, any key and value size up to 512, any
// head ratio, both tile layouts; all arithmetic float32 with expf and tanhf), and what joins the segments of it and of the second.
//
// General kernel: a block has 32 rows (node, query head) of one kv head and a segment of the keys, and takes a page (64 keys)
// at a time through shared memory in float32: scores by register tiles of 4 rows x 4 keys (the two float32 products of one instruction
// are neighbouring numbers of a key), the softmax with a running maximum and sum, values by tiles of 8 rows x 8 columns a thread (two
// rows an instruction), the even keys by one half of the block, the odd ones by the other. What bounds it is what shared memory
// hands to registers, 128 bytes a cycle: a tile's side is what counts, and reads that all lanes share cost as much as others (scores of 8
// rows x 2 keys a lane, a warp's rows read by all its lanes, took longer). Float32 tiles are asked for ahead, by
// asynchronous copies: keys under the products of the values before them and the other way round; bfloat16 tiles are
// converted on the way, and tiles that do not fit twice are taken one behind the other.
#include "tmem_attn.cuh"
#include "tree_plan.cuh"

#define TA_THREADS 128
#define TA_ROWS 32
#define TA_PROW 36                // numbers a key's row of weights takes in shared memory
#define TA_LOADS 8                // 16-byte loads that a thread has under way

struct TreeArgs {
    const void* q;
    const void* kcache;
    const void* vcache;
    const int* block_table;
    const int* cu_q;
    const int* seq_start;
    const int* tok_pos;
    const unsigned long long* mask;
    void* out;
    float* part_o;                // [pairs][nq][dv]
    float2* part_ml;              // [pairs][nq]: running maximum and sum
    const float* sink;
    int bt_stride, width, W, B, N, n_pages, nq, nkv, d, dv, window, layout, v_layout, vec, seg_min, seg_rows;
    float scale, softcap;
};

// the denominator's reciprocal for sums whose reference is m (natural units), beside the sink's term; rescales by `f`
__device__ __forceinline__ float ta_close(float m, float l, const float* sink, int head) {
    if (m == -INFINITY) return l == 0.0f ? 0.0f : l;        // no weight at all, or a score that is no number
    if (!sink) return 1.0f / l;
    const float s = sink[head], top = fmaxf(m, s), f = expf(m - top);
    return f / (l * f + expf(s - top));
}

// A page tile of `cols` numbers a row into rows of `stride` float32: whole numbers up to `pad` columns (zeros behind cols); rows from
// `valid` on are zeros.
template <typename T>
__device__ __forceinline__ void ta_stage(float* dst, int stride, int pad, const T* tile, int cols, int layout, int valid, bool vec) {
    if (vec) {
        constexpr int E = 16 / (int)sizeof(T);
        const int pieces = cols / E, all = LUMEN_PAGE * pieces;
        const int step_r = TA_THREADS / pieces, step_c = TA_THREADS - step_r * pieces;
        int r = threadIdx.x / pieces, c = threadIdx.x - r * pieces;
        for (int base = threadIdx.x; base < all; base += TA_LOADS * TA_THREADS) {
            uint4 raw[TA_LOADS];
            int at[TA_LOADS];
#pragma unroll
            for (int i = 0; i < TA_LOADS; ++i) {
                raw[i] = make_uint4(0u, 0u, 0u, 0u);
                at[i] = r * stride + c * E;
                if (r < valid) raw[i] = *reinterpret_cast<const uint4*>(tile + tile_offset(layout, r, c * E, cols));
                r += step_r;
                c += step_c;
                if (c >= pieces) { c -= pieces; ++r; }
            }
#pragma unroll
            for (int i = 0; i < TA_LOADS; ++i) {
                if (base + i * TA_THREADS >= all) break;
                const T* x = reinterpret_cast<const T*>(&raw[i]);
#pragma unroll
                for (int e = 0; e < E; e += 4)
                    *reinterpret_cast<float4*>(dst + at[i] + e) = make_float4(to_f32(x[e]), to_f32(x[e + 1]), to_f32(x[e + 2]), to_f32(x[e + 3]));
            }
        }
    } else {
        for (int idx = threadIdx.x; idx < LUMEN_PAGE * pad; idx += TA_THREADS) {
            const int r = idx / pad, e = idx - r * pad;
            dst[r * stride + e] = (r < valid && e < cols) ? to_f32(tile[tile_offset(layout, r, e, cols)]) : 0.0f;
        }
    }
}
// The same for float32 rows of whole 16 bytes, without waiting for them.
__device__ __forceinline__ void ta_stage_async(float* dst, int stride, const float* tile, int cols, int valid) {
    const int pieces = cols >> 2, step_r = TA_THREADS / pieces, step_c = TA_THREADS - step_r * pieces;
    int r = threadIdx.x / pieces, c = threadIdx.x - r * pieces;
    for (int idx = threadIdx.x; idx < LUMEN_PAGE * pieces; idx += TA_THREADS) {
        const int bytes = r < valid ? 16 : 0;           // 0: zeros, nothing is read
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst + r * stride + 4 * c)),
                     "l"(tile + (r < valid ? r * cols + 4 * c : 0)), "r"(bytes)
                     : "memory");
        r += step_r;
        c += step_c;
        if (c >= pieces) { c -= pieces; ++r; }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
}

// ASYNC: keys and values have places of their own, and copies run ahead (float32 in rows of whole 16 bytes).
template <typename T, int NC, bool ASYNC>
__global__ void __launch_bounds__(TA_THREADS)
attn_tree_kernel(const TreeArgs a) {
    pdl_wait();      // nothing of this kernel touches global memory before this
    pdl_trigger();
    extern __shared__ __align__(16) float ta_smem[];
    __shared__ __align__(16) float s_corr[TA_ROWS];
    __shared__ int s_unit[2], s_tok[TA_ROWS], s_head[TA_ROWS];
    __shared__ float2 s_ml[TA_ROWS];
    const int G = a.nq / a.nkv, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int kvh = blockIdx.x % a.nkv, seg = blockIdx.y;
    if (tid < 32) {
        int b, tile;
        tree_find(a.cu_q, a.B, a.N, G, TA_ROWS, blockIdx.x / a.nkv, b, tile);
        if (tid == 0) { s_unit[0] = b; s_unit[1] = tile; }
    }
    __syncthreads();
    const int b = s_unit[0];
    if (b >= a.B) return;
    const TreeSeq sq = tree_seq(a.cu_q, a.seq_start, b, a.N, a.width);
    const TreePlan plan = tree_plan(sq, a.window, G, a.seg_min, a.seg_rows);
    if (seg >= plan.nseg) return;
    const int f0 = s_unit[1] * TA_ROWS, nrows = min(TA_ROWS, sq.q * G - f0);
    const int dp = (a.d + 3) & ~3, ks = dp + 4;
    constexpr int VS = 128 * NC;
    float* qs = ta_smem;                          // [32][ks]
    float* ps = qs + TA_ROWS * ks;                // [64][TA_PROW]: weights, a key's rows together
    float* keys = ps + LUMEN_PAGE * TA_PROW;      // [64][ks]
    float* vals = ASYNC ? keys + LUMEN_PAGE * ks : keys;      // [64][VS]
    const T* q = (const T*)a.q;
    const int* bt = a.block_table + (size_t)b * a.bt_stride;
    const int pg0 = plan.first(seg), npages = plan.count(seg);
    auto tile_of = [&](int i) {
        const int page = bt[pg0 + i];
        return ((size_t)((unsigned)page < (unsigned)a.n_pages ? page : 0) * a.nkv + kvh) * (size_t)LUMEN_PAGE;
    };
    auto valid_of = [&](int i) { return min(LUMEN_PAGE, sq.end - (pg0 + i) * LUMEN_PAGE); };
    if (ASYNC) {
        const size_t tile = tile_of(0);
        ta_stage_async(keys, ks, (const float*)a.kcache + tile * a.d, a.d, valid_of(0));
        ta_stage_async(vals, VS, (const float*)a.vcache + tile * a.dv, a.dv, valid_of(0));
    }
    {
        // Q: four threads a row
        const int r = tid >> 2, f = f0 + min(r, nrows - 1), node = f / G, head = kvh * G + f - node * G;
        if ((tid & 3) == 0) { s_tok[r] = sq.n0 + node; s_head[r] = head; }
        const T* src = q + ((size_t)(sq.n0 + node) * a.nq + head) * a.d;
        float* dst = qs + r * ks;
        if (a.vec & 4) {
            constexpr int E = 16 / (int)sizeof(T);
            const int pieces = r < nrows ? a.d / E : 0;
            for (int c0 = tid & 3; c0 < pieces; c0 += 4 * TA_LOADS) {
                uint4 raw[TA_LOADS];
#pragma unroll
                for (int i = 0; i < TA_LOADS; ++i)
                    if (c0 + 4 * i < pieces) raw[i] = *reinterpret_cast<const uint4*>(src + (c0 + 4 * i) * E);
#pragma unroll
                for (int i = 0; i < TA_LOADS; ++i) {
                    if (c0 + 4 * i >= pieces) break;
                    const T* x = reinterpret_cast<const T*>(&raw[i]);
#pragma unroll
                    for (int e = 0; e < E; e += 4)
                        *reinterpret_cast<float4*>(dst + (c0 + 4 * i) * E + e) = make_float4(to_f32(x[e]), to_f32(x[e + 1]), to_f32(x[e + 2]), to_f32(x[e + 3]));
                }
            }
        }
        if (r >= nrows || !(a.vec & 4))                  // rows that there are not, columns behind the last
            for (int e = tid & 3; e < dp; e += 4) dst[e] = r < nrows && e < a.d ? to_f32(src[e]) : 0.0f;
    }
    __syncthreads();
    // scores: rows 4 rg .. 4 rg + 3, keys kg, kg + 16, kg + 32, kg + 48 (a warp that has no rows there sits out)
    const int rg = tid >> 4, kg = tid & 15;
    const bool idle = 8 * warp >= nrows;
    const unsigned long long* mask[4];
    int pos[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const int n = s_tok[4 * rg + r];
        mask[r] = a.mask + (size_t)n * a.W;
        pos[r] = max(a.tok_pos[n], sq.start);
    }
    float m[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY}, l[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    // values: rows 8 vr .. 8 vr + 7 in pairs, columns col0 + 64 j .. + 3; the halves of the block have every other key each, or (values
    // beyond 256, for the registers) half of the columns each
    constexpr bool BY_KEYS = NC < 4;
    constexpr int CN = BY_KEYS ? 2 * NC : NC;
    const int half = tid >> 6, vr = (tid >> 4) & 3, col0 = 4 * (tid & 15) + (BY_KEYS ? 0 : 256 * half);
    const bool v_idle = 8 * vr >= nrows;
    pt_f2 acc[4][4 * CN];
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int c = 0; c < 4 * CN; ++c) acc[r][c] = 0ull;

    for (int i = 0; i < npages; ++i) {
        const int jb = (pg0 + i) * LUMEN_PAGE, valid = valid_of(i);
        const size_t tile = tile_of(i);
        if (ASYNC) {
            asm volatile("cp.async.wait_group 1;" ::: "memory");        // the keys; the values may still be under way
        } else {
            __syncthreads();                      // the values before have been read
            ta_stage<T>(keys, ks, dp, (const T*)a.kcache + tile * a.d, a.d, a.layout, valid, a.vec & 1);
        }
        __syncthreads();
        const bool all = jb + LUMEN_PAGE <= sq.start && a.window == 0;       // every row sees the whole page
        if (!idle) {
            pt_f2 s2[4][4];
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int k = 0; k < 4; ++k) s2[r][k] = 0ull;
#pragma unroll 2
            for (int e = 0; e < dp; e += 4) {
                ulonglong2 x[4], y[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) x[r] = *reinterpret_cast<const ulonglong2*>(qs + (4 * rg + r) * ks + e);
#pragma unroll
                for (int k = 0; k < 4; ++k) y[k] = *reinterpret_cast<const ulonglong2*>(keys + (kg + 16 * k) * ks + e);
#pragma unroll
                for (int r = 0; r < 4; ++r)
#pragma unroll
                    for (int k = 0; k < 4; ++k) s2[r][k] = pt_fma2(x[r].y, y[k].y, pt_fma2(x[r].x, y[k].x, s2[r][k]));
            }
            float s[4][4], corr[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const unsigned long long seen = all ? ~0ull : tree_seen(jb, sq, mask[r], a.W, pos[r], a.window, a.tok_pos + sq.n0);
                float top = -INFINITY;
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    float even, odd;
                    pt_unpair(s2[r][k], even, odd);
                    float x = (even + odd) * a.scale;
                    if (a.softcap > 0.0f) x = a.softcap * tanhf(x / a.softcap);
                    s[r][k] = (seen >> (kg + 16 * k)) & 1 ? x : -INFINITY;
                    top = fmaxf(top, s[r][k]);
                }
                __syncwarp();
#pragma unroll
                for (int o = 8; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
                const float mn = fmaxf(m[r], top), base = mn == -INFINITY ? 0.0f : mn;
                corr[r] = m[r] == -INFINITY ? 0.0f : expf(m[r] - mn);
                float sum = 0.0f;
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    s[r][k] = expf(s[r][k] - base);      // 0 for a masked key, also where none has been seen yet
                    sum += s[r][k];
                }
#pragma unroll
                for (int o = 8; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
                l[r] = l[r] * corr[r] + sum;
                m[r] = mn;
            }
#pragma unroll
            for (int k = 0; k < 4; ++k)
                *reinterpret_cast<float4*>(ps + (kg + 16 * k) * TA_PROW + 4 * rg) = make_float4(s[0][k], s[1][k], s[2][k], s[3][k]);
            if (kg == 0) *reinterpret_cast<float4*>(s_corr + 4 * rg) = make_float4(corr[0], corr[1], corr[2], corr[3]);
        }
        __syncthreads();                          // the keys have been read, the weights are there
        if (ASYNC) {
            if (i + 1 < npages) ta_stage_async(keys, ks, (const float*)a.kcache + tile_of(i + 1) * a.d, a.d, valid_of(i + 1));
            else asm volatile("cp.async.commit_group;" ::: "memory");
            asm volatile("cp.async.wait_group 1;" ::: "memory");        // the values
        } else {
            ta_stage<T>(vals, VS, VS, (const T*)a.vcache + tile * a.dv, a.dv, a.v_layout, valid, a.vec & 2);
        }
        __syncthreads();
        bool any_bad = false;
        if (!all) {
            // a value that is no number, on a page that some row does not see whole
            bool bad = false;
            for (int r = warp; r < valid; r += TA_THREADS / 32)
                for (int e = lane; e < a.dv; e += 32) bad |= !(fabsf(vals[r * VS + e]) <= 3.402823466e38f);
            any_bad = __syncthreads_or(bad);
        }
        if (!v_idle) {
            {
                const ulonglong2 c01 = *reinterpret_cast<const ulonglong2*>(s_corr + 8 * vr), c23 = *reinterpret_cast<const ulonglong2*>(s_corr + 8 * vr + 4);
                const pt_f2 c[4] = {c01.x, c01.y, c23.x, c23.y};
#pragma unroll
                for (int r = 0; r < 4; ++r)
#pragma unroll
                    for (int x = 0; x < 4 * CN; ++x) acc[r][x] = pt_fma2(acc[r][x], c[r], 0ull);
            }
#pragma unroll 2
            for (int k = BY_KEYS ? half : 0; k < valid; k += BY_KEYS ? 2 : 1) {
                const ulonglong2 w01 = *reinterpret_cast<const ulonglong2*>(ps + k * TA_PROW + 8 * vr);
                const ulonglong2 w23 = *reinterpret_cast<const ulonglong2*>(ps + k * TA_PROW + 8 * vr + 4);
                const pt_f2 w[4] = {w01.x, w01.y, w23.x, w23.y};
#pragma unroll
                for (int c = 0; c < CN; ++c) {
                    const float4 v = *reinterpret_cast<const float4*>(vals + k * VS + 64 * c + col0);
                    const pt_f2 vv[4] = {pt_pair(v.x, v.x), pt_pair(v.y, v.y), pt_pair(v.z, v.z), pt_pair(v.w, v.w)};
                    if (any_bad) {                // nothing of a masked value, not even 0 times infinity
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            float w0, w1;
                            pt_unpair(w[r], w0, w1);
#pragma unroll
                            for (int x = 0; x < 4; ++x) {
                                float a0, a1, p0, p1;
                                pt_unpair(acc[r][4 * c + x], a0, a1);
                                pt_unpair(pt_fma2(w[r], vv[x], acc[r][4 * c + x]), p0, p1);
                                acc[r][4 * c + x] = pt_pair(w0 != 0.0f ? p0 : a0, w1 != 0.0f ? p1 : a1);
                            }
                        }
                    } else {
#pragma unroll
                        for (int r = 0; r < 4; ++r)
#pragma unroll
                            for (int x = 0; x < 4; ++x) acc[r][4 * c + x] = pt_fma2(w[r], vv[x], acc[r][4 * c + x]);
                    }
                }
            }
        }
        if (ASYNC) {
            __syncthreads();                      // the values have been read
            if (i + 1 < npages) ta_stage_async(vals, VS, (const float*)a.vcache + tile_of(i + 1) * a.dv, a.dv, valid_of(i + 1));
            else asm volatile("cp.async.commit_group;" ::: "memory");
        }
    }
    if (kg == 0)
#pragma unroll
        for (int r = 0; r < 4; ++r) s_ml[4 * rg + r] = make_float2(m[r], l[r]);
    // the two halves' sums come together in the values' place, the even keys' first
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();
    float* sums = vals;                           // [32][VS]
    if (BY_KEYS && half == 1 && !v_idle) {
#pragma unroll
        for (int r = 0; r < 8; ++r)
#pragma unroll
            for (int c = 0; c < CN; ++c) {
                float x[4][2];
#pragma unroll
                for (int i = 0; i < 4; ++i) pt_unpair(acc[r >> 1][4 * c + i], x[i][0], x[i][1]);
                *reinterpret_cast<float4*>(sums + (8 * vr + r) * VS + 64 * c + col0) = make_float4(x[0][r & 1], x[1][r & 1], x[2][r & 1], x[3][r & 1]);
            }
    }
    __syncthreads();
    if ((BY_KEYS && half == 1) || v_idle) return;
    const bool whole = plan.nseg == 1;
    const long long pair0 = tree_part_base(b, sq.n0, a.width, G);
#pragma unroll
    for (int r = 0; r < 8; ++r) {
        const int row = 8 * vr + r;
        if (row >= nrows) break;
        const int tok = s_tok[row], head = s_head[row];
        const float2 ml = s_ml[row];
        const long long at = (pair0 + (long long)(tok - sq.n0) * plan.nseg + seg) * a.nq + head;
        const float inv = whole ? ta_close(ml.x, ml.y, a.sink, head) : 1.0f;
        if (!whole && col0 == 0) a.part_ml[at] = ml;
        T* dst = (T*)a.out + ((size_t)tok * a.nq + head) * a.dv;
        float* part = a.part_o + at * a.dv;
#pragma unroll
        for (int c = 0; c < CN; ++c) {
            const int e = 64 * c + col0;
            float4 y = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (BY_KEYS) y = *reinterpret_cast<const float4*>(sums + row * VS + e);
            float x[4][2];
#pragma unroll
            for (int i = 0; i < 4; ++i) pt_unpair(acc[r >> 1][4 * c + i], x[i][0], x[i][1]);
            const float v[4] = {x[0][r & 1] + y.x, x[1][r & 1] + y.y, x[2][r & 1] + y.z, x[3][r & 1] + y.w};
            if (!whole && (a.dv & 3) == 0) {
                if (e < a.dv) *reinterpret_cast<float4*>(part + e) = make_float4(v[0], v[1], v[2], v[3]);
                continue;
            }
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (e + i < a.dv) {
                    if (whole) dst[e + i] = from_f32<T>(v[i] * inv);
                    else part[e + i] = v[i];
                }
        }
    }
}

__device__ __forceinline__ unsigned ta_pack(float lo, float hi) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const unsigned*>(&v);
}

// Joins the segments of the sequences that have more than one, in rising order: a thread has four columns of a (token, head).
template <typename T>
__global__ void __launch_bounds__(128)
attn_tree_join_kernel(const TreeArgs a, const int* __restrict__ tok_seq) {
    pdl_wait();
    pdl_trigger();
    const int n = blockIdx.x, b = tok_seq[n];
    if ((unsigned)b >= (unsigned)a.B) return;
    const int G = a.nq / a.nkv;
    const TreeSeq sq = tree_seq(a.cu_q, a.seq_start, b, a.N, a.width);
    if (n < sq.n0 || n >= sq.n0 + sq.q) return;
    const TreePlan plan = tree_plan(sq, a.window, G, a.seg_min, a.seg_rows);
    if (plan.nseg == 1) return;                   // done by its own block
    const int quads = (a.dv + 3) / 4, idx = blockIdx.y * 128 + threadIdx.x;
    if (idx >= a.nq * quads) return;
    const int head = idx / quads, e = (idx - head * quads) * 4;
    const long long pair = tree_part_base(b, sq.n0, a.width, G) + (long long)(n - sq.n0) * plan.nseg;
    const float2* ml = a.part_ml + pair * a.nq + head;
    const float* src = a.part_o + (pair * a.nq + head) * (long long)a.dv + e;
    const long long row = (long long)a.nq * a.dv;
    const bool quad = (a.dv & 3) == 0, quad_out = quad && ((uintptr_t)a.out & 7) == 0;
    // one pass, a batch of segments at a time: their loads are under way together
    constexpr int BATCH = 8;
    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    float l = 0.0f, top = -INFINITY;
    for (int s0 = 0; s0 < plan.nseg; s0 += BATCH) {
        float2 x[BATCH];
        float4 v[BATCH];
#pragma unroll
        for (int i = 0; i < BATCH; ++i) {
            x[i] = make_float2(-INFINITY, 0.0f);
            v[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (s0 + i < plan.nseg) {
                x[i] = ml[(long long)(s0 + i) * a.nq];
                const float* p = src + (s0 + i) * row;
                if (quad) v[i] = *reinterpret_cast<const float4*>(p);
                else {
                    v[i].x = p[0];
                    if (e + 1 < a.dv) v[i].y = p[1];
                    if (e + 2 < a.dv) v[i].z = p[2];
                    if (e + 3 < a.dv) v[i].w = p[3];
                }
            }
        }
        float mn = top;
#pragma unroll
        for (int i = 0; i < BATCH; ++i) mn = fmaxf(mn, x[i].x);
        const float c = top == -INFINITY ? (l == 0.0f ? 0.0f : 1.0f) : expf(top - mn);
        o.x *= c; o.y *= c; o.z *= c; o.w *= c;
        l *= c;
        top = mn;
#pragma unroll
        for (int i = 0; i < BATCH; ++i) {
            if (x[i].x == -INFINITY && x[i].y == 0.0f) continue;      // no key of that segment is in the row's sight
            const float f = x[i].x == -INFINITY ? 1.0f : expf(x[i].x - mn);
            o.x = fmaf(f, v[i].x, o.x); o.y = fmaf(f, v[i].y, o.y); o.z = fmaf(f, v[i].z, o.z); o.w = fmaf(f, v[i].w, o.w);
            l = fmaf(f, x[i].y, l);
        }
    }
    const float inv = ta_close(top, l, a.sink, head);
    T* dst = (T*)a.out + ((size_t)n * a.nq + head) * a.dv + e;
    const float v[4] = {o.x * inv, o.y * inv, o.z * inv, o.w * inv};
    if (quad_out && sizeof(T) == 2) {
        *reinterpret_cast<uint2*>(dst) = make_uint2(ta_pack(v[0], v[1]), ta_pack(v[2], v[3]));
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (e + i < a.dv) dst[i] = from_f32<T>(v[i]);
}

template <typename T, int NC, bool ASYNC>
static cudaError_t ta_run(const TreeArgs& a, const int* tok_seq, int smem, int max_segs, cudaStream_t stream) {
    auto k = attn_tree_kernel<T, NC, ASYNC>;
    cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    const long long tiles = (long long)a.N * (a.nq / a.nkv) / TA_ROWS + a.B;
    e = lumen_launch(k, dim3((unsigned)(tiles * a.nkv), max_segs), dim3(TA_THREADS), smem, stream, a);
    if (e != cudaSuccess || max_segs == 1) return e;
    return lumen_launch(attn_tree_join_kernel<T>, dim3(a.N, ((a.dv + 3) / 4 * a.nq + 127) / 128), dim3(128), 0, stream, a, tok_seq);
}
template <typename T, int NC>
static cudaError_t ta_go(const TreeArgs& a, const int* tok_seq, int max_segs, cudaStream_t stream) {
    const int ks = ((a.d + 3) & ~3) + 4, vs = 128 * NC, fixed = TA_ROWS * ks + LUMEN_PAGE * TA_PROW;
    const int both = (fixed + LUMEN_PAGE * (ks + vs)) * (int)sizeof(float), one = (fixed + LUMEN_PAGE * (ks > vs ? ks : vs)) * (int)sizeof(float);
    if (sizeof(T) == 4 && NC < 4 && (a.vec & 3) == 3 && both <= 226 * 1024) return ta_run<T, NC, sizeof(T) == 4 && NC < 4>(a, tok_seq, both, max_segs, stream);
    return ta_run<T, NC, false>(a, tok_seq, one, max_segs, stream);
}

#include "attn_tree_mma.cuh"
#include "attn_tree_tc.cuh"

// Which kernel a call takes whose operands lie on 16 bytes and its output on 32: 1 the tensor cores' (positive: the scale is above 0).
LUMEN_API int lumen_attn_tree_tc(int is_bf16, int B, int N, int width, int nq, int nkv, int d, int dv, int layout, int v_layout,
                                 int positive) {
    return nkv > 0 && nq >= nkv && tt_takes(is_bf16, B, N, width, nq, nkv, d, dv, layout, v_layout, positive ? 1.0f : 0.0f) ? 1 : 0;
}
// Thousands (1,024s) of float32 numbers of scratch that a call needs, -1: more than there can be.
LUMEN_API int lumen_attn_tree_scratch(int tc, int B, int N, int width, int nq, int nkv, int d, int dv) {
    if (B <= 0 || N <= 0 || width < 1 || nkv < 1 || nq < nkv || d < 1 || dv < 1) return 0;
    const int G = nq / nkv;
    const long long n = tc ? tt_floats(tt_blocks(B, N, width, nq, nkv, d, dv), dv)
                           : tree_max_segs(width) == 1 ? 0 : tree_pairs(B, N, width, G) * nq * (dv + 2);
    return n > 1024LL * 2147483647LL ? -1 : (int)((n + 1023) / 1024);
}

// q [N, nq, d], out [N, nq, dv] in the cache's type; keys [n_pages, nkv, 64, d], values [n_pages, nkv, 64, dv]; mask
// [N, W] 64-bit words; tc and scratch (on 32 bytes) as the two functions above say.
LUMEN_API int lumen_attn_tree(const void* q, const void* kcache, const void* vcache, const int* block_table, int bt_stride,
                              int width, const int* cu_q, const int* seq_start, const int* tok_seq, const int* tok_pos,
                              const void* mask, int W, void* out, int tc, float* scratch, int scratch_k, int is_bf16, int B, int N,
                              int n_pages, int nq, int nkv, int d, int dv, int window, float scale, float softcap,
                              const float* sink, int layout, int v_layout, int* err, cudaStream_t stream) {
    if (B <= 0 || N <= 0) return 0;
    if (nq <= 0 || nkv <= 0 || nq % nkv || d <= 0 || d > 512 || dv <= 0 || dv > 512 || window < 0 || softcap < 0.0f || W < 1 ||
        width < 1 || width > (1 << 24) || n_pages < 1)
        return LUMEN_ERR_UNSUPPORTED;
    if ((layout == LUMEN_LAYOUT_SW128 && (!is_bf16 || d % 64)) || (v_layout == LUMEN_LAYOUT_SW128 && (!is_bf16 || dv % 64)))
        return LUMEN_ERR_UNSUPPORTED;
    const int G = nq / nkv, es = is_bf16 ? 2 : 4, max_segs = tree_max_segs(width);
    if ((long long)N * G > (1 << 30) || ((long long)N * G / TA_ROWS + B) * nkv > 2147483647LL || (long long)(dv + 3) / 4 * nq > 128LL * 65535) return LUMEN_ERR_UNSUPPORTED;
    const int need = lumen_attn_tree_scratch(tc, B, N, width, nq, nkv, d, dv);
    if (need < 0) return LUMEN_ERR_UNSUPPORTED;
    if ((tc && (!tt_takes(is_bf16, B, N, width, nq, nkv, d, dv, layout, v_layout, scale) || !tt_aligned(q, kcache, vcache, out))) || scratch_k < need ||
        (need && !scratch) || ((uintptr_t)scratch & 31))
        return LUMEN_ERR_BAD_ARGUMENT;
    const int vec = (((uintptr_t)kcache & 15) == 0 && d * es % 16 == 0 ? 1 : 0) | (((uintptr_t)vcache & 15) == 0 && dv * es % 16 == 0 ? 2 : 0) |
                    (((uintptr_t)q & 15) == 0 && d * es % 16 == 0 ? 4 : 0);
    // the maxima and sums first: the rows behind them lie on 16 bytes where dv is a multiple of 4
    const long long pairs = tree_pairs(B, N, width, G);
    TreeArgs a = {q, kcache, vcache, block_table, cu_q, seq_start, tok_pos, (const unsigned long long*)mask, out,
                        scratch ? scratch + pairs * nq * 2 : nullptr, (float2*)scratch, sink, bt_stride, width, W, B, N, n_pages, nq, nkv,
                        d, dv, window, layout, v_layout, vec, TREE_MIN_SEG, TREE_SEG_ROWS, scale, softcap};
    const bool mma = !tc && tm_takes(a, is_bf16);
    if (mma) { a.seg_min = TREE_MMA_MIN_SEG; a.seg_rows = TREE_MMA_SEG_ROWS; }
    cudaError_t e;
#define TA_GO(T) (dv <= 128 ? ta_go<T, 1>(a, tok_seq, max_segs, stream) : dv <= 256 ? ta_go<T, 2>(a, tok_seq, max_segs, stream) \
                                                                                   : ta_go<T, 4>(a, tok_seq, max_segs, stream))
    e = tc ? tt_launch(a, scratch, err, stream) : mma ? tm_go(a, tok_seq, max_segs, stream) : is_bf16 ? TA_GO(__nv_bfloat16) : TA_GO(float);
#undef TA_GO
    if (e != cudaSuccess) return (int)e;
    LUMEN_LAUNCH_CHECK();
    return 0;
}
