// Attention of new tokens over a pool of cache pages.
//
//     o_i = sum_j p_ij v_j,   p_ij = exp(scale q_i . k_j - m_i) / l_i,   j over the positions up to token i's own
//
// One pass over a sequence's K and V rows with a running maximum and sum.  The rows of a kv head serve all new tokens and all q heads of
// its group at once.  Work is dealt out as q3_paged_plan.h says; items that more than one block worked on are put together by
// paged_join_kernel, part by part in the order of their keys: no atomics, the same bits on every run.
#include <cfloat>

#include <cuda.h>
#include <cuda_fp16.h>

#include "q3_engine.h"
#include "q3_gemm_tc.h"
#include "q3_paged.h"
#include "q3_tc_ptx.cuh"

namespace q3 {

struct PagedAttnArgs {
    PagedView c;
    PgShape sh;
    int group;                       // q heads a kv head serves
    const unsigned char* q;
    unsigned char* out;
    long long q_token, q_head, o_token, o_head;      // bytes
    float scale;                     // times log2(e): scores are kept in units of log2
    float* part;                     // two partial results a block
    int least;                       // units a block takes at least
    uint32_t* status;
};

__device__ __forceinline__ float pg_ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// the two types of pages: packing, unpacking, products
struct PgBf16 {
    static constexpr bool BF = true;
    static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
        uint32_t d;
        asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
        return d;
    }
    static __device__ __forceinline__ float2 unpack(uint32_t u) { return make_float2(bf_lo(u), bf_hi(u)); }
    static __device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    }
};
struct PgFp16 {
    static constexpr bool BF = false;
    static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
        uint32_t d;
        asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
        return d;
    }
    static __device__ __forceinline__ float2 unpack(uint32_t u) { return __half22float2(*reinterpret_cast<const __half2*>(&u)); }
    static __device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    }
};

// What a segment is about: the keys [key0, key1) that its unit range holds, and per row of the tile (token row / group, q head row % group of the kv head's)
struct PgKeys { int key0, key1, qpos0, rows; };
__device__ __forceinline__ PgKeys pg_keys(const PagedAttnArgs& a, const PgSegment& s) {
    PgKeys k;
    const int tok0 = s.r * a.sh.tile, live = min(a.sh.tile, s.seq.q - tok0);
    k.qpos0 = s.seq.kv - s.seq.q + tok0;                       // position of the tile's first token (below 0: a token without a position)
    const int seen = max(0, min(s.seq.kv, k.qpos0 + live));
    k.key0 = min(s.k0 * a.sh.unit, seen);
    k.key1 = min((long long)s.k1 * a.sh.unit, (long long)seen);
    k.rows = live * a.group;
    return k;
}
__device__ __forceinline__ const unsigned char* pg_q_row(const PagedAttnArgs& a, const PgSegment& s, int row) {
    return a.q + (long long)(s.seq.q0 + s.r * a.sh.tile + row / a.group) * a.q_token + (long long)(s.h * a.group + row % a.group) * a.q_head;
}
__device__ __forceinline__ unsigned char* pg_o_row(const PagedAttnArgs& a, const PgSegment& s, int row) {
    return a.out + (long long)(s.seq.q0 + s.r * a.sh.tile + row / a.group) * a.o_token + (long long)(s.h * a.group + row % a.group) * a.o_head;
}

// A row again, key by key, reading only what it sees: for rows whose result is not finite.  A product adds 0 * v for keys that a row does not see
// beside those that its tile's later tokens see, and 0 * inf is no number.  Warps of the block take keys in turn (a lane four dims); leaves maximum, sum and
// output in res[0], res[1], res[4 ..].  `buf` holds 132 floats a warp.  Every thread of the block calls it; ends with a barrier.
template <typename T, int WARPS>
__device__ __noinline__ void pg_redo_row(const PagedAttnArgs& a, const PgSegment& s, const PgKeys& k, int row, float* buf, float* res, int threads_bar) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    auto sync = [&] { asm volatile("bar.sync %0, %1;" ::"r"(threads_bar), "n"(WARPS * 32) : "memory"); };
    const uint2 q2 = *reinterpret_cast<const uint2*>(pg_q_row(a, s, row) + lane * 8);
    const float2 qa = T::unpack(q2.x), qb = T::unpack(q2.y);
    const int end = min(k.key1, k.qpos0 + row / a.group + 1);
    float m = -INFINITY, l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
    for (int p = k.key0 + warp; p < end; p += WARPS) {
        const int page = pg_page(a.c, s.b, p);
        if (page < 0) continue;
        const long long at = pg_offset(a.c, page, p & ((1 << a.c.page_log) - 1), s.h) + lane * 8;
        const uint2 kk = *reinterpret_cast<const uint2*>(a.c.k + at), vv = *reinterpret_cast<const uint2*>(a.c.v + at);
        const float2 ka = T::unpack(kk.x), kb = T::unpack(kk.y), va = T::unpack(vv.x), vb = T::unpack(vv.y);
        const float x = warp_sum(qa.x * ka.x + qa.y * ka.y + qb.x * kb.x + qb.y * kb.y) * a.scale;
        if (x == -INFINITY) continue;
        const float top = x > m || x != x ? x : m, f = m == top ? 1.f : pg_ex2(m - top), e = pg_ex2(x - top);
        m = top;
        l = l * f + e;
        o[0] = o[0] * f + e * va.x; o[1] = o[1] * f + e * va.y; o[2] = o[2] * f + e * vb.x; o[3] = o[3] * f + e * vb.y;
    }
    sync();
    float* mine = buf + warp * 132;
    if (lane == 0) { mine[0] = m; mine[1] = l; }
#pragma unroll
    for (int i = 0; i < 4; ++i) mine[4 + lane * 4 + i] = o[i];
    sync();
    float top = -INFINITY;
    bool nan = false;
    for (int w = 0; w < WARPS; ++w) { top = fmaxf(top, buf[w * 132]); nan = nan || buf[w * 132] != buf[w * 132]; }
    if (nan) top = NAN;
    float sum = 0.f, v = 0.f;
    if (warp < 4) {
        for (int w = 0; w < WARPS; ++w) {
            const float mw = buf[w * 132];
            if (mw == -INFINITY) continue;
            const float f = mw == top ? 1.f : pg_ex2(mw - top);
            sum += buf[w * 132 + 1] * f;
            v += buf[w * 132 + 4 + threadIdx.x] * f;
        }
    }
    sync();
    if (warp < 4) {
        res[4 + threadIdx.x] = v;
        if (threadIdx.x == 0) { res[0] = top; res[1] = sum; }
    }
    sync();
}

// ------------------------------------------------------------------------------------------------------------------------------
// Few new tokens a sequence: NB blocks of eight columns hold the tile's rows (token, q head of the group), and the positions are the M dimension of
// mma.sync m16n8k16, as in q3_attn_mma.cu:
//     S^T [16 pos x 8 rows]  = K [16 pos x 128 dims]  Q^T          A = K by ldmatrix, B = Q in registers
//     O^T [128 dims x 8 rows] += V^T [128 dims x 16 pos]  P^T      A = V by ldmatrix.trans, B = P
// K and V rows stream through shared memory by cp.async (16 positions a stage, three stages a warp; 16 positions never leave a page), every
// fragment of them serves all NB blocks.
// ------------------------------------------------------------------------------------------------------------------------------
constexpr int PR_WARPS = 4, PR_THREADS = PR_WARPS * 32, PR_TILE = 16, PR_STAGES = 3, PR_HALF = PR_TILE * 256, PR_STAGE = 2 * PR_HALF;
constexpr int PR_UNIT = 64;                           // keys of a unit: a tile of 16 for every warp
constexpr size_t PR_SMEM = (size_t)PR_WARPS * PR_STAGES * PR_STAGE;
constexpr int PG_PART = 132;                          // floats of a row of a partial result: maximum, sum, two unused, output

__device__ __forceinline__ uint32_t pg_transpose(uint32_t w) {
    uint32_t d;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(w));
    return d;
}

template <typename T, int NB>
__global__ void __launch_bounds__(PR_THREADS, 2) paged_rows_kernel(const PagedAttnArgs a) {
    constexpr int COLS = 8 * NB, LD = 132;
    constexpr int PL = NB <= 2 ? 2 : 1;               // planes of P: two where the products have room beside the bytes
    static_assert(COLS * LD * 4 <= PR_STAGES * PR_STAGE, "a warp's outputs fit its stages");
    extern __shared__ __align__(128) unsigned char pr_raw[];
    __shared__ long long s_prefix[PG_MAX_BATCH + 1], s_sum[PR_WARPS];
    __shared__ float s_m[PR_WARPS][COLS], s_l[PR_WARPS][COLS];
    __shared__ unsigned s_bad;
    __shared__ float s_res[132];
    const int tid = threadIdx.x, lane = tid & 31, warp = uniform_warp();
    const int fg = lane >> 2, ft = lane & 3, lrow = lane & 7, lmat = lane >> 3;
    pdl_launch();
    pdl_wait();
    if (tid == 0) s_bad = 0;
    pg_block_prefix<PR_THREADS>(a.sh, a.c.q_start, a.c.kv_len, s_prefix, s_sum);
    const long long total = s_prefix[a.sh.batch];
    const int blocks = pg_blocks(total, (int)gridDim.x, a.least);
    if ((int)blockIdx.x >= blocks) return;
    PgWalk walk;
    if (!walk.begin(a.sh, s_prefix, a.c.q_start, a.c.kv_len, pg_run_start(total, blocks, blockIdx.x), pg_run_start(total, blocks, blockIdx.x + 1))) return;
    unsigned char* const stage0 = pr_raw + (size_t)warp * PR_STAGES * PR_STAGE;
    float* const s_o = reinterpret_cast<float*>(stage0);
    const int page_mask = (1 << a.c.page_log) - 1;

    bool first = true;
    do {
        const PgSegment& s = walk.s;
        const PgKeys k = pg_keys(a, s);
        const int n_pos = k.key1 - k.key0, per = (n_pos + PR_WARPS * PR_TILE - 1) / (PR_WARPS * PR_TILE) * PR_TILE;
        const int w0 = k.key0 + warp * per, w1 = min(w0 + per, k.key1);
        const int n_tiles = w1 > w0 ? (w1 - w0 + PR_TILE - 1) / PR_TILE : 0;

        // pages of 32 tiles at a time, a lane each; hist: whether the page of the last tiles that were asked for is there
        int pages = -1;
        unsigned hist = 0;
        auto issue = [&](int i) {
            if ((i & 31) == 0) {
                const int p = w0 + (i + lane) * PR_TILE;
                pages = p < w1 ? pg_page(a.c, s.b, p) : -1;
            }
            const int page = __shfl_sync(0xffffffffu, pages, i & 31);
            hist = hist << 1 | (page >= 0 ? 1u : 0u);
            if (i < n_tiles) {
                const uint32_t st = tc_smem(stage0 + (size_t)(i % PR_STAGES) * PR_STAGE);
                const int p0 = w0 + i * PR_TILE, count = page >= 0 ? min(PR_TILE, w1 - p0) : 0;      // rows past the run, and of no page, are zeros
                const long long base = pg_offset(a.c, max(page, 0), p0 & page_mask, s.h) + (lane & 15) * 16;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const int row = j * 2 + (lane >> 4), c = lane & 15;
                    const uint32_t bytes = row < count ? 16u : 0u;
                    const long long src = base + (row < count ? (long long)row * a.c.slot_bytes : 0);
                    const uint32_t dst = st + (uint32_t)(row * 256 + ((c ^ (row & 7)) << 4));
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(a.c.k + src), "r"(bytes) : "memory");
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst + PR_HALF), "l"(a.c.v + src), "r"(bytes) : "memory");
                }
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
#pragma unroll
        for (int i = 0; i < PR_STAGES - 1; ++i) issue(i);

        // Q^T as the B operand: column fg of block nb is row 8 nb + fg of the tile
        uint32_t q[NB][8][2];
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
            const int row = 8 * nb + fg;
            const unsigned char* src = pg_q_row(a, s, min(row, k.rows - 1)) + ft * 4;
#pragma unroll
            for (int ks = 0; ks < 8; ++ks)
#pragma unroll
                for (int h = 0; h < 2; ++h) q[nb][ks][h] = row < k.rows ? *reinterpret_cast<const uint32_t*>(src + ks * 32 + h * 16) : 0u;
        }
        float o[NB][8][4], m[NB][2], l[NB][2];
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
            m[nb][0] = m[nb][1] = -INFINITY; l[nb][0] = l[nb][1] = 0.f;
#pragma unroll
            for (int mt = 0; mt < 8; ++mt) o[nb][mt][0] = o[nb][mt][1] = o[nb][mt][2] = o[nb][mt][3] = 0.f;
        }
        for (int i = 0; i < n_tiles; ++i) {
            issue(i + PR_STAGES - 1);
            asm volatile("cp.async.wait_group %0;" ::"n"(PR_STAGES - 1) : "memory");
            __syncwarp();
            const uint32_t kst = tc_smem(stage0 + (size_t)(i % PR_STAGES) * PR_STAGE), vst = kst + PR_HALF;
            const bool there = (hist >> (PR_STAGES - 1)) & 1u;
            float c[NB][4];
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) c[nb][0] = c[nb][1] = c[nb][2] = c[nb][3] = 0.f;
            {
                const int row = lrow + (lmat & 1) * 8;
#pragma unroll
                for (int ks = 0; ks < 8; ++ks) {
                    uint32_t af[4];
                    const uint32_t addr = kst + (uint32_t)(row * 256 + (((2 * ks + (lmat >> 1)) ^ (row & 7)) << 4));
                    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(af[0]), "=r"(af[1]), "=r"(af[2]), "=r"(af[3]) : "r"(addr) : "memory");
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb) T::mma(c[nb], af, q[nb][ks][0], q[nb][ks][1]);
                }
            }
            // c[nb][0], [1]: position fg, rows 2 ft, 2 ft + 1 of block nb; [2], [3]: position fg + 8
            const int p0 = w0 + i * PR_TILE, pa = p0 + fg;
            const bool all = there && p0 + PR_TILE <= w1 && p0 + PR_TILE - 1 <= k.qpos0;      // every row sees every position of the tile
            uint32_t b0[NB][PL], b1[NB][PL];
            float f[NB][2];
            bool moved = false;
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float sa = c[nb][e] * a.scale, sb = c[nb][2 + e] * a.scale;
                    if (!all) {
                        const int last = there ? min(w1 - 1, k.qpos0 + (8 * nb + 2 * ft + e) / a.group) : -1;
                        if (pa > last) sa = -INFINITY;
                        if (pa + 8 > last) sb = -INFINITY;
                    }
                    float t = fmaxf(sa, sb);
#pragma unroll
                    for (int sh = 4; sh <= 16; sh <<= 1) t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, sh));
                    const float n = fmaxf(m[nb][e], t), ms = n == -INFINITY ? 0.f : n;
                    f[nb][e] = pg_ex2(m[nb][e] - ms);
                    moved = moved || m[nb][e] != n;
                    m[nb][e] = n;
                    c[nb][e] = pg_ex2(sa - ms);
                    c[nb][2 + e] = pg_ex2(sb - ms);
                    l[nb][e] = fmaf(l[nb][e], f[nb][e], c[nb][e] + c[nb][2 + e]);
                }
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) {
                float xa0 = c[nb][0], xa1 = c[nb][1], xb0 = c[nb][2], xb1 = c[nb][3];
#pragma unroll
                for (int j = 0; j < PL; ++j) {
                    const uint32_t pa2 = T::pack(xa0, xa1), pb2 = T::pack(xb0, xb1);
                    if (j + 1 < PL) {
                        const float2 ra = T::unpack(pa2), rb = T::unpack(pb2);
                        xa0 -= ra.x; xa1 -= ra.y; xb0 -= rb.x; xb1 -= rb.y;
                    }
                    b0[nb][j] = pg_transpose(pa2); b1[nb][j] = pg_transpose(pb2);
                }
            }
            if (__any_sync(0xffffffffu, moved))
#pragma unroll
                for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                    for (int mt = 0; mt < 8; ++mt) { o[nb][mt][0] *= f[nb][0]; o[nb][mt][1] *= f[nb][1]; o[nb][mt][2] *= f[nb][0]; o[nb][mt][3] *= f[nb][1]; }
            {
                const int row = lrow + (lmat >> 1) * 8;
#pragma unroll
                for (int mt = 0; mt < 8; ++mt) {
                    uint32_t af[4];
                    const uint32_t addr = vst + (uint32_t)(row * 256 + (((2 * mt + (lmat & 1)) ^ (row & 7)) << 4));
                    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(af[0]), "=r"(af[1]), "=r"(af[2]), "=r"(af[3]) : "r"(addr) : "memory");
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                        for (int j = 0; j < PL; ++j) T::mma(o[nb][mt], af, b0[nb][j], b1[nb][j]);
                }
            }
            __syncwarp();                                            // the stage is refilled by the next iteration's copies
        }
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        __syncwarp();
        // the warp's maxima, sums and outputs; its own stages hold them
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
#pragma unroll
                for (int sh = 4; sh <= 16; sh <<= 1) l[nb][e] += __shfl_xor_sync(0xffffffffu, l[nb][e], sh);
                const int col = 8 * nb + 2 * ft + e;
                if (fg == 0) { s_m[warp][col] = m[nb][e]; s_l[warp][col] = l[nb][e]; }
#pragma unroll
                for (int mt = 0; mt < 8; ++mt) { s_o[col * LD + mt * 16 + fg] = o[nb][mt][e]; s_o[col * LD + mt * 16 + fg + 8] = o[nb][mt][2 + e]; }
            }
        __syncthreads();
        const bool whole = walk.whole();
        float* const part = a.part + (size_t)(2 * blockIdx.x + (first ? 0 : 1)) * COLS * PG_PART;
        auto store = [&](int row, float M, float L, float v) {       // dim tid of a row
            if (whole) {
                const float r = L > 0.f || L != L ? v / L : 0.f;      // (nothing seen, or nothing with a weight: zeros)
                const float up = __shfl_down_sync(0xffffffffu, r, 1);
                if (!(tid & 1)) *reinterpret_cast<uint32_t*>(pg_o_row(a, s, row) + tid * 2) = T::pack(r, up);
            } else {
                part[row * PG_PART + 4 + tid] = v;
                if (tid == 0) { part[row * PG_PART] = M; part[row * PG_PART + 1] = L; }
            }
        };
        for (int row = 0; row < k.rows && row < COLS; ++row) {
            float M = s_m[0][row];
#pragma unroll
            for (int w = 1; w < PR_WARPS; ++w) M = fmaxf(M, s_m[w][row]);
            const float Ms = M == -INFINITY ? 0.f : M;
            float L = 0.f, v = 0.f;
#pragma unroll
            for (int w = 0; w < PR_WARPS; ++w) {
                const float wgt = pg_ex2(s_m[w][row] - Ms);
                L = fmaf(s_l[w][row], wgt, L);
                v = fmaf(*reinterpret_cast<const float*>(pr_raw + (size_t)w * PR_STAGES * PR_STAGE + (size_t)(row * LD + tid) * 4), wgt, v);
            }
            store(row, M, L, v);
            if (!(fabsf(v) <= FLT_MAX && L <= FLT_MAX)) atomicOr(&s_bad, 1u << row);
        }
        __syncthreads();
        for (unsigned bad = s_bad; bad; bad &= bad - 1) {
            const int row = __ffs(bad) - 1;
            pg_redo_row<T, PR_WARPS>(a, s, k, row, reinterpret_cast<float*>(pr_raw), s_res, 0);
            store(row, s_res[0], s_res[1], s_res[4 + tid]);
        }
        __syncthreads();
        if (tid == 0) s_bad = 0;
        first = false;
    } while (walk.next(a.sh, a.c.q_start, a.c.kv_len));
}

// ------------------------------------------------------------------------------------------------------------------------------
// Items that were cut: a block per cut, the one at an item's first cut puts the item together.  A warp a row, a lane four dims.
// ------------------------------------------------------------------------------------------------------------------------------
constexpr int PJ_THREADS = 128;

template <typename T>
__global__ void __launch_bounds__(PJ_THREADS) paged_join_kernel(const PagedAttnArgs a, int grid, int part_rows) {
    __shared__ long long s_prefix[PG_MAX_BATCH + 1], s_sum[PJ_THREADS / 32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    pdl_launch();
    pdl_wait();
    pg_block_prefix<PJ_THREADS>(a.sh, a.c.q_start, a.c.kv_len, s_prefix, s_sum);
    const long long total = s_prefix[a.sh.batch];
    const int blocks = pg_blocks(total, grid, a.least), cut = (int)blockIdx.x + 1;
    if (cut >= blocks) return;
    const long long at = pg_run_start(total, blocks, cut);
    PgWalk walk;
    if (!walk.begin(a.sh, s_prefix, a.c.q_start, a.c.kv_len, at, at + 1)) return;
    const PgSegment& s = walk.s;
    const long long from = at - s.k0, to = from + s.units, before = pg_run_start(total, blocks, cut - 1);
    if (s.k0 == 0 || before > from) return;            // no item is cut here, or this is not its first cut
    const int live = min(a.sh.tile, s.seq.q - s.r * a.sh.tile) * a.group;
    int parts = 1;
    while (cut + parts - 1 < blocks && pg_run_start(total, blocks, cut + parts - 1) < to) ++parts;      // blocks cut - 1 .. cut + parts - 2
    const size_t slot0 = (size_t)2 * (cut - 1) + (before == from ? 0 : 1);
    auto part = [&](int i, int row) { return a.part + ((i == 0 ? slot0 : (size_t)2 * (cut - 1 + i)) * part_rows + row) * PG_PART; };
    for (int row = blockIdx.y * (PJ_THREADS / 32) + warp; row < live; row += gridDim.y * (PJ_THREADS / 32)) {
        float M = -INFINITY;
        bool nan = false;
        for (int i = lane; i < parts; i += 32) { const float x = part(i, row)[0]; M = fmaxf(M, x); nan = nan || x != x; }
        M = warp_max(M);
        if (__any_sync(0xffffffffu, nan)) M = NAN;
        const float Ms = M == -INFINITY ? 0.f : M;
        float L = 0.f;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int i0 = 0; i0 < parts; i0 += 32) {
            float w = 0.f, lw = 0.f;
            if (i0 + lane < parts) {
                const float2 ml = *reinterpret_cast<const float2*>(part(i0 + lane, row));
                w = ml.x == -INFINITY ? 0.f : ml.x == Ms ? 1.f : pg_ex2(ml.x - Ms);
                lw = ml.x == -INFINITY ? 0.f : ml.y * w;
            }
            const int n = min(32, parts - i0);
#pragma unroll 4
            for (int i = 0; i < n; ++i) {
                const float wi = __shfl_sync(0xffffffffu, w, i);
                L += __shfl_sync(0xffffffffu, lw, i);
                const float4 x = *reinterpret_cast<const float4*>(part(i0 + i, row) + 4 + lane * 4);
                if (wi != 0.f) { v.x = fmaf(x.x, wi, v.x); v.y = fmaf(x.y, wi, v.y); v.z = fmaf(x.z, wi, v.z); v.w = fmaf(x.w, wi, v.w); }
            }
        }
        const float r = L > 0.f || L != L ? 1.f / L : 0.f;
        *reinterpret_cast<uint2*>(pg_o_row(a, s, row) + lane * 8) = make_uint2(T::pack(v.x * r, v.y * r), T::pack(v.z * r, v.w * r));
    }
}

// ------------------------------------------------------------------------------------------------------------------------------
static int pg_blocks_of_device() { return 2 * tc_sm_count(); }

template <typename T, int NB>
static cudaError_t launch_rows(const PagedAttnArgs& a, int grid, cudaStream_t st) {
    cudaError_t e = cudaFuncSetAttribute(paged_rows_kernel<T, NB>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)PR_SMEM);
    if (e == cudaSuccess) e = launch_chain(paged_rows_kernel<T, NB>, dim3(grid), dim3(PR_THREADS), PR_SMEM, st, a);
    if (e == cudaSuccess && grid > 1) e = launch_chain(paged_join_kernel<T>, dim3(grid - 1, 2 * NB), dim3(PJ_THREADS), 0, st, a, grid, 8 * NB);
    return e;
}

template <typename T>
static cudaError_t launch_attn(PagedAttnArgs& a, int max_new, cudaStream_t st) {
    const int cols = max_new > 32 / a.group ? 32 : max_new * a.group, nb = cols <= 8 ? 1 : cols <= 16 ? 2 : 4;
    a.sh.unit = PR_UNIT;
    a.sh.tile = 8 * nb / a.group;
    a.least = 1;
    const int grid = pg_blocks_of_device();
    return nb == 1 ? launch_rows<T, 1>(a, grid, st) : nb == 2 ? launch_rows<T, 2>(a, grid, st) : launch_rows<T, 4>(a, grid, st);
}

int paged_check(const char* who, const q3_paged* c) {
    auto bad = [&](const char* what) { return engine_fail(nullptr, Q3_ERR_INVALID, "%s: %s", who, what); };
    if (!c) return bad("null argument");
    if (!c->k_pages || !c->v_pages || !c->page_table || !c->q_start || !c->kv_len) return bad("k_pages, v_pages, page_table, q_start and kv_len are required");
    if (c->page_size < 16 || c->page_size > 256 || (c->page_size & (c->page_size - 1))) return bad("page_size must be 16, 32, 64, 128 or 256");
    if (c->batch < 1 || c->batch > Q3_PAGED_MAX_BATCH) return engine_fail(nullptr, Q3_ERR_INVALID, "%s: batch %d outside 1..%d", who, c->batch, Q3_PAGED_MAX_BATCH);
    if (c->n_pages < 1 || c->table_pages < 1 || c->table_stride < c->table_pages || c->n_tokens < 0 || c->max_new < 0 || c->kv_heads < 1 || c->kv_heads > 1024)
        return engine_fail(nullptr, Q3_ERR_INVALID, "%s: n_pages=%d table_pages=%d (row stride %lld) n_tokens=%d max_new=%d kv_heads=%d out of range", who, c->n_pages, c->table_pages,
                           (long long)c->table_stride, c->n_tokens, c->max_new, c->kv_heads);
    if ((int64_t)c->table_pages * c->page_size > 0x7fffff00ll) return bad("a row of the page table holds more than 2^31 - 256 positions");
    if (c->type != Q3_TYPE_BF16 && c->type != Q3_TYPE_FP16) return bad("pages are bf16 or fp16");
    if ((reinterpret_cast<uintptr_t>(c->k_pages) | reinterpret_cast<uintptr_t>(c->v_pages)) & 15) return bad("pages must be 16-byte aligned");
    const int64_t most = 1ll << 38;
    for (int64_t s : {c->page_stride, c->slot_stride, c->head_stride})
        if (s < 0 || s > most || s % 8) return bad("strides of the pages must be multiples of 8 elements, not negative");
    if ((reinterpret_cast<uintptr_t>(c->page_table) | reinterpret_cast<uintptr_t>(c->q_start) | reinterpret_cast<uintptr_t>(c->kv_len)) & 3)
        return bad("page_table, q_start and kv_len must be 4-byte aligned");
    return Q3_OK;
}

PagedView paged_view(const q3_paged* c) {
    PagedView v{};
    v.k = static_cast<unsigned char*>(c->k_pages);
    v.v = static_cast<unsigned char*>(c->v_pages);
    v.page_bytes = 2 * c->page_stride; v.slot_bytes = 2 * c->slot_stride; v.head_bytes = 2 * c->head_stride;
    v.table = c->page_table; v.q_start = c->q_start; v.kv_len = c->kv_len;
    v.table_stride = c->table_stride;
    v.n_pages = c->n_pages;
    for (v.page_log = 4; (1 << v.page_log) < c->page_size; ++v.page_log) {}
    return v;
}

}  // namespace q3

using namespace q3;

// two partial results a block: at most 32 rows for every one of two blocks an SM
extern "C" int64_t q3_paged_attn_workspace(const q3_paged* c, int32_t q_heads) {
    if (!c || q_heads < 1) return engine_fail(nullptr, Q3_ERR_INVALID, "q3_paged_attn_workspace: bad argument");
    const int sms = tc_sm_count();
    if (sms < 1) return engine_fail(nullptr, Q3_ERR_CUDA, "q3_paged_attn_workspace: no CUDA device");
    return (int64_t)2 * pg_blocks_of_device() * 32 * PG_PART * 4;
}

extern "C" int q3_paged_attn(const q3_paged* c, const q3_paged_attn_args* p, void* stream) {
    const char* who = "q3_paged_attn";
    if (const int rc = paged_check(who, c)) return rc;
    auto bad = [&](const char* what) { return engine_fail(nullptr, Q3_ERR_INVALID, "%s: %s", who, what); };
    if (!p) return bad("null argument");
    if (c->n_tokens == 0) return Q3_OK;
    if (!p->q || !p->out || !p->workspace) return bad("q, out and workspace are required");
    const int group = p->q_heads / c->kv_heads;
    if (p->q_heads < 1 || p->q_heads % c->kv_heads || (group != 1 && group != 2 && group != 4 && group != 8))
        return engine_fail(nullptr, Q3_ERR_INVALID, "%s: %d q heads over %d kv heads: a kv head serves 1, 2, 4 or 8", who, p->q_heads, c->kv_heads);
    if (!(p->scale > 0.f) || p->scale > 1e30f) return bad("scale must be positive and at most 1e30");
    if ((reinterpret_cast<uintptr_t>(p->q) | reinterpret_cast<uintptr_t>(p->out) | reinterpret_cast<uintptr_t>(p->workspace)) & 15) return bad("q, out and workspace must be 16-byte aligned");
    const int64_t most = 1ll << 38;
    for (int64_t s : {p->q_token, p->q_head, p->out_token, p->out_head})
        if (s < 0 || s > most || s % 8) return bad("strides of q and out must be multiples of 8 elements, not negative");
    const int64_t need = q3_paged_attn_workspace(c, p->q_heads);
    if (need < 0) return (int)need;
    if (p->workspace_bytes < need) return engine_fail(nullptr, Q3_ERR_INVALID, "%s: workspace holds %lld bytes, %lld needed", who, (long long)p->workspace_bytes, (long long)need);
    PagedAttnArgs a{};
    a.c = paged_view(c);
    a.sh.heads = c->kv_heads; a.sh.batch = c->batch; a.sh.n_tokens = c->n_tokens; a.sh.most_keys = c->table_pages * c->page_size;
    a.group = group;
    a.q = static_cast<const unsigned char*>(p->q);
    a.out = static_cast<unsigned char*>(p->out);
    a.q_token = 2 * p->q_token; a.q_head = 2 * p->q_head; a.o_token = 2 * p->out_token; a.o_head = 2 * p->out_head;
    a.scale = p->scale * 1.4426950408889634f;
    a.part = static_cast<float*>(p->workspace);
    a.status = p->status;
    cudaStream_t st = (cudaStream_t)stream;
    const int max_new = c->max_new < 1 ? 1 : c->max_new;
    const cudaError_t err = c->type == Q3_TYPE_BF16 ? launch_attn<PgBf16>(a, max_new, st) : launch_attn<PgFp16>(a, max_new, st);
    if (err != cudaSuccess) return engine_fail(nullptr, Q3_ERR_CUDA, "%s: %s", who, cudaGetErrorString(err));
    return Q3_OK;
}
