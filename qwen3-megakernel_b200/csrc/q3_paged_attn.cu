// Attention of new tokens over a pool of cache pages.
//
//     o_i = sum_j p_ij v_j,   p_ij = exp(scale q_i . k_j - m_i) / l_i,   j over the positions up to token i's own
//
// One pass over a sequence's K and V rows with a running maximum and sum.  The rows of a kv head serve all new tokens and all q heads of
// its group at once.  Work is dealt out as q3_paged_plan.h says; items that more than one block worked on are put together by
// paged_join_kernel, part by part in the order of their keys: no atomics, the same bits on every run.
#include <cfloat>

#include <cuda.h>
#include <cudaTypedefs.h>
#include <cuda_fp16.h>

#include "q3_engine.h"
#include "q3_gemm_tc.h"
#include "q3_paged.h"
#include "q3_rows_meet.h"
#include "q3_tc_ptx.cuh"

namespace q3 {

struct PagedAttnArgs {
    PagedView c;
    PgShape sh;
    int group_log;                   // a kv head serves 2^group_log q heads
    const unsigned char* q;
    unsigned char* out;
    long long q_token, q_head, o_token, o_head;      // bytes
    float scale;                     // times log2(e): scores are kept in units of log2
    struct PgCut* cuts;              // one a block
    float* part;                     // two partial results a block
    int least;                       // units a block takes at least
    uint32_t* status;
    unsigned long long wait_ns;      // how long a wait of the tile kernel lasts at most,
    unsigned wait_looks;             // and at which looks at the barrier it asks for the time (a mask of their number)
};

// What a block leaves behind: the item that is cut at its end and began in its run, to be put together of the results of `parts` blocks (0: none)
struct PgCut { int parts, slot, b, h, r, unused[3]; };

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
__device__ __forceinline__ void pg_leave_cut(const PagedAttnArgs& a, const PgWalk& w, bool first, long long total, int blocks) {      // one thread, for a run's last segment
    const PgSegment& s = w.s;
    const bool begins = !w.whole() && s.k0 == 0;
    a.cuts[blockIdx.x] = PgCut{begins ? pg_runs_before(total, blocks, w.at + s.units) - (int)blockIdx.x : 0, first ? 0 : 1, s.b, s.h, s.r, {0, 0, 0}};
}
struct PgKeys { int key0, key1, qpos0, rows; };
__device__ __forceinline__ PgKeys pg_keys(const PagedAttnArgs& a, const PgSegment& s) {
    PgKeys k;
    const int tok0 = s.r << a.sh.tile_log, live = min(1 << a.sh.tile_log, s.seq.q - tok0);
    k.qpos0 = s.seq.kv - s.seq.q + tok0;                       // position of the tile's first token (below 0: a token without a position)
    const int seen = max(0, min(s.seq.kv, k.qpos0 + live));
    k.key0 = (int)min((long long)s.k0 << a.sh.unit_log, (long long)seen);
    k.key1 = (int)min((long long)s.k1 << a.sh.unit_log, (long long)seen);
    k.rows = live << a.group_log;
    return k;
}
__device__ __forceinline__ const unsigned char* pg_q_row(const PagedAttnArgs& a, const PgSegment& s, int row) {
    return a.q + (long long)(s.seq.q0 + (s.r << a.sh.tile_log) + (row >> a.group_log)) * a.q_token + (long long)((s.h << a.group_log) + (row & ((1 << a.group_log) - 1))) * a.q_head;
}
__device__ __forceinline__ unsigned char* pg_o_row(const PagedAttnArgs& a, const PgSegment& s, int row) {
    return a.out + (long long)(s.seq.q0 + (s.r << a.sh.tile_log) + (row >> a.group_log)) * a.o_token + (long long)((s.h << a.group_log) + (row & ((1 << a.group_log) - 1))) * a.o_head;
}

__device__ __forceinline__ float pg_max_nan(float a, float b) {      // NaN if either is
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
}
// Rows again, key by key, each reading only what it sees: for rows whose result is not finite.  A product adds 0 * v for keys that a row does not see
// beside those that its tile's later tokens see, and 0 * inf is no number.  PG_REDO rows of a tile at once (row[i] < 0: none), for which a key is fetched once; the
// warps of the block take keys in turn (a lane four dims).  Leaves a row's maximum, sum and output in res[0], res[1], res[4 ..] of its PG_PART floats.  `buf` holds
// PG_REDO * PG_PART floats a warp.  Every thread of WARPS warps calls it, `warp` is its place among them; `sync` is their barrier, and the last thing done.
constexpr int PG_PART = 132;                          // floats of a row of a partial result: maximum, sum, two unused, output
constexpr int PG_REDO = 4;
template <typename T, int WARPS, typename Sync>
__device__ __noinline__ void pg_redo_rows(const PagedAttnArgs& a, const PgSegment& s, const PgKeys& k, int4 which, int warp, float* buf, float* res, const Sync& sync) {
    constexpr int R = PG_REDO, AHEAD = 4;            // keys of a warp whose loads are under way
    static_assert(AHEAD * R == 16 && R == 4, "a pair of lanes a (key, row)");
    const int lane = threadIdx.x & 31, tid = warp * 32 + lane;
    const int row[R] = {which.x, which.y, which.z, which.w};
    float2 qa[R], qb[R];
    float o[R][4];
    int end[R], stop = k.key0;
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const uint2 q2 = *reinterpret_cast<const uint2*>(pg_q_row(a, s, max(row[r], 0)) + lane * 8);
        qa[r] = T::unpack(q2.x); qb[r] = T::unpack(q2.y);
        end[r] = row[r] < 0 ? k.key0 : min(k.key1, k.qpos0 + (row[r] >> a.group_log) + 1);
        stop = max(stop, end[r]);
        o[r][0] = o[r][1] = o[r][2] = o[r][3] = 0.f;
    }
    // lanes 2 j and 2 j + 1 stand for key j / R of the batch and row j % R: they hold that row's maximum and sum
    const int my_key = lane >> 3, my_row = (lane >> 1) & 3, my_end = my_row == 0 ? end[0] : my_row == 1 ? end[1] : my_row == 2 ? end[2] : end[3];
    float m = -INFINITY, l = 0.f;
    for (long long p0 = k.key0 + warp; p0 < stop; p0 += AHEAD * WARPS) {
        int page[AHEAD];
        uint2 kk[AHEAD], vv[AHEAD];
        float x[AHEAD * R];
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) page[i] = p0 + i * WARPS < stop ? pg_page(a.c, s.b, (int)p0 + i * WARPS) : -1;
        if (max(max(page[0], page[1]), max(page[2], page[3])) < 0) continue;
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            kk[i] = vv[i] = make_uint2(0u, 0u);
            if (page[i] < 0) continue;
            const long long at = pg_offset(a.c, page[i], ((int)p0 + i * WARPS) & ((1 << a.c.page_log) - 1), s.h) + lane * 8;
            kk[i] = *reinterpret_cast<const uint2*>(a.c.k + at); vv[i] = *reinterpret_cast<const uint2*>(a.c.v + at);
        }
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            const float2 ka = T::unpack(kk[i].x), kb = T::unpack(kk[i].y);
#pragma unroll
            for (int r = 0; r < R; ++r) x[i * R + r] = qa[r].x * ka.x + qa[r].y * ka.y + qb[r].x * kb.x + qb[r].y * kb.y;
        }
        // sixteen sums over the warp: each step halves what a lane holds
#pragma unroll
        for (int half = 8; half > 0; half >>= 1) {
            const bool upper = lane & (2 * half);
#pragma unroll
            for (int j = 0; j < half; ++j) {
                const float other = __shfl_xor_sync(0xffffffffu, upper ? x[j] : x[j + half], 2 * half);
                x[j] = (upper ? x[j + half] : x[j]) + other;
            }
        }
        float y = (x[0] + __shfl_xor_sync(0xffffffffu, x[0], 1)) * a.scale;
        const int my_page = my_key == 0 ? page[0] : my_key == 1 ? page[1] : my_key == 2 ? page[2] : page[3];
        if (my_page < 0 || p0 + my_key * WARPS >= my_end) y = -INFINITY;
        const unsigned seen = __ballot_sync(0xffffffffu, y != -INFINITY);
        float top = pg_max_nan(m, y);
        top = pg_max_nan(top, __shfl_xor_sync(0xffffffffu, top, 8));
        top = pg_max_nan(top, __shfl_xor_sync(0xffffffffu, top, 16));
        const float ref = top == -INFINITY ? 0.f : top, f = m == top ? 1.f : pg_ex2(m - ref), e = pg_ex2(y - ref);
        const bool moved = __any_sync(0xffffffffu, m != top);
        m = top;
        float sum = e;
        sum += __shfl_xor_sync(0xffffffffu, sum, 8);
        sum += __shfl_xor_sync(0xffffffffu, sum, 16);
        l = l * f + sum;
        if (moved)
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const float fr = __shfl_sync(0xffffffffu, f, 2 * r);
#pragma unroll
                for (int d = 0; d < 4; ++d) o[r][d] *= fr;
            }
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            const float2 va = T::unpack(vv[i].x), vb = T::unpack(vv[i].y);
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const int from = 2 * (i * R + r);
                const float w = __shfl_sync(0xffffffffu, e, from);
                if ((seen >> from) & 1u) { o[r][0] += w * va.x; o[r][1] += w * va.y; o[r][2] += w * vb.x; o[r][3] += w * vb.y; }
            }
        }
    }
    sync();
#pragma unroll
    for (int r = 0; r < R; ++r) {
        float* mine = buf + (warp * R + r) * PG_PART;
        if (lane == 2 * r) { mine[0] = m; mine[1] = l; }
#pragma unroll
        for (int i = 0; i < 4; ++i) mine[4 + lane * 4 + i] = o[r][i];
    }
    sync();
    if (warp < 4)
        for (int r = 0; r < R; ++r) {
            const float* const all = buf + r * PG_PART;
            float top = -INFINITY;
            bool nan = false;
            for (int w = 0; w < WARPS; ++w) { const float mw = all[w * R * PG_PART]; top = fmaxf(top, mw); nan = nan || mw != mw; }
            if (nan) top = NAN;
            float sum = 0.f, v = 0.f;
            for (int w = 0; w < WARPS; ++w) {
                const float mw = all[w * R * PG_PART];
                if (mw == -INFINITY) continue;
                const float f = mw == top ? 1.f : pg_ex2(mw - top);
                sum += all[w * R * PG_PART + 1] * f;
                v += all[w * R * PG_PART + 4 + tid] * f;
            }
            res[r * PG_PART + 4 + tid] = v;
            if (tid == 0) { res[r * PG_PART] = top; res[r * PG_PART + 1] = sum; }
        }
    sync();
}
// the next rows of a set that are done again together; they leave it
__device__ __forceinline__ int4 pg_take_rows(unsigned& set, int first) {
    int r[PG_REDO];
#pragma unroll
    for (int i = 0; i < PG_REDO; ++i) { r[i] = set ? first + __ffs(set) - 1 : -1; set &= set - 1; }
    return make_int4(r[0], r[1], r[2], r[3]);
}

// ------------------------------------------------------------------------------------------------------------------------------
// Few new tokens a sequence: NB blocks of eight columns hold the tile's rows (token, q head of the group), and the positions are the M dimension of
// mma.sync m16n8k16, as in q3_attn_mma.cu:
//     S^T [16 pos x 8 rows]  = K [16 pos x 128 dims]  Q^T          A = K by ldmatrix, B = Q in registers
//     O^T [128 dims x 8 rows] += V^T [128 dims x 16 pos]  P^T      A = V by ldmatrix.trans, B = P
// K and V rows stream through shared memory by cp.async (16 positions a stage, three stages a warp; 16 positions never leave a page), every
// fragment of them serves all NB blocks.  Bound by the pages' bytes: 64 sequences with a new token behind up to 2048 read 336 MB in 62 us with start and join, 5.4 TB/s of the 6.5
// that a copy reaches (one token behind 1000: 8 us, three dependent loads, a page's way and the join).
// ------------------------------------------------------------------------------------------------------------------------------
constexpr int PR_WARPS = 4, PR_THREADS = PR_WARPS * 32, PR_TILE = 16, PR_STAGES = 3, PR_HALF = PR_TILE * 256, PR_STAGE = 2 * PR_HALF;
constexpr int PR_UNIT_LOG = 6;                        // 64 keys a unit: a tile of 16 for every warp
constexpr size_t PR_SMEM = (size_t)PR_WARPS * PR_STAGES * PR_STAGE;

__device__ __forceinline__ uint32_t pg_transpose(uint32_t w) {
    uint32_t d;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(w));
    return d;
}

template <typename T, int NB>
__global__ void __launch_bounds__(PR_THREADS, 2) paged_rows_kernel(const __grid_constant__ PagedAttnArgs a) {
    constexpr int COLS = 8 * NB, LD = 132;
    constexpr int PL = 2;                             // planes of P: the products have room beside the bytes
    static_assert(COLS * LD * 4 <= PR_STAGES * PR_STAGE, "a warp's outputs fit its stages");
    extern __shared__ __align__(128) unsigned char pr_raw[];
    __shared__ long long s_prefix[PG_MAX_BATCH + 1], s_sum[PR_WARPS];
    __shared__ float s_m[PR_WARPS][COLS], s_l[PR_WARPS][COLS];
    __shared__ unsigned s_bad;
    __shared__ float s_res[PG_REDO * PG_PART];
    const int tid = threadIdx.x, lane = tid & 31, warp = uniform_warp();
    const int fg = lane >> 2, ft = lane & 3, lrow = lane & 7, lmat = lane >> 3;
    pdl_launch();
    pdl_wait();
    if (tid == 0) s_bad = 0;
    pg_block_prefix<PR_THREADS>(a.sh, a.c.q_start, a.c.kv_len, s_prefix, s_sum);
    const long long total = s_prefix[a.sh.batch];
    const int blocks = pg_blocks(total, (int)gridDim.x, a.least);
    PgWalk walk;
    if ((int)blockIdx.x >= blocks || !walk.begin(a.sh, s_prefix, a.c.q_start, a.c.kv_len, pg_run_start(total, blocks, blockIdx.x), pg_run_start(total, blocks, blockIdx.x + 1))) {
        if (tid == 0) a.cuts[blockIdx.x].parts = 0;
        return;
    }
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
                        const int last = there ? min(w1 - 1, k.qpos0 + ((8 * nb + 2 * ft + e) >> a.group_log)) : -1;
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
        auto sync = [] { __syncthreads(); };
        for (unsigned bad = s_bad; bad;) {
            const int4 which = pg_take_rows(bad, 0);
            const PgSegment seg = s;                 // (copies: what a call is handed by address would live in memory all along)
            const PgKeys keys = k;
            pg_redo_rows<T, PR_WARPS>(a, seg, keys, which, warp, reinterpret_cast<float*>(pr_raw), s_res, sync);
            const int row[PG_REDO] = {which.x, which.y, which.z, which.w};
#pragma unroll
            for (int i = 0; i < PG_REDO; ++i)
                if (row[i] >= 0) store(row[i], s_res[i * PG_PART], s_res[i * PG_PART + 1], s_res[i * PG_PART + 4 + tid]);
        }
        __syncthreads();
        if (tid == 0) {
            s_bad = 0;
            if (walk.at + s.k1 - s.k0 >= walk.end) pg_leave_cut(a, walk, first, total, blocks);
        }
        first = false;
    } while (walk.next(a.sh, a.c.q_start, a.c.kv_len));
}

// ------------------------------------------------------------------------------------------------------------------------------
// Chunks of new tokens: 128 rows (128 / group tokens of every q head of a kv head) against tiles of 128 keys on tcgen05.mma, accumulators in TMEM.
//     S  = Q K^T     M 128 x N 128 keys x K 128 dims, both K-major        -> TMEM columns [128 i, 128 i + 128) of NS buffers
//     P  = 2^(S - m) NS groups of four warps, a thread a row, take turns at the tiles: a group a buffer.  P takes the place of S in TMEM
//     O += P V       V is the MN-major operand straight from its tile                          -> columns [384, 512) (fp16: an O a group)
// K and V come page by page (a TMA box a page and half of the dims; a page that is not there, or that no row of the tile sees, lies
// outside the tensor and reads as zeros), each by a warp of its own, S and O are issued by a warp each.  A block walks the segments of its run without draining: the warp that
// loads K works them out ahead of the others (code that runs once a segment comes from far away: 4000 clocks where every warp walked for itself), tiles are counted over all
// of them, the next segment's Q has a buffer of its own, its first scores are under way while the last one's rows are finished.
//
// bf16: P has fp32's exponents, so that m need not be the maximum: the largest score of the segment's first tile (0 where a row sees none of it) serves all its
// tiles.  Nothing is rescaled, no other tile is searched for its maximum, one O serves all groups, and there is room for three S.  A row that leaves fp32's range (scores 88 above the first tile's) is not finite at the end, one that has vanished (no weight
// above 2^-100 though it sees keys) is seen by its sum: both are marked, and done again row by row once the block's run is over and nobody waits any more.
// fp16: P must not leave [2^-24, 2^16), so m follows a group's maximum, and its O is rescaled when a score exceeds m by 2^8; two S and two O.
// P is rounded to the pages' type and its sum is that of the rounded values: where few keys hold a row's weight their roundings leave the quotient.  2048 tokens
// behind 8192: 2.3e-3 off, 1.7e-3 of it the output's own rounding (P truncated, as fast: 2.4e-3, and 2.6e-3 with short sequences; a second plane of P would be a third product, 1700 clocks a tile
// for products alone).
//
// Measured: 2048 tokens behind 8192 143 to 168 us from box to box (the clock that the power cap leaves), 0.92 to 1.08 PFLOP/s of the 1.64 that a large product reaches, fp16 205 where bf16
// takes 147; 1650 clocks a tile, of which the special-function pipe has 1024 (an exponential a score),
// the products 1150, the rest are hand-offs.  (Steps: K and V loaded by warps of their own, a thread a row 247 -> 211; one O, scores two tiles ahead 208 -> 178;
// segments worked out ahead, one lane that looks for a group 166 -> 149; masks as bits, O free before its rows are stored 145 -> 143.  A third group of warps that only writes: 128 registers a thread, 153.)  Few rows: 8 sequences of 13 tokens behind up
// to 5000, fp16, 37 to 39 us; the pages at 6.7 TB/s in the steady state (15.9), start, segment ends and join 11, the rest not accounted for.
//
// A wait that gives up lets every later one give up at once (those in which the softmax warps meet are waits like the others); the block then drains what is under way and
// leaves NaN in all rows of its run.
// ------------------------------------------------------------------------------------------------------------------------------
constexpr int PT_MMA_O = 0, PT_LOAD_K = 1, PT_LOAD_V = 2, PT_MMA_S = 3, PT_FIRST = 4;      // warps: products with V and TMEM, TMA of Q and K, TMA of V, scores; from 4 on softmax and
                                                                                           // output (a warp's place in its four is its quarter of the rows)
template <typename T> struct PtShape {
    static constexpr bool ONE = T::BF;                        // one O, m from the first tile
    static constexpr int NS = ONE ? 3 : 2;                    // buffers of S and P
};
constexpr int PT_RING = 4;                                    // segments that have been worked out ahead
constexpr int PT_SCAN = 1 << 15;                              // entries of the page table that are looked at for that: 1024 loads a lane, a millisecond at most of the 200 that a wait has
constexpr int PT_GROUPS = 2, PT_THREADS = 32 * PT_FIRST + PT_GROUPS * 128;
struct PtSeg { int n, b, h, q_row, key0, key1, qpos0, rows, whole, every; };      // n tiles of one item's keys; n < 0: the run is over
constexpr int PT_KEYS = 128;                                  // keys of a tile, the unit of work
constexpr uint32_t PT_BOX = 128 * 128, PT_TILE = 2 * PT_BOX;  // [128 rows][64 dims] with 128-byte swizzle; 128 x 128
constexpr size_t PT_SMEM = 2 * PT_TILE + 2 * 2 * PT_TILE;     // two of Q, two stages of K and V
constexpr float PT_LAG = 8.f;

// The thread looks at the barrier without being parked: a tile has eight hand-offs.
// PARK: it may sleep up to 20 us between two looks (it wakes when the phase completes).
template <bool PARK = false>
__device__ __forceinline__ bool pt_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag, const PagedAttnArgs& a, uint32_t site) {
    unsigned it = 0;
    unsigned long long t0 = 0;
    for (;;) {
        uint32_t ok;
        if constexpr (PARK)
            asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                         : "=r"(ok) : "r"(tc_smem(bar)), "r"(parity), "r"(20000u) : "memory");
        else
            asm volatile("{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                         : "=r"(ok) : "r"(tc_smem(bar)), "r"(parity) : "memory");
        if (ok) return true;
        if (*abort_flag) return false;
        if ((++it & a.wait_looks) == 0) {
            const unsigned long long t = tc_ns();
            if (t0 == 0) t0 = t;
            else if (t - t0 > a.wait_ns) {
                if (a.status) report(a.status, ST_MBAR_TIMEOUT, site, parity);
                *abort_flag = 1;
                return false;
            }
        }
    }
}
template <bool PARK = false>
__device__ __forceinline__ bool pt_wait_warp(uint64_t* bar, uint32_t parity, volatile int* abort_flag, const PagedAttnArgs& a, uint32_t site) {
    return one_lane_waits([&] { return pt_wait<PARK>(bar, parity, abort_flag, a, site); });
}
// MN-major operand: rows are keys (the K index), 64 dims a row; the next 64 dims a box further, the next 8 keys 1024 bytes
__device__ __forceinline__ uint64_t pt_desc_mn(uint32_t smem_addr) {
    return (uint64_t)((smem_addr & 0x3ffffu) >> 4) | (uint64_t)(PT_BOX >> 4) << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
__device__ __forceinline__ void pt_st16(uint32_t taddr, const uint32_t* r) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15};"
                 ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
                   "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(taddr) : "memory");
}
__device__ __forceinline__ float pt_max3(float a, uint32_t b, uint32_t c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(__uint_as_float(b)), "f"(__uint_as_float(c)));
    return d;
}
__device__ __forceinline__ uint64_t pt_pair(float lo, float hi) {
    uint64_t d;
    asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(lo), "f"(hi));
    return d;
}
__device__ __forceinline__ float2 pt_unpair(uint64_t v) {
    float2 d;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(d.x), "=f"(d.y) : "l"(v));
    return d;
}
__device__ __forceinline__ uint64_t pt_fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ uint64_t pt_add2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ void pt_init(uint64_t* bar, uint32_t count) { asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(tc_smem(bar)), "r"(count) : "memory"); }
__device__ __forceinline__ void pt_expect(uint64_t* bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.release.cta.shared::cta.b64 _, [%0], %1;" ::"r"(tc_smem(bar)), "r"(bytes) : "memory");
}
__device__ __forceinline__ void pt_arrive(uint64_t* bar) { asm volatile("mbarrier.arrive.release.cta.shared::cta.b64 _, [%0];" ::"r"(tc_smem(bar)) : "memory"); }
__device__ __forceinline__ void pt_commit(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(tc_smem(bar)) : "memory");
}

// How a group of four softmax warps waits: one lane looks at the barrier, the others sleep at a named barrier (a look takes 100 clocks of the barrier unit: twelve
// warps that looked for themselves saw finished scores 1500 clocks late).  The four warps take every decision together, so they always meet again.
struct PtGroup {
    int grp, quad, lane;
    volatile int* abort_flag;
    const PagedAttnArgs& a;
    __device__ __forceinline__ void sync() const { asm volatile("bar.sync %0, 128;" ::"r"(2 + grp) : "memory"); }
    __device__ __forceinline__ void wait(uint64_t* bar, uint32_t parity, uint32_t site) const {
        if (quad == 0 && lane == 0) pt_wait(bar, parity, abort_flag, a, site);
        __syncwarp();
        sync();
    }
};
// What a row begins with that is to be done again: no number, and not the NaN that a conversion gives.  In a partial result: a maximum that is NaN with a sum of 0.
constexpr uint32_t PT_AGAIN = 0x7fff7ffeu;

template <typename T>
__global__ void __launch_bounds__(PT_THREADS, 1) paged_tile_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                                                                            const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ PagedAttnArgs a) {
    using S = PtShape<T>;
    constexpr bool ONE = S::ONE;
    constexpr int NS = S::NS, GROUPS = PT_GROUPS;
    extern __shared__ __align__(1024) unsigned char pt_raw[];
    __shared__ long long s_prefix[PG_MAX_BATCH + 1], s_sum[PT_THREADS / 32];
    __shared__ __align__(8) uint64_t k_full[2], v_full[2], k_empty[2], v_empty[2], q_full[2], q_empty[2], s_full[NS], p_full[NS], s_free[NS], o_full[2], o_free, ref_full[2], l_full[2], drain_bar[2];
    __shared__ __align__(8) uint64_t seg_full[PT_RING], seg_empty[PT_RING];
    __shared__ PtSeg s_seg[PT_RING];
    __shared__ uint32_t tmem_base_s;
    __shared__ volatile int abort_flag;
    __shared__ float s_ref[2][128];                 // ONE: what a row's P is taken under, by the segment's parity
    __shared__ float s_m[2][128], s_l[2][128];      // what the group that does not write a segment's rows leaves to the other: maximum (fp16) and sum, by the segment's parity
    __shared__ unsigned s_again[4];                 // rows of a segment that are done again, once the run is over
    __shared__ int s_any;                           // whether there are any
    __shared__ int s_ok[GROUPS][2];                   // per group: what its first warp has decided for all four, by the segment's parity (a group without a tile of a segment meets once in it:
                                                      // its first warp may be at the next decision before the others have read this one)
    __shared__ float s_res[PG_REDO * PG_PART];

    const int tid = threadIdx.x, warp = uniform_warp(), lane = tid & 31;
    if (tid < 96 && lane == 0) asm volatile("prefetch.tensormap [%0];" ::"l"(warp == 0 ? &tm_q : warp == 1 ? &tm_k : &tm_v) : "memory");
    pdl_launch();
    pdl_wait();
    pg_block_prefix<PT_THREADS>(a.sh, a.c.q_start, a.c.kv_len, s_prefix, s_sum);
    const long long total = s_prefix[a.sh.batch];
    const int blocks = pg_blocks(total, (int)gridDim.x, a.least);
    if ((int)blockIdx.x >= blocks) {
        if (tid == 0) a.cuts[blockIdx.x].parts = 0;
        return;
    }
    unsigned char* const sKV = pt_raw + 2 * PT_TILE;  // stage s: K at s * 2 * PT_TILE, V right behind it
    if (tid == 0) {
        for (int s = 0; s < 2; ++s) {
            pt_init(&k_full[s], 1); pt_init(&v_full[s], 1); pt_init(&k_empty[s], 1); pt_init(&v_empty[s], 1);
            pt_init(&q_full[s], 1); pt_init(&q_empty[s], 1); pt_init(&l_full[s], 4); pt_init(&ref_full[s], 4);
            pt_init(&o_full[s], 1); pt_init(&drain_bar[s], 1);
        }
        for (int s = 0; s < NS; ++s) { pt_init(&s_full[s], 1); pt_init(&p_full[s], 4); pt_init(&s_free[s], 1); }
        for (int s = 0; s < PT_RING; ++s) { pt_init(&seg_full[s], 1); pt_init(&seg_empty[s], 3 + 4 * GROUPS); }
        pt_init(&o_free, 4);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        abort_flag = 0;
        s_any = 0;
    }
    if (warp == PT_MMA_O) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tc_smem(&tmem_base_s)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem_base = tmem_base_s;
    const int *qs = a.c.q_start, *kl = a.c.kv_len;
    const long long from = pg_run_start(total, blocks, blockIdx.x), to = pg_run_start(total, blocks, blockIdx.x + 1);

    // segment number i as the loader of K has worked it out; n < 0 at the run's end, or after a wait gave up.  One thread, or a warp.
    auto segment = [&](int i) {
        PtSeg d;
        d.n = -1;
        if (pt_wait(&seg_full[i % PT_RING], (uint32_t)(i / PT_RING) & 1u, &abort_flag, a, 95)) {
            d = s_seg[i % PT_RING];
            pt_arrive(&seg_empty[i % PT_RING]);
        }
        return d;
    };
    auto segment_warp = [&](int i) {
        PtSeg d;
        d.n = -1;
        if (pt_wait_warp<true>(&seg_full[i % PT_RING], (uint32_t)(i / PT_RING) & 1u, &abort_flag, a, 95)) {
            d = s_seg[i % PT_RING];
            __syncwarp();
            if (lane == 0) pt_arrive(&seg_empty[i % PT_RING]);
        }
        return d;
    };

    int armed = 0, armed_q = 0;                     // tiles of K (V) and of Q that this warp has requested
    if (warp == PT_LOAD_K || warp == PT_LOAD_V) {
        // ---------------------------------------------------------------------- TMA: a lane a box
        const bool is_v = warp == PT_LOAD_V;
        const int rows_log = min(a.c.page_log, 7), boxes = PT_KEYS >> rows_log, j = lane >> 1, half = lane & 1;      // a page's rows are cut into boxes of 128 at most
        const bool mine = j < boxes;
        const CUtensorMap* const map = is_v ? &tm_v : &tm_k;
        uint64_t *const full = is_v ? v_full : k_full, *const empty = is_v ? v_empty : k_empty;
        const uint32_t dst0 = tc_smem(sKV + (is_v ? PT_TILE : 0)) + (uint32_t)half * PT_BOX + ((uint32_t)j << (rows_log + 7));
        int g = 0, n_q = 0;
        auto load = [&](const PtSeg& d) -> bool {
            const int key0 = d.key0 + (j << rows_log);
            const int* const table = a.c.table + (long long)d.b * a.c.table_stride;
            // the page of this lane's box of tile t, as the table has it
            auto entry = [&](int t) { const int key = key0 + t * PT_KEYS; return mine && key < d.key1 ? table[key >> a.c.page_log] : -1; };
            int next = d.n > 0 ? entry(0) : -1;
            if (d.n > 0 && !is_v) {
                const int buf = n_q & 1;
                if (n_q >= 2 && !pt_wait_warp<true>(&q_empty[buf], ((n_q >> 1) - 1) & 1, &abort_flag, a, 80)) return false;
                if (lane == 0) {
                    pt_expect(&q_full[buf], PT_TILE);
#pragma unroll
                    for (int b = 0; b < 2; ++b)       // rows past q are zeros
                        asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
                                     ::"r"(tc_smem(pt_raw + buf * PT_TILE + b * PT_BOX)), "l"(&tm_q), "r"(64 * b), "r"(d.h << a.group_log), "r"(d.q_row),
                                       "r"(tc_smem(&q_full[buf])) : "memory");
                }
                armed_q = ++n_q;
            }
            for (int t = 0; t < d.n; ++t, ++g) {
                const int s = g & 1, slot = (key0 + t * PT_KEYS) & ((1 << a.c.page_log) - 1);
                const int page = (unsigned)next < (unsigned)a.c.n_pages ? next : a.c.n_pages;      // no such page: outside the tensor
                if (t + 1 < d.n) next = entry(t + 1);  // (on its way while this tile is waited for)
                if (g >= 2 && !pt_wait_warp<true>(&empty[s], ((g >> 1) - 1) & 1, &abort_flag, a, 81)) return false;
                if (lane == 0) pt_expect(&full[s], PT_TILE);
                __syncwarp();
                if (mine)
                    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];"
                                 ::"r"(dst0 + (uint32_t)s * 2u * PT_TILE), "l"(map), "r"(64 * half), "r"(slot), "r"(d.h), "r"(page), "r"(tc_smem(&full[s])) : "memory");
                armed = g + 1;
            }
            return true;
        };
        if (is_v) {
            for (int i = 0;; ++i) {
                const PtSeg d = segment_warp(i);
                if (d.n < 0 || !load(d)) break;
            }
        } else {
            PgWalk w;
            bool left = w.begin(a.sh, s_prefix, qs, kl, from, to), first = true;
            for (int i = 0;; ++i) {
                PtSeg d;
                d.n = -1;
                if (left) {
                    const PgKeys k = pg_keys(a, w.s);
                    d = PtSeg{(k.key1 - k.key0 + PT_KEYS - 1) / PT_KEYS, w.s.b, w.s.h, w.s.seq.q0 + (w.s.r << a.sh.tile_log), k.key0, k.key1, k.qpos0, k.rows, w.whole(), 1};
                    bool every = true, some = false;         // all pages of the segment are there; at least one is
                    const int e0 = k.key0 >> a.c.page_log, e1 = d.n > 0 ? ((k.key1 - 1) >> a.c.page_log) + 1 : e0;
                    const bool known = e1 - e0 <= PT_SCAN;                   // (of more pages every tile looks for its own: the others wait for this)
                    if (!known) { every = false; some = true; }
                    for (int e = e0 + lane; known && e < e1; e += 32) {
                        const bool there = (unsigned)a.c.table[(long long)d.b * a.c.table_stride + e] < (unsigned)a.c.n_pages;
                        every = every && there; some = some || there;
                    }
                    d.every = __all_sync(0xffffffffu, every);
                    if (!__any_sync(0xffffffffu, some)) d.n = 0;             // (a segment without a page, of a caller who drops old ones: as if it had no keys)
                }
                if (i >= PT_RING && !pt_wait_warp<true>(&seg_empty[i % PT_RING], (uint32_t)(i / PT_RING - 1) & 1u, &abort_flag, a, 96)) break;
                if (lane == 0) {
                    s_seg[i % PT_RING] = d;
                    pt_arrive(&seg_full[i % PT_RING]);
                }
                __syncwarp();
                if (d.n < 0 || !load(d)) break;
                if (lane == 0 && w.at + w.s.k1 - w.s.k0 >= w.end) pg_leave_cut(a, w, first, total, blocks);
                first = false;
                left = w.next(a.sh, qs, kl);
            }
        }
    } else if (warp == PT_MMA_S) {
        // ---------------------------------------------------------------------- scores
        if (elect_one()) {
            constexpr uint32_t idesc = (1u << 4) | (T::BF ? (1u << 7) | (1u << 10) : 0u) | ((uint32_t)(128 >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
            constexpr uint64_t BOX = PT_BOX >> 4, TILE = PT_TILE >> 4;
            const uint64_t dq = tc_desc(tc_smem(pt_raw)), dk = tc_desc(tc_smem(sKV));
            bool ok = true;
            for (int i = 0, g = 0, n_q = 0, b = 0, use = 0; ok; ++i) {       // tile, segments with tiles, buffer of S and how often it has been used
                const int n = segment(i).n;
                if (n < 0) break;
                for (int t = 0; t < n; ++t, ++g) {
                    const int s = g & 1, buf = n_q & 1;
                    if (t == 0) ok = pt_wait(&q_full[buf], (n_q >> 1) & 1, &abort_flag, a, 83);
                    ok = ok && pt_wait(&k_full[s], (g >> 1) & 1, &abort_flag, a, 84);
                    if (use > 0) ok = ok && pt_wait(&s_free[b], (use - 1) & 1, &abort_flag, a, 92);      // P of the tile before in this buffer has been multiplied
                    if (!ok) break;
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    const uint64_t dqs = dq + (uint64_t)buf * TILE, dks = dk + (uint64_t)s * 2 * TILE;
#pragma unroll
                    for (int k = 0; k < 8; ++k) {    // 16 dims a step: four steps a box
                        const uint64_t o = (uint64_t)(k >> 2) * BOX + (uint64_t)(k & 3) * 2;
                        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, {%5, %6, %7, %8}, p;\n\t}"
                                     ::"r"(tmem_base + (uint32_t)b * 128u), "l"(dqs + o), "l"(dks + o), "r"(idesc), "r"(k ? 1u : 0u), "r"(0u), "r"(0u), "r"(0u), "r"(0u) : "memory");
                    }
                    pt_commit(&s_full[b]);
                    pt_commit(&k_empty[s]);
                    if (t == n - 1) pt_commit(&q_empty[buf]);
                    if (++b == NS) { b = 0; ++use; }
                }
                if (n > 0) ++n_q;
            }
        }
    } else if (warp == PT_MMA_O) {
        // ---------------------------------------------------------------------- products with V
        if (elect_one()) {
            constexpr uint32_t idesc = (1u << 4) | (T::BF ? (1u << 7) | (1u << 10) : 0u) | (1u << 16) | ((uint32_t)(128 >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
            constexpr uint64_t TILE = PT_TILE >> 4;
            const uint64_t dv = pt_desc_mn(tc_smem(sKV + PT_TILE));
            bool ok = true;
            for (int i = 0, g = 0, seg = 0, b = 0, use = 0; ok; ++i) {
                const int n = segment(i).n;
                if (n < 0) break;
                for (int t = 0; t < n; ++t, ++g) {
                    const int s = g & 1;
                    if (t == 0 && seg > 0) ok = pt_wait(&o_free, (seg - 1) & 1, &abort_flag, a, 85);      // the rows of the segment before have been read
                    ok = ok && pt_wait(&v_full[s], (g >> 1) & 1, &abort_flag, a, 87) && pt_wait(&p_full[b], use & 1, &abort_flag, a, 86);
                    if (!ok) break;
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    const uint64_t dvs = dv + (uint64_t)s * 2 * TILE;
                    const uint32_t tp = tmem_base + (uint32_t)b * 128u, to_o = tmem_base + (ONE ? 384u : 256u + (uint32_t)b * 128u);
#pragma unroll
                    for (int k = 0; k < 8; ++k)      // 16 keys a step: eight columns of P (two a column)
                        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, {%5, %6, %7, %8}, p;\n\t}"
                                     ::"r"(to_o), "r"(tp + (uint32_t)k * 8u), "l"(dvs + (uint64_t)k * (2048 >> 4)), "r"(idesc), "r"((t >= (ONE ? 1 : 2) || k) ? 1u : 0u),
                                       "r"(0u), "r"(0u), "r"(0u), "r"(0u) : "memory");
                    pt_commit(&s_free[b]);
                    pt_commit(&v_empty[s]);
                    if (!ONE) pt_commit(&o_full[b]);
                    else if (t == n - 1) pt_commit(&o_full[0]);
                    if (++b == NS) { b = 0; ++use; }
                }
                if (n > 0) ++seg;
            }
        }
    } else {
        // ---------------------------------------------------------------------- softmax and output: row = TMEM lane
        const int quad = warp & 3, row = quad * 32 + lane, grp = (warp >> 2) - 1, st = tid - 32 * PT_FIRST;
        const uint32_t trow = tmem_base + ((uint32_t)(quad * 32) << 16);
        const PtGroup group{grp, quad, lane, &abort_flag, a};
        bool first = true;
        int g0 = 0, n_q = 0;                         // number of the segment's first tile; segments with tiles
        for (int i = 0;; ++i) {
            if (quad == 0 && lane == 0) s_ok[grp][i & 1] = pt_wait(&seg_full[i % PT_RING], (uint32_t)(i / PT_RING) & 1u, &abort_flag, a, 97);
            __syncwarp();
            group.sync();
            if (!s_ok[grp][i & 1]) break;
            const PtSeg d = s_seg[i % PT_RING];
            __syncwarp();
            if (lane == 0) pt_arrive(&seg_empty[i % PT_RING]);
            const int n = d.n;
            if (n < 0) break;
            const int last = min(d.qpos0 + (row >> a.group_log), d.key1 - 1);       // the last key this row sees
            const bool live = quad * 32 < d.rows;                            // (the warp has a row)
            const int t0 = (grp + GROUPS - g0 % GROUPS) % GROUPS;            // this group's first tile
            float m = -INFINITY, lsum = 0.f;
            auto pages_of = [&](int tile0) {         // bit i: whether the keys 16 i .. of a tile have a page (or nobody sees them)
                const int key = tile0 + 16 * (lane & 7);
                return __ballot_sync(0xffffffffu, key >= d.key1 || pg_page(a.c, d.b, key) >= 0) & 0xffu;
            };
            for (int t = t0; t < n; t += GROUPS) {
                const int g = g0 + t, tile0 = d.key0 + t * PT_KEYS, b = g % NS;
                const uint32_t ts = trow + (uint32_t)b * 128u;
                const unsigned pages = d.every ? 0xffu : pages_of(tile0);
                const bool masked = tile0 + PT_KEYS - 1 > d.qpos0 || tile0 + PT_KEYS > d.key1 || pages != 0xffu;
                group.wait(&s_full[b], (uint32_t)(g / NS) & 1u, 88);
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                auto hide = [&](uint32_t (&r)[32], int h) {                  // what the row does not see of the tile's quarter h
                    const int most = last - tile0 - h * 32;
                    const unsigned there = (pages >> (h * 2)) & 3u;
                    const unsigned sees = (most >= 31 ? 0xffffffffu : most < 0 ? 0u : (2u << most) - 1u) & ((there & 1u ? 0xffffu : 0u) | (there & 2u ? 0xffff0000u : 0u));
#pragma unroll
                    for (int j = 0; j < 32; ++j)
                        if (!((sees >> j) & 1u)) r[j] = 0xff800000u;            // -inf
                };
                if (live && (!ONE || t == 0)) {
                    float x[2] = {-INFINITY, -INFINITY};
#pragma unroll 1
                    for (int h = 0; h < 4; ++h) {
                        uint32_t r[32];
                        tc_ld32(r, ts + (uint32_t)(h * 32));
                        asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
                        if (masked) hide(r, h);
#pragma unroll
                        for (int j = 0; j < 32; j += 4) { x[0] = pt_max3(x[0], r[j], r[j + 1]); x[1] = pt_max3(x[1], r[j + 2], r[j + 3]); }
                    }
                    const float top = fmaxf(x[0], x[1]) * a.scale;
                    if constexpr (ONE) {
                        m = top == -INFINITY ? 0.f : top;
                        s_ref[n_q & 1][row] = m;
                    } else {
                        const bool raise = !(top <= m + PT_LAG);
                        if (__any_sync(0xffffffffu, raise)) {
                            const float c = raise ? pg_ex2(m - top) : 1.f;       // (m of -inf: 0)
                            if (raise) m = top;
                            lsum *= c;
                            if (t >= GROUPS) {       // O of the group's tiles so far, once the last of them has been added
                                pt_wait_warp(&o_full[grp], (uint32_t)((g >> 1) - 1) & 1u, &abort_flag, a, 89);      // (not every warp of the group comes here)
                                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll 1
                                for (int h = 0; h < 128; h += 16) {
                                    uint32_t o[16];
                                    tc_ld16(o, trow + 256u + (uint32_t)(grp * 128 + h));
                                    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
                                    for (int j = 0; j < 16; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * c);
                                    pt_st16(trow + 256u + (uint32_t)(grp * 128 + h), o);
                                }
                            }
                        }
                    }
                }
                if constexpr (ONE) {                 // the group of the first tile leaves its m to the others
                    if (t == 0) {
                        __syncwarp();
                        if (lane == 0) pt_arrive(&ref_full[n_q & 1]);
                    } else if (t == t0) {
                        group.wait(&ref_full[n_q & 1], (uint32_t)(n_q >> 1) & 1u, 93);
                        m = s_ref[n_q & 1][row];
                    }
                }
                if (live) {
                    const float ms = m == -INFINITY ? 0.f : m;               // (nothing seen so far: every exponential is 0)
                    const uint64_t c2 = pt_pair(a.scale, a.scale), m2 = pt_pair(-ms, -ms);
                    uint64_t sum2[2] = {0ull, 0ull};                         // (two elements an instruction where it is one of the FMA pipe's)
                    auto weigh = [&](const uint32_t (&r)[32], int h) {
                        uint32_t pk[16];
#pragma unroll
                        for (int j = 0; j < 16; ++j) {
                            const float2 x2 = pt_unpair(pt_fma2(pt_pair(__uint_as_float(r[2 * j]), __uint_as_float(r[2 * j + 1])), c2, m2));
                            const float e0 = pg_ex2(x2.x), e1 = pg_ex2(x2.y);
                            pk[j] = T::pack(e0, e1);
                            const float2 y = T::unpack(pk[j]);
                            sum2[j & 1] = pt_add2(sum2[j & 1], pt_pair(y.x, y.y));
                        }
                        pt_st16(ts + (uint32_t)(h * 16), pk);                // (over scores that have been read)
                    };
                    if (!masked) {
                        uint32_t r[2][32];
                        tc_ld32(r[0], ts);
                        asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
                        for (int h = 0; h < 4; ++h) {
                            if (h < 3) tc_ld32(r[(h + 1) & 1], ts + (uint32_t)(h * 32 + 32));
                            weigh(r[h & 1], h);
                            if (h < 3) asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
                        }
                    } else {
#pragma unroll 1
                        for (int h = 0; h < 4; ++h) {
                            uint32_t r[32];
                            tc_ld32(r, ts + (uint32_t)(h * 32));
                            asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
                            hide(r, h);
                            weigh(r, h);
                        }
                    }
                    const float2 s2 = pt_unpair(pt_add2(sum2[0], sum2[1]));
                    lsum += s2.x + s2.y;
                    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                }
                if (tile0 + PT_KEYS > d.key1) {
                    // rows of V that no row of this tile sees but whose page is there: what they hold is not ours to multiply, even by 0
                    const int rows_log = min(a.c.page_log, 7), z0 = d.key1 - tile0, z1 = min(PT_KEYS, ((z0 + (1 << rows_log) - 1) >> rows_log) << rows_log);
                    // (with three S a group may be here before V of two tiles ago has landed in this stage, and a barrier that is a phase behind passes for one that is done: first
                    // that tile's product, which is done once at most before this tile's)
                    if (ONE && g >= 2) group.wait(&s_free[(g - 2) % NS], (uint32_t)((g - 2) / NS) & 1u, 99);
                    group.wait(&v_full[g & 1], (uint32_t)(g >> 1) & 1u, 90);
                    for (int e = st & 127; e < (z1 - z0) * 16; e += 128)
                        *reinterpret_cast<uint4*>(sKV + (size_t)(g & 1) * 2 * PT_TILE + PT_TILE + (size_t)((e >> 3) & 1) * PT_BOX + (size_t)(z0 + (e >> 4)) * 128 + (e & 7) * 16) = make_uint4(0, 0, 0, 0);
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                }
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                __syncwarp();
                if (lane == 0) pt_arrive(&p_full[b]);
            }
            // ---- the segment's rows: the groups write in turn, the other goes on to the next segment's tiles ----
            const int par = i & 1;
            if (par != grp) {
                s_l[par][row] = lsum;
                if (!ONE) s_m[par][row] = m;
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                __syncwarp();
                if (lane == 0) pt_arrive(&l_full[par]);
            } else {
                group.wait(&l_full[par], (uint32_t)(i >> 1) & 1u, 94);
                if constexpr (ONE) {
                    if (n > 0) group.wait(&o_full[0], (uint32_t)n_q & 1u, 91);
                } else {
#pragma unroll
                    for (int e = 0; e < 2; ++e) {                            // the last tile of either group
                        const int te = (e + 2 - (g0 & 1)) & 1;
                        if (te < n) group.wait(&o_full[e], (uint32_t)((g0 + te + (n - 1 - te) / 2 * 2) >> 1) & 1u, 91);
                    }
                }
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const bool whole = d.whole != 0;
                float* const parts = a.part + (size_t)(2 * blockIdx.x + (first ? 0 : 1)) * 128 * PG_PART;
                float mx, sum, f[2] = {1.f, 0.f};    // the row's m and sum; what the groups' O are multiplied by (ONE: the one's)
                if constexpr (ONE) {
                    mx = n > 0 ? s_ref[n_q & 1][row] : -INFINITY;
                    sum = lsum + s_l[par][row];
                } else {
                    const float me[2] = {grp == 0 ? m : s_m[par][row], grp == 0 ? s_m[par][row] : m}, le[2] = {grp == 0 ? lsum : s_l[par][row], grp == 0 ? s_l[par][row] : lsum};
                    mx = fmaxf(me[0], me[1]);
                    sum = 0.f;
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        f[e] = me[e] == -INFINITY ? 0.f : me[e] == mx ? 1.f : pg_ex2(me[e] - mx);
                        sum += le[e] * f[e];
                    }
                }
                bool bad = !(sum <= FLT_MAX) || (ONE && n > 0 && last >= d.key0 && sum < 7.9e-31f);      // (2^-100)
                float r = 1.f;                       // the last factor: the sum's inverse, or what makes the sum of a partial result lie between 1 and 4
                if (whole) {
                    r = sum > 0.f || sum != sum ? 1.f / sum : 0.f;
                } else if (ONE && sum > 0.f && sum <= FLT_MAX) {
                    const int e = min(max((int)(__float_as_uint(sum) >> 23) - 127, -126), 126);
                    r = __uint_as_float((unsigned)(127 - e) << 23);
                    sum *= r; mx += (float)e;
                } else if (ONE && sum == 0.f) {
                    mx = -INFINITY;                  // nothing of this part has a weight: what m it would have been taken under is not a maximum that the join may count
                }
                // (a partial result's maxima and sums lie behind its outputs, [32 quarters of 16 bytes][128 rows])
                if (!whole && row < d.rows) reinterpret_cast<float2*>(parts + 128 * HEAD_DIM)[row] = make_float2(mx, sum);
                unsigned char* const o_row = a.out + (long long)(d.q_row + (row >> a.group_log)) * a.o_token + (long long)((d.h << a.group_log) + (row & ((1 << a.group_log) - 1))) * a.o_head;
                uint64_t odd = 0ull;                 // 0, or NaN once an output is not finite
                if (ONE && live && whole && n > 0) {         // O is free for the next segment's before its rows are stored
                    uint32_t pk[64];
                    const uint64_t r2 = pt_pair(r, r);
#pragma unroll
                    for (int e = 0; e < HEAD_DIM; e += 32) {
                        uint32_t v[32];
                        tc_ld32(v, trow + 384u + (uint32_t)e);
                        asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
                        for (int j = 0; j < 16; ++j) {
                            const uint64_t o = pt_pair(__uint_as_float(v[2 * j]), __uint_as_float(v[2 * j + 1]));
                            odd = pt_fma2(o, 0ull, odd);
                            const float2 x = pt_unpair(pt_fma2(o, r2, 0x8000000080000000ull));
                            pk[e / 2 + j] = T::pack(x.x, x.y);
                        }
                    }
                    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                    __syncwarp();
                    if (lane == 0) pt_arrive(&o_free);
                    if (row < d.rows)
#pragma unroll
                        for (int j = 0; j < 16; ++j) *reinterpret_cast<uint4*>(o_row + j * 16) = make_uint4(pk[4 * j], pk[4 * j + 1], pk[4 * j + 2], pk[4 * j + 3]);
                } else if (live) {
#pragma unroll 1
                    for (int e = 0; e < HEAD_DIM; e += 32) {
                        uint64_t o[16];
                        if (n > 0) {
                            uint32_t v[32];
                            tc_ld32(v, trow + (ONE ? 384u : 256u) + (uint32_t)e);
                            asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
                            // (a group without a tile, or without a key that the row sees, has a factor of 0: TMEM may hold anything there)
#pragma unroll
                            for (int j = 0; j < 16; ++j)
                                o[j] = ONE ? pt_pair(__uint_as_float(v[2 * j]), __uint_as_float(v[2 * j + 1]))
                                           : f[0] != 0.f ? pt_pair(__uint_as_float(v[2 * j]) * f[0], __uint_as_float(v[2 * j + 1]) * f[0]) : 0ull;
                            if constexpr (!ONE) {
                                tc_ld32(v, trow + 384u + (uint32_t)e);
                                asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
                                if (f[1] != 0.f)
#pragma unroll
                                    for (int j = 0; j < 16; ++j) o[j] = pt_fma2(pt_pair(__uint_as_float(v[2 * j]), __uint_as_float(v[2 * j + 1])), pt_pair(f[1], f[1]), o[j]);
                            }
                        } else {
#pragma unroll
                            for (int j = 0; j < 16; ++j) o[j] = 0ull;
                        }
                        if (e == HEAD_DIM - 32 && n > 0) {       // O has been read
                            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                            __syncwarp();
                            if (lane == 0) pt_arrive(&o_free);
                        }
                        const uint64_t r2 = pt_pair(r, r);
#pragma unroll
                        for (int j = 0; j < 16; ++j) {
                            odd = pt_fma2(o[j], 0ull, odd);
                            o[j] = pt_fma2(o[j], r2, 0x8000000080000000ull);      // (minus zero: added to anything it changes nothing)
                        }
                        if (row < d.rows) {
                            if (!whole) {
#pragma unroll
                                for (int j = 0; j < 8; ++j) {
                                    const float2 lo = pt_unpair(o[2 * j]), hi = pt_unpair(o[2 * j + 1]);
                                    reinterpret_cast<float4*>(parts)[(e / 4 + j) * 128 + row] = make_float4(lo.x, lo.y, hi.x, hi.y);
                                }
                            } else {
#pragma unroll
                                for (int j = 0; j < 4; ++j) {
                                    uint32_t pk[4];
#pragma unroll
                                    for (int q = 0; q < 4; ++q) { const float2 x = pt_unpair(o[4 * j + q]); pk[q] = T::pack(x.x, x.y); }
                                    *reinterpret_cast<uint4*>(o_row + e * 2 + j * 16) = make_uint4(pk[0], pk[1], pk[2], pk[3]);
                                }
                            }
                        }
                    }
                } else if (n > 0) {
                    __syncwarp();
                    if (lane == 0) pt_arrive(&o_free);
                }
                const float2 odd2 = pt_unpair(odd);
                bad = (bad || odd2.x != 0.f || odd2.y != 0.f) && row < d.rows;
                // A sum that is NaN has a seen score that is NaN or infinite in it (what is hidden is -inf before the exponential): the row is NaN, and once more would not change it.
                // All others are marked, and done again when nobody waits any more.
                const bool spoiled = sum != sum;
                if (bad && !spoiled) s_any = 1;
                if (bad && whole && !spoiled) *reinterpret_cast<uint32_t*>(o_row) = PT_AGAIN;
                if (bad && !whole) reinterpret_cast<float2*>(parts + 128 * HEAD_DIM)[row] = make_float2(NAN, spoiled ? NAN : 0.f);
            }
            if (n > 0) {
                ++n_q;
                g0 += n;
            }
            first = false;
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (abort_flag) {
        // A wait gave up (nobody waits any more): the loads land and the products end before this block's memory and columns are somebody else's, and no row of the run
        // passes for finished.
        if ((warp == PT_LOAD_K || warp == PT_LOAD_V) && lane == 0) {
            for (int i = max(0, armed_q - 2); i < armed_q; ++i) tc_drain(&q_full[i & 1], (i >> 1) & 1);
            for (int i = max(0, armed - 2); i < armed; ++i) tc_drain(warp == PT_LOAD_K ? &k_full[i & 1] : &v_full[i & 1], (i >> 1) & 1);
        }
        if ((warp == PT_MMA_O || warp == PT_MMA_S) && elect_one()) {
            pt_commit(&drain_bar[warp == PT_MMA_S]);
            tc_drain(&drain_bar[warp == PT_MMA_S], 0);
        }
        __syncthreads();
    }
    if (warp == PT_MMA_O) {                          // (before the rows that are done again: another kernel's block may be waiting for columns)
        __syncwarp();
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(512u) : "memory");
    }
    if (abort_flag) {
        PgWalk w;
        bool left = w.begin(a.sh, s_prefix, qs, kl, from, to), first = true;
        while (left) {
            const int rows = pg_keys(a, w.s).rows;
            float* const parts = a.part + (size_t)(2 * blockIdx.x + (first ? 0 : 1)) * 128 * PG_PART;
            for (int e = tid; e < rows * 64; e += PT_THREADS) {
                if (w.whole()) *reinterpret_cast<uint32_t*>(pg_o_row(a, w.s, e >> 6) + (e & 63) * 4) = 0x7fff7fffu;
                else if ((e & 63) == 0) reinterpret_cast<float2*>(parts + 128 * HEAD_DIM)[e >> 6] = make_float2(NAN, NAN);
            }
            if (tid == 0 && w.at + w.s.k1 - w.s.k0 >= w.end) pg_leave_cut(a, w, first, total, blocks);
            first = false;
            left = w.next(a.sh, qs, kl);
        }
    } else if (s_any) {
        // The run is over, its memory is free and no wait depends on how long this takes: the marked rows, all warps at their keys.  (64 tokens of 16 heads behind
        // 33000 positions, whose last V row holds an infinity: 2.2 ms instead of 70 us; 2048 behind 8192 with scores that rise by 120: 19 ms instead of 170 us.)
        float* const room = reinterpret_cast<float*>(pt_raw);
        auto sync = [] { __syncthreads(); };
        PgWalk w;
        bool left = w.begin(a.sh, s_prefix, qs, kl, from, to), first = true;
        while (left) {
            const PgSegment seg = w.s;
            const PgKeys keys = pg_keys(a, seg);
            const bool whole = w.whole();
            float* const parts = a.part + (size_t)(2 * blockIdx.x + (first ? 0 : 1)) * 128 * PG_PART;
            float2* const stats = reinterpret_cast<float2*>(parts + 128 * HEAD_DIM);
            if (warp < 4) {
                bool bad = tid < keys.rows;
                if (bad) bad = whole ? *reinterpret_cast<const uint32_t*>(pg_o_row(a, seg, tid)) == PT_AGAIN : stats[tid].x != stats[tid].x && stats[tid].y == 0.f;
                const unsigned again = __ballot_sync(0xffffffffu, bad);
                if (lane == 0) s_again[warp] = again;
            }
            __syncthreads();
            for (int q = 0; q < 4; ++q)
                for (unsigned set = s_again[q]; set;) {
                    const int4 which = pg_take_rows(set, q * 32);
                    pg_redo_rows<T, PT_THREADS / 32>(a, seg, keys, which, warp, room, s_res, sync);
                    const int row[PG_REDO] = {which.x, which.y, which.z, which.w};
                    if (warp < 4)
#pragma unroll
                        for (int i = 0; i < PG_REDO; ++i) {
                            const int rr = row[i];
                            const float* const done = s_res + i * PG_PART;
                            const float L = done[1], inv = L > 0.f || L != L ? 1.f / L : 0.f, x = done[4 + tid], up = __shfl_down_sync(0xffffffffu, x, 1);
                            if (rr < 0) continue;
                            if (whole) {
                                if (!(tid & 1)) *reinterpret_cast<uint32_t*>(pg_o_row(a, seg, rr) + tid * 2) = T::pack(x * inv, up * inv);
                            } else {
                                parts[((tid >> 2) * 128 + rr) * 4 + (tid & 3)] = x;
                                if (tid == 0) stats[rr] = make_float2(done[0], L);
                            }
                        }
                }
            __syncthreads();                         // (the marks have been read)
            first = false;
            left = w.next(a.sh, qs, kl);
        }
    }
}

// ------------------------------------------------------------------------------------------------------------------------------
// Items that were cut: the block in whose run an item began has left word of it.  Blocks take rows in turn; the four warps of a block a quarter of the parts each, a lane
// four dims; everything is added in a fixed order.
// ------------------------------------------------------------------------------------------------------------------------------
constexpr int PJ_THREADS = 128;

template <typename T>
__global__ void __launch_bounds__(PJ_THREADS) paged_join_kernel(const PagedAttnArgs a, int part_rows) {
    __shared__ float4 s_v[4][32];
    __shared__ float2 s_ml[4];
    pdl_launch();
    pdl_wait();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, block = blockIdx.x;
    const int4 cut = *reinterpret_cast<const int4*>(&a.cuts[block]);
    const int parts = cut.x;
    if (parts == 0) return;
    PgSegment s;
    s.b = cut.z; s.h = cut.w; s.r = a.cuts[block].r;
    s.seq = pg_seq(a.sh, a.c.q_start, a.c.kv_len, s.b);
    const int live = min(1 << a.sh.tile_log, s.seq.q - (s.r << a.sh.tile_log)) << a.group_log;
    auto part = [&](int i, int row) { return a.part + ((size_t)(2 * (block + i) + (i == 0 ? cut.y : 0)) * part_rows + row) * PG_PART; };
    const int each = (parts + 3) / 4, p0 = min(warp * each, parts), p1 = min(p0 + each, parts);
    for (int row = blockIdx.y; row < live; row += gridDim.y) {
        float M = -INFINITY, L = 0.f;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int i0 = p0; i0 < p1; i0 += 8) {        // eight parts' loads under way
            float2 ml[8];
            float4 x[8];
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (i0 + i < p1) {
                    ml[i] = *reinterpret_cast<const float2*>(part(i0 + i, row));
                    x[i] = *reinterpret_cast<const float4*>(part(i0 + i, row) + 4 + lane * 4);
                }
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (i0 + i < p1 && ml[i].x != -INFINITY) {
                    const float top = ml[i].x > M || ml[i].x != ml[i].x ? ml[i].x : M, f = M == top ? 1.f : pg_ex2(M - top), w = ml[i].x == top ? 1.f : pg_ex2(ml[i].x - top);
                    M = top;
                    L = L * f + ml[i].y * w;
                    v.x = v.x * f + x[i].x * w; v.y = v.y * f + x[i].y * w; v.z = v.z * f + x[i].z * w; v.w = v.w * f + x[i].w * w;
                }
        }
        s_v[warp][lane] = v;
        if (lane == 0) s_ml[warp] = make_float2(M, L);
        __syncthreads();
        if (warp == 0) {
            float top = -INFINITY;
            bool nan = false;
#pragma unroll
            for (int i = 0; i < 4; ++i) { top = fmaxf(top, s_ml[i].x); nan = nan || s_ml[i].x != s_ml[i].x; }
            if (nan) top = NAN;
            L = 0.f;
            v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float m = s_ml[i].x;
                if (m == -INFINITY) continue;
                const float w = m == top ? 1.f : pg_ex2(m - top);
                const float4 x = s_v[i][lane];
                L += s_ml[i].y * w;
                v.x = fmaf(x.x, w, v.x); v.y = fmaf(x.y, w, v.y); v.z = fmaf(x.z, w, v.z); v.w = fmaf(x.w, w, v.w);
            }
            const float r = L > 0.f || L != L ? 1.f / L : 0.f;
            *reinterpret_cast<uint2*>(pg_o_row(a, s, row) + lane * 8) = make_uint2(T::pack(v.x * r, v.y * r), T::pack(v.z * r, v.w * r));
        }
        __syncthreads();
    }
}

// The same for results of the tile kernel, whose outputs lie [32 quarters of 16 bytes][128 rows] with the maxima and sums behind them: a lane a row, a warp eight quarters (8 answers 39.1 us, 38.2 with two parts at a time).
template <typename T>
__global__ void __launch_bounds__(PJ_THREADS) paged_join_tiles_kernel(const PagedAttnArgs a) {
    pdl_launch();
    pdl_wait();
    const int lane = threadIdx.x & 31, d0 = (threadIdx.x >> 5) * 8, block = blockIdx.x, row = blockIdx.y * 32 + lane;
    const int4 cut = *reinterpret_cast<const int4*>(&a.cuts[block]);
    const int parts = cut.x;
    if (parts == 0) return;
    PgSegment s;
    s.b = cut.z; s.h = cut.w; s.r = a.cuts[block].r;
    s.seq = pg_seq(a.sh, a.c.q_start, a.c.kv_len, s.b);
    const int live = min(1 << a.sh.tile_log, s.seq.q - (s.r << a.sh.tile_log)) << a.group_log;
    if (row >= live) return;
    auto part = [&](int i) { return a.part + (size_t)(2 * (block + i) + (i == 0 ? cut.y : 0)) * 128 * PG_PART; };
    auto stats = [&](int i) { return reinterpret_cast<const float2*>(part(i) + 128 * HEAD_DIM)[row]; };
    float M = -INFINITY;
    bool nan = false;
#pragma unroll 4
    for (int i = 0; i < parts; ++i) { const float x = stats(i).x; M = fmaxf(M, x); nan = nan || x != x; }
    if (nan) M = NAN;
    const float Ms = M == -INFINITY ? 0.f : M;
    float L = 0.f;
    float4 v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int i0 = 0; i0 < parts; i0 += 2) {          // two parts' loads under way
        float4 x[2][8];
        float2 ml[2];
#pragma unroll
        for (int i = 0; i < 2; ++i)
            if (i0 + i < parts) {
                ml[i] = stats(i0 + i);
#pragma unroll
                for (int j = 0; j < 8; ++j) x[i][j] = reinterpret_cast<const float4*>(part(i0 + i))[(d0 + j) * 128 + row];
            }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const float w = i0 + i >= parts || ml[i].x == -INFINITY ? 0.f : ml[i].x == Ms ? 1.f : pg_ex2(ml[i].x - Ms);
            if (w != 0.f) {
                L = fmaf(ml[i].y, w, L);
#pragma unroll
                for (int j = 0; j < 8; ++j) { v[j].x = fmaf(x[i][j].x, w, v[j].x); v[j].y = fmaf(x[i][j].y, w, v[j].y); v[j].z = fmaf(x[i][j].z, w, v[j].z); v[j].w = fmaf(x[i][j].w, w, v[j].w); }
            }
        }
    }
    const float r = L > 0.f || L != L ? 1.f / L : 0.f;
    unsigned char* const out = pg_o_row(a, s, row) + d0 * 8;
#pragma unroll
    for (int j = 0; j < 8; j += 2)
        *reinterpret_cast<uint4*>(out + j * 8) = make_uint4(T::pack(v[j].x * r, v[j].y * r), T::pack(v[j].z * r, v[j].w * r), T::pack(v[j + 1].x * r, v[j + 1].y * r), T::pack(v[j + 1].z * r, v[j + 1].w * r));
}

// ------------------------------------------------------------------------------------------------------------------------------
// Up to 16 rows (new tokens times the q heads of a kv head) the few-row kernel has the products, beyond the tile kernel.  us a call, few-row / tile kernel: 8 sequences of up to
// 5000 positions with 6 new tokens each, group 2 (12 rows) 31.4 / 37.2, fp16 31.6 / 38.5, 13 (26 rows, four column blocks) 48.7 / 39.1, fp16 48.6 / 40.3;
// 16 sequences, 2 tokens, group 8 (16 rows) 24.8 / 28.4; one sequence of 300 positions and 13 tokens 24.9 / 22.7.
static bool pg_few(int max_new, int group) { return max_new * (long long)group <= 16; }
static int pg_log(int n) {
    int l = 0;
    while ((1 << l) < n) ++l;
    return l;
}

// what a kernel asks for beyond the defaults, once for every device (a benign race between host threads: the same value is set)
template <typename K>
static cudaError_t pg_shared(K* kernel, size_t bytes, bool (&set)[64]) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess || dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
    if (!set[dev]) {
        if ((e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes)) != cudaSuccess) return e;
        set[dev] = true;
    }
    return cudaSuccess;
}

template <typename T, int NB>
static cudaError_t launch_rows(PagedAttnArgs& a, int rows, cudaStream_t st) {
    a.sh.unit_log = PR_UNIT_LOG;
    a.sh.tile_log = (NB == 1 ? 3 : 4) - a.group_log;
    a.least = 1;
    const int grid = 2 * tc_sm_count();
    static bool set[64] = {};
    cudaError_t e = pg_shared(paged_rows_kernel<T, NB>, PR_SMEM, set);
    if (e == cudaSuccess) e = launch_chain(paged_rows_kernel<T, NB>, dim3(grid), dim3(PR_THREADS), PR_SMEM, st, a);
    if (e == cudaSuccess) e = launch_chain(paged_join_kernel<T>, dim3(grid, rows), dim3(PJ_THREADS), 0, st, a, 8 * NB);
    return e;
}

// Tensor maps of q [tokens][heads][128] and of the pages [pages][heads][slots][128]: boxes of 64 dims, 128-byte swizzle
static bool pg_make_map(CUtensorMap* m, bool bf, const void* p, int rank, const uint64_t* dims, const int64_t* strides, const uint32_t* box) {
    static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;      // (a benign race between host threads: the same value is written)
    if (!fn) {
        void* f = nullptr;
        cudaDriverEntryPointQueryResult found;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault, &found) != cudaSuccess || found != cudaDriverEntryPointSuccess) return false;
        fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(f);
    }
    cuuint64_t d[4], s[3];
    cuuint32_t b[4];
    const cuuint32_t step[4] = {1, 1, 1, 1};
    for (int i = 0; i < rank; ++i) { d[i] = dims[i]; b[i] = box[i]; }
    for (int i = 1; i < rank; ++i) s[i - 1] = dims[i] > 1 ? strides[i - 1] : 256;      // (a dimension of one element has no stride)
    return fn(m, bf ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, rank, const_cast<void*>(p), d, s, b, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T>
static cudaError_t launch_tiles(PagedAttnArgs& a, int q_heads, cudaStream_t st) {
    a.sh.unit_log = 7;
    a.sh.tile_log = 7 - a.group_log;
    a.least = 1;
    CUtensorMap q, k, v;
    const uint64_t dq[3] = {HEAD_DIM, (uint64_t)q_heads, (uint64_t)a.sh.n_tokens}, dk[4] = {HEAD_DIM, 1ull << a.c.page_log, (uint64_t)a.sh.heads, (uint64_t)a.c.n_pages};
    const int64_t sq[2] = {a.q_head, a.q_token}, sk[3] = {a.c.slot_bytes, a.c.head_bytes, a.c.page_bytes};
    const uint32_t bq[3] = {64, 1u << a.group_log, 1u << a.sh.tile_log}, bk[4] = {64, 1u << (a.c.page_log < 7 ? a.c.page_log : 7), 1, 1};
    if (!pg_make_map(&q, T::BF, a.q, 3, dq, sq, bq) || !pg_make_map(&k, T::BF, a.c.k, 4, dk, sk, bk) || !pg_make_map(&v, T::BF, a.c.v, 4, dk, sk, bk)) return cudaErrorInvalidValue;
    const int grid = tc_sm_count();
    static bool set[64] = {};
    cudaError_t e = pg_shared(paged_tile_kernel<T>, PT_SMEM, set);
    if (e == cudaSuccess) e = launch_chain(paged_tile_kernel<T>, dim3(grid), dim3(PT_THREADS), PT_SMEM, st, q, k, v, a);
    if (e == cudaSuccess) e = launch_chain(paged_join_tiles_kernel<T>, dim3(grid, 4), dim3(PJ_THREADS), 0, st, a);
    return e;
}

template <typename T>
static cudaError_t launch_attn(PagedAttnArgs& a, int max_new, int q_heads, cudaStream_t st) {
    if (!pg_few(max_new, 1 << a.group_log)) return launch_tiles<T>(a, q_heads, st);
    const int cols = max_new << a.group_log;
    return cols <= 8 ? launch_rows<T, 1>(a, cols, st) : launch_rows<T, 2>(a, cols, st);
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
    const struct { int64_t stride; int32_t count; } dims[3] = {{c->page_stride, c->n_pages}, {c->slot_stride, c->page_size}, {c->head_stride, c->kv_heads}};
    for (const auto& d : dims)
        if (d.stride < 0 || d.stride > most || d.stride % 8 || (d.count > 1 && d.stride < HEAD_DIM)) return bad("strides of the pages must be multiples of 8 elements, at least 128");
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

static int64_t pg_cut_bytes() { return ((int64_t)2 * tc_sm_count() * (int64_t)sizeof(PgCut) + 1023) / 1024 * 1024; }
// a record a block, two partial results a block: 16 rows at most for each of two blocks an SM, or 128 for one
extern "C" int64_t q3_paged_attn_workspace(const q3_paged* c, int32_t q_heads) {
    if (!c || q_heads < 1) return engine_fail(nullptr, Q3_ERR_INVALID, "q3_paged_attn_workspace: bad argument");
    const int sms = tc_sm_count();
    if (sms < 1) return engine_fail(nullptr, Q3_ERR_CUDA, "q3_paged_attn_workspace: no CUDA device");
    const int group = q_heads / (c->kv_heads < 1 ? 1 : c->kv_heads);
    return pg_cut_bytes() + (int64_t)2 * sms * (pg_few(c->max_new, group) ? 2 * 16 : 128) * PG_PART * 4;
}

extern "C" int q3_paged_attn(const q3_paged* c, const q3_paged_attn_args* p, void* stream) { return q3_paged_attn_limited(c, p, 0, stream); }
extern "C" int q3_paged_attn_limited(const q3_paged* c, const q3_paged_attn_args* p, int32_t wait_limit_us, void* stream) {
    const char* who = "q3_paged_attn";
    if (const int rc = paged_check(who, c)) return rc;
    auto bad = [&](const char* what) { return engine_fail(nullptr, Q3_ERR_INVALID, "%s: %s", who, what); };
    if (!p) return bad("null argument");
    if (wait_limit_us < 0) return bad("wait_limit_us must not be negative");
    if (c->n_tokens == 0) return Q3_OK;
    if (!p->q || !p->out || !p->workspace) return bad("q, out and workspace are required");
    if (reinterpret_cast<uintptr_t>(p->status) & 3) return bad("status must be 4-byte aligned");
    const int group = p->q_heads / c->kv_heads;
    if (p->q_heads < 1 || p->q_heads % c->kv_heads || (group != 1 && group != 2 && group != 4 && group != 8))
        return engine_fail(nullptr, Q3_ERR_INVALID, "%s: %d q heads over %d kv heads: a kv head serves 1, 2, 4 or 8", who, p->q_heads, c->kv_heads);
    if (p->out == p->q) return bad("out must not be q (rows are read again where a result is not finite)");
    if (!(p->scale > 0.f) || p->scale > 1e30f) return bad("scale must be positive and at most 1e30");
    if ((reinterpret_cast<uintptr_t>(p->q) | reinterpret_cast<uintptr_t>(p->out) | reinterpret_cast<uintptr_t>(p->workspace)) & 15) return bad("q, out and workspace must be 16-byte aligned");
    const int64_t most = 1ll << 38;
    const struct { int64_t stride; int32_t count; } dims[4] = {{p->q_token, c->n_tokens}, {p->out_token, c->n_tokens}, {p->q_head, p->q_heads}, {p->out_head, p->q_heads}};
    for (const auto& d : dims)
        if (d.stride < 0 || d.stride > most || d.stride % 8 || (d.count > 1 && d.stride < HEAD_DIM)) return bad("strides of q and out must be multiples of 8 elements, at least 128");
    // (rows are stored while others are still read, and q is read again where a result is not finite)
    const RowSet q_rows{reinterpret_cast<uintptr_t>(p->q), 2 * p->q_token, 2 * p->q_head, c->n_tokens, p->q_heads, 2 * HEAD_DIM};
    const RowSet o_rows{reinterpret_cast<uintptr_t>(p->out), 2 * p->out_token, 2 * p->out_head, c->n_tokens, p->q_heads, 2 * HEAD_DIM};
    if (rows_meet_themselves(o_rows)) return bad("rows of out must not overlap");
    const Meet meet = rows_meet(q_rows, o_rows);
    if (meet == Meet::Yes) return bad("q and out must not overlap");
    if (meet == Meet::Unknown) return bad("q and out must not overlap: where their address ranges meet, their token strides must be the same");
    const int64_t need = q3_paged_attn_workspace(c, p->q_heads);
    if (need < 0) return (int)need;
    if (p->workspace_bytes < need) return engine_fail(nullptr, Q3_ERR_INVALID, "%s: workspace holds %lld bytes, %lld needed", who, (long long)p->workspace_bytes, (long long)need);
    PagedAttnArgs a{};
    a.c = paged_view(c);
    a.sh.heads = c->kv_heads; a.sh.batch = c->batch; a.sh.n_tokens = c->n_tokens; a.sh.most_keys = c->table_pages * c->page_size;
    a.group_log = pg_log(group);
    a.q = static_cast<const unsigned char*>(p->q);
    a.out = static_cast<unsigned char*>(p->out);
    a.q_token = 2 * p->q_token; a.q_head = 2 * p->q_head; a.o_token = 2 * p->out_token; a.o_head = 2 * p->out_head;
    a.scale = p->scale * 1.4426950408889634f;
    a.cuts = static_cast<PgCut*>(p->workspace);
    a.part = reinterpret_cast<float*>(static_cast<char*>(p->workspace) + pg_cut_bytes());
    a.status = p->status;
    a.wait_ns = wait_limit_us > 0 ? (unsigned long long)wait_limit_us * 1000ull : TC_WAIT_NS;
    a.wait_looks = wait_limit_us > 0 && wait_limit_us < 100 ? 0u : 63u;      // (64 looks take 3 us)
    cudaStream_t st = (cudaStream_t)stream;
    const int max_new = c->max_new < 1 ? 1 : c->max_new;
    const cudaError_t err = c->type == Q3_TYPE_BF16 ? launch_attn<PgBf16>(a, max_new, p->q_heads, st) : launch_attn<PgFp16>(a, max_new, p->q_heads, st);
    if (err != cudaSuccess) return engine_fail(nullptr, Q3_ERR_CUDA, "%s: %s", who, cudaGetErrorString(err));
    return Q3_OK;
}
