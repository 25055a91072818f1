// Sampling with a temperature, top-k, top-p and min-p of its own for every row, from given random numbers.
//
//     w_i = exp((l_i - max) / T);  keep the k largest (ties at the k-th value are all kept);  of these the most likely ones, equal words in the order of
//     their indices, until their weights reach p times the sum;  of these w_i >= min_p;  the first index whose inclusive sum exceeds u times the total.
//
// A word is an ELEMENT, (order-preserving key of its logit, ~index) in 64 bits: no two are alike and descending order is the order above, so every filter but
// min-p is "elements >= some element".  Weights are added as integers, in units of 2^-40 of the most likely word's: sums do not depend on the
// order of the adds, prefix sums meet without gaps, and the same logits and numbers draw the same word on every run.  (Rounding to units moves a sum of
// 2^17 words by 2^-24 at most; where the whole row takes part, words of less than half a unit count by the sum of a thread's.)
//
// A CLUSTER of blocks a row.  Usually few words are kept:
//   1. every thread finds the maximum of its words (and, where top-p or no filter at all needs the sum over the row, that sum, under its running maximum);
//   2. the threads' maxima are binned over the cluster; the bins of the K largest maxima (K = top_k, or for a nucleus so many that about 850 words are expected there) bound the row's K largest words from below.  A nucleus
//      is usually far smaller: the bound is where the maxima alone weigh enough; and no bound is lower than min_p's.  The few words at or above it go to the cluster's first block;
//   3. which sorts them, cuts the sorted list by k, p and min_p, adds up what is kept in the order of the indices and draws.
// Where that is not enough (the nucleus is wider than the candidates, k of about 1000 and more, many equal words) the element at the cut is searched with passes over the row (from
// L2): bins of all words' counts and weights, then, while the words about the cut do not fit the list, eight brackets a pass; the draw then walks the row.
//
// Bound by latencies: 64 rows (39 MB, 6 us as a copy) 24 to 31 us, of which the pass over the row 10, two exchanges 2, bins 2.6, candidates 2 to 4, order, cut and draw 2 to 5; one row of
// top-k 20 14.5; a wide nucleus among 27 rows up to 45.
#include <cooperative_groups.h>

#include <cfloat>

#include "q3_engine.h"

namespace cg = cooperative_groups;

namespace q3 {

typedef unsigned long long u64;

constexpr int SR_THREADS = 1024, SR_WARPS = 32, SR_MAX_CLUSTER = 16, SR_BINS = 512, SR_LIST = 1024, SR_NUCLEUS = 850, SR_FEW = 256, SR_CUTS = 7;
constexpr float SR_FAR = 96.f;          // logits further than this many temperatures below the maximum weigh e^-96: no unit
constexpr float SR_UNIT = 1099511627776.f;      // 2^40

struct SampleRowsArgs {
    const float* logits;
    long long row_stride;
    int vocab, nucleus;                 // nucleus: thread maxima that bound the candidates where no top-k does
    const float *temperature, *top_p, *min_p;
    const int* top_k;
    float temperature1, top_p1, min_p1;      // where the arrays are not given
    int top_k1;
    const float* uniform;
    long long* out;
};

__device__ __forceinline__ unsigned sr_key(float f) {
    const unsigned b = __float_as_uint(f + 0.f);      // (-0 and 0 are equal words)
    return b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float sr_value(unsigned k) { return __uint_as_float((k >> 31) ? k ^ 0x80000000u : ~k); }
__device__ __forceinline__ u64 sr_element(float v, int i) { return (u64)sr_key(v) << 32 | (unsigned)~i; }
__device__ __forceinline__ float sr_warp_max(float v) {
    float m;
    asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(m) : "f"(v));
    return m;
}
__device__ __forceinline__ u64 sr_units(float w) { return __float2ull_rn(w * SR_UNIT); }
__device__ __forceinline__ u64 sr_shfl_xor(u64 v, int o) { return __shfl_xor_sync(0xffffffffu, v, o); }
__device__ __forceinline__ u64 sr_warp_sum(u64 v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += sr_shfl_xor(v, o);
    return v;
}

__device__ __forceinline__ u64 sr_pair(float lo, float hi) {
    u64 d;
    asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(lo), "f"(hi));
    return d;
}
__device__ __forceinline__ float2 sr_unpair(u64 v) {
    float2 d;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(d.x), "=f"(d.y) : "l"(v));
    return d;
}
__device__ __forceinline__ u64 sr_add2(u64 a, u64 b) {
    u64 d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ u64 sr_mul2(u64 a, u64 b) {
    u64 d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ float sr_ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float sr_max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

struct SampleRowsShared {
    float bmax[SR_MAX_CLUSTER], blo[SR_MAX_CLUSTER];      // per block of the cluster: its maximum, the smallest of its threads' finite maxima,
    u64 bsum[SR_MAX_CLUSTER];                             // the sum of its weights under its own maximum, then under the row's
    int bidx[SR_MAX_CLUSTER], bnan[SR_MAX_CLUSTER];
    float wf[SR_WARPS], wg[SR_WARPS];
    u64 wsum[SR_WARPS];
    unsigned wcount[SR_WARPS];
    unsigned hist[SR_BINS];
    u64 list[SR_LIST];                                    // first block: the candidates, then the sorted list
    u64 weight[SR_LIST];                                  // ... and its weights
    u64 place[SR_FEW];                                    // of few elements: how many are larger, the weights at lower indices
    u64 cutw[SR_MAX_CLUSTER][SR_CUTS];                    // search: weights and counts at or above each cut, per block
    unsigned cutc[SR_MAX_CLUSTER][SR_CUTS];
    u64 wcutw[SR_WARPS][SR_CUTS];
    unsigned wcutc[SR_WARPS][SR_CUTS];
    unsigned n, sel, hit, verdict;
    u64 found;
};

// Inclusive prefix sum over the block's threads; ends with a barrier.
__device__ __forceinline__ u64 sr_scan(SampleRowsShared& sh, u64 v) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const u64 p = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += p;
    }
    if (lane == 31) sh.wsum[warp] = v;
    __syncthreads();
    u64 before = lane < warp ? sh.wsum[lane] : 0ull;
    before = sr_warp_sum(before);
    __syncthreads();
    return v + before;
}

__device__ __forceinline__ int sr_power(int n) { return n <= 1 ? 1 : 1 << (32 - __clz(n - 1)); }

// Few things are compared each with all others, by the whole block: f(mine, other) for things 0 .. n - 1 (n at most SR_FEW), several threads a thing.
template <typename F>
__device__ __forceinline__ void sr_pairs(int n, F&& f) {
    const int n2 = max(32, sr_power(n)), parts = SR_THREADS / n2, each = (n + parts - 1) / parts, one = threadIdx.x & (n2 - 1), j0 = threadIdx.x / n2 * each;
    f(one < n ? one : 0, one < n, j0, min(j0 + each, n));
}

// The n elements of sh.list in descending order, there and (one a thread) returned; threads from n on get 0.  No two are alike.  Up to SR_FEW of them by counting how many are
// larger; more by a bitonic network, whose exchanges within a warp are shuffles, by as many warps as have elements.  (The network by all warps for any n: one row's top 20
// 16.5 us, now 14.7, 27 mixed rows 23.5 and 18.8, 64 nuclei 34.6 and 30.9.)
__device__ __forceinline__ u64 sr_sort(SampleRowsShared& sh, int n) {
    const int t = threadIdx.x;
    if (n <= SR_FEW) {
        if (t < SR_FEW) sh.place[t] = 0ull;
        const u64 v = t < n ? sh.list[t] : 0ull;
        __syncthreads();
        sr_pairs(n, [&](int one, bool real, int j0, int j1) {
            const u64 own = sh.list[one];
            unsigned c = 0u;
            for (int j = j0; j < j1; ++j) c += sh.list[j] > own;
            if (real && c) atomicAdd(reinterpret_cast<unsigned*>(&sh.place[one]), c);
        });
        __syncthreads();
        if (t < n) sh.list[(unsigned)sh.place[t]] = v;
        __syncthreads();
        return t < n ? sh.list[t] : 0ull;
    }
    const int n2 = sr_power(n);
    u64 v = t < n ? sh.list[t] : 0ull;
    if (t < n2) {
        auto meet = [&] { asm volatile("bar.sync 1, %0;" ::"r"(n2) : "memory"); };
        for (int k = 2; k <= n2; k <<= 1)
            for (int j = k >> 1; j > 0; j >>= 1) {
                u64 o;
                if (j >= 32) {
                    meet();
                    sh.list[t] = v;
                    meet();
                    o = sh.list[t ^ j];
                } else {
                    o = sr_shfl_xor(v, j);
                }
                const bool larger = ((t & j) == 0) == ((t & k) == 0);     // this place takes the larger one
                v = larger ? max(v, o) : min(v, o);
            }
        meet();
        sh.list[t] = v;
    }
    __syncthreads();
    return v;
}

__global__ void __launch_bounds__(SR_THREADS, 1) sample_rows_kernel(const SampleRowsArgs a) {
    __shared__ SampleRowsShared sh;
    cg::cluster_group cluster = cg::this_cluster();
    const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int row_id = blockIdx.x / C, vocab = a.vocab;
    const float* row = a.logits + (long long)row_id * a.row_stride;
    // warp w of block r: elements [i0, i1), `per` of them but for the row's last runs; four neighbours a lane, in groups of 128
    const int per = ((vocab + C * SR_WARPS - 1) / (C * SR_WARPS) + 127) / 128 * 128;
    auto run_start = [&](int w) { return (int)min((long long)vocab, (long long)(rank * SR_WARPS + w) * per); };
    const int i0 = run_start(warp), i1 = run_start(warp + 1);
    const bool vec = (reinterpret_cast<uintptr_t>(row) & 15) == 0;
    // (below 1e-36 the factor and its products would leave fp32's range; words that differ by more than 1e-34 have weights of 0 or 1 there, too)
    const float T0 = a.temperature ? a.temperature[row_id] : a.temperature1, T = T0 > 0.f ? fmaxf(T0, 1e-36f) : T0, u = a.uniform[row_id];
    const int k = a.top_k ? a.top_k[row_id] : a.top_k1;
    float p = a.top_p ? a.top_p[row_id] : a.top_p1, min_p = a.min_p ? a.min_p[row_id] : a.min_p1;
    if (!(p < 1.f)) p = 1.f;
    if (!(min_p > 0.f)) min_p = 0.f;
    const bool by_k = k > 0 && k < vocab, by_p = p < 1.f, filtered = by_k || by_p || min_p > 0.f;
    bool greedy = !(T > 0.f) || k == 1 || min_p > 1.f || !(p > 0.f) || !(u >= 0.f && u < 1.f);
    const bool summed = !greedy && !by_k && (by_p || !filtered);      // the sum over the whole row is needed
    const float inv_t = 1.f / T;
    // (a masked word, -inf, weighs nothing at any temperature)
    auto weight = [&](float v, float top) { return v < -FLT_MAX ? 0.f : __expf(fmaxf(v - top, -FLT_MAX) * inv_t); };
    cluster.barrier_arrive();           // (waited for before the first write to a peer)

    auto fetch = [&](int j, int of) -> float4 {                        // group j of lane `of`; what lies past the run is -inf
        const int i = i0 + 128 * j + 4 * of;
        if (vec && i + 3 < i1) return *reinterpret_cast<const float4*>(row + i);
        float4 v;
        v.x = i < i1 ? row[i] : -INFINITY; v.y = i + 1 < i1 ? row[i + 1] : -INFINITY;
        v.z = i + 2 < i1 ? row[i + 2] : -INFINITY; v.w = i + 3 < i1 ? row[i + 3] : -INFINITY;
        return v;
    };
    const int groups = (i1 - i0 + 127) / 128, whole = vec ? (i1 - i0) / 128 : 0;
    auto batches = [&](auto&& f) {                                     // f(four groups' words); the next four are under way meanwhile
        float4 v[2][4];
        auto load = [&](int j, float4 (&d)[4]) {
            if (j + 4 <= whole) {                                      // (no guards)
#pragma unroll
                for (int q = 0; q < 4; ++q) d[q] = *reinterpret_cast<const float4*>(row + i0 + 128 * (j + q) + 4 * lane);
            } else {
#pragma unroll
                for (int q = 0; q < 4; ++q) d[q] = fetch(j + q, lane);
            }
        };
        if (groups > 0) load(0, v[0]);
        for (int j = 0; j < groups; j += 8) {
            if (j + 4 < groups) load(j + 4, v[1]);
            f(v[0]);
            if (j + 8 < groups) load(j + 8, v[0]);
            if (j + 4 < groups) f(v[1]);
        }
    };
    auto each = [&](auto&& f) {                                        // f(index, word) over this thread's words, in ascending order (paths that few rows take)
        float4 next = groups > 0 ? fetch(0, lane) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
        for (int j = 0; j < groups; ++j) {
            const float4 v = next;
            if (j + 1 < groups) next = fetch(j + 1, lane);
            const int i = i0 + 128 * j + 4 * lane;
#pragma unroll 1
            for (int q = 0; q < 4; ++q)
                if (i + q < i1) f(i + q, q == 0 ? v.x : q == 1 ? v.y : q == 2 ? v.z : v.w);
        }
    };

    // ---- 1. maxima and, where needed, sums ----
    float mine = -INFINITY, wsum = 0.f;
    bool odd = false;                                                  // a word is no number
    const float c_t = inv_t * 1.4426950408889634f;
    const u64 c2 = sr_pair(c_t, c_t);
    u64 sum2 = 0ull;                                                   // (two words an instruction)
    batches([&](const float4 (&v)[4]) {
        float top = -INFINITY;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            top = sr_max3(sr_max3(top, v[q].x, v[q].y), v[q].z, v[q].w);
            odd = odd || v[q].x != v[q].x || v[q].y != v[q].y || v[q].z != v[q].z || v[q].w != v[q].w;
        }
        if (!summed) { mine = fmaxf(mine, top); return; }
        if (top > mine) {
            if (mine > -INFINITY) { const float f = sr_ex2(fmaxf(mine - top, -FLT_MAX) * c_t); sum2 = sr_mul2(sum2, sr_pair(f, f)); }
            mine = top;
        }
        if (mine == -INFINITY) return;
        const u64 less = sr_pair(-mine, -mine);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            // (a masked word: -inf times the factor is -inf, of weight 0; only a factor of 0 needs a look)
            float2 x = sr_unpair(sr_mul2(sr_add2(sr_pair(v[q].x, v[q].y), less), c2)), y = sr_unpair(sr_mul2(sr_add2(sr_pair(v[q].z, v[q].w), less), c2));
            if (c_t == 0.f) {
                x.x = v[q].x < -FLT_MAX ? -INFINITY : 0.f; x.y = v[q].y < -FLT_MAX ? -INFINITY : 0.f;
                y.x = v[q].z < -FLT_MAX ? -INFINITY : 0.f; y.y = v[q].w < -FLT_MAX ? -INFINITY : 0.f;
            }
            sum2 = sr_add2(sum2, sr_add2(sr_pair(sr_ex2(x.x), sr_ex2(x.y)), sr_pair(sr_ex2(y.x), sr_ex2(y.y))));
        }
    });
    if (summed) { const float2 s = sr_unpair(sum2); wsum = s.x + s.y; }
    for (int b = tid; b < SR_BINS; b += SR_THREADS) sh.hist[b] = 0u;
    {
        const float bv = sr_warp_max(mine), lo = -sr_warp_max(mine >= -FLT_MAX ? -mine : -INFINITY);
        if (lane == 0) { sh.wf[warp] = bv; sh.wg[warp] = lo; }
        if (tid == 0) { sh.n = 0u; sh.hit = 0u; sh.verdict = 0u; }
    }
    const bool nan = __syncthreads_or(odd);
    const float bmax = sr_warp_max(sh.wf[lane]), blo = -sr_warp_max(-sh.wg[lane]);
    cluster.barrier_wait();
    if (tid < C) {
        SampleRowsShared* peer = cluster.map_shared_rank(&sh, tid);
        peer->bmax[rank] = bmax; peer->blo[rank] = blo; peer->bnan[rank] = nan;
    }
    cluster.sync();
    const float vmax = sr_warp_max(lane < C ? sh.bmax[lane] : -INFINITY), vlo = -sr_warp_max(lane < C ? -sh.blo[lane] : -INFINITY);
    // a NaN, an infinite maximum, a row without a word: no draw
    greedy = greedy || __any_sync(0xffffffffu, lane < C && sh.bnan[lane] != 0) || !(vmax >= -FLT_MAX && vmax <= FLT_MAX);

    if (greedy) {                       // the lowest index that holds the maximum
        __syncthreads();
        if (tid == 0) sh.hit = 0x7fffffffu;
        __syncthreads();
        if (mine == vmax) {
            int first = 0x7fffffff;
            each([&](int i, float v) { if (v == vmax) first = min(first, i); });
            atomicMin(&sh.hit, (unsigned)first);
        }
        __syncthreads();
        if (tid == 0) cluster.map_shared_rank(&sh, 0)->bidx[rank] = (int)sh.hit;
        cluster.sync();
        if (rank == 0 && tid == 0) {
            int best = sh.bidx[0];
            for (int r = 1; r < C; ++r) best = min(best, sh.bidx[r]);
            a.out[row_id] = best < vocab ? best : 0;      // (a row of NaNs has no maximum)
        }
        return;
    }

    // ---- the sum of the row's weights, thread by thread in units ----
    u64 own_sum = 0ull, row_sum = 0ull;                   // this warp's and the row's
    auto exchange_sums = [&](u64 mine_units) {            // own_sum, sh.wsum per warp, sh.bsum per block, row_sum
        own_sum = sr_warp_sum(mine_units);
        __syncthreads();
        if (lane == 0) sh.wsum[warp] = own_sum;
        __syncthreads();
        const u64 block = sr_warp_sum(sh.wsum[lane]);
        if (tid < C) cluster.map_shared_rank(&sh, tid)->bsum[rank] = block;
        cluster.sync();
        row_sum = sr_warp_sum(lane < C ? sh.bsum[lane] : 0ull);
    };
    if (summed) exchange_sums(sr_units(mine > -INFINITY ? wsum * __expf(fmaxf(mine - vmax, -FLT_MAX) * inv_t) : 0.f));

    u64 least = 0ull;                                     // the smallest element that is kept (min-p aside)
    if (filtered) {
        // ---- 2. candidates ----
        const float range = fminf(vmax - vlo, SR_FAR * T);
        const bool clipped = range < vmax - vlo;          // what the last bin holds weighs nothing
        const float scale = (float)(SR_BINS - 1) / range;
        auto bin = [&](float v) -> int {
            const float d = (vmax - v) * scale;
            return d >= 0.f ? (int)fminf(d, (float)(SR_BINS - 1)) : 0;
        };
        if (mine >= -FLT_MAX) atomicAdd(&sh.hist[bin(mine)], 1u);
        if (tid == 0) sh.sel = SR_BINS - 1;
        cluster.sync();
        {
            // thread t: bin t over the cluster.  The bound is the bin in which the count of the threads' maxima reaches K, or, for a nucleus, before that the one with which
            // these maxima alone weigh enough (each taken at its bin's far end).  (512 bins: every block reads every other's, 2048 cost one row 2 us more)
            unsigned c = 0u;
            if (tid < SR_BINS)
#pragma unroll
                for (int r = 0; r < SR_MAX_CLUSTER; ++r)
                    if (r < C) c += cluster.map_shared_rank(&sh, r)->hist[tid];
            const unsigned need = by_k ? (unsigned)k : (unsigned)a.nucleus;
            const u64 incl = sr_scan(sh, (u64)c), before = incl - c;
            if (before < need && incl >= need) atomicMin(&sh.sel, (unsigned)tid);
            if (by_p && !by_k) {
                const u64 mass = (u64)c * sr_units(sr_ex2(-(float)(tid + 1) * (c_t / scale))), upto = sr_scan(sh, mass);
                const double reach = (double)p * (double)row_sum * 1.00001;
                if ((double)(upto - mass) < reach && (double)upto >= reach) atomicMin(&sh.sel, (unsigned)tid);
            }
            __syncthreads();
        }
        int last = (int)sh.sel;
        if (clipped) last = min(last, SR_BINS - 2);
        // words below min_p are not kept, whatever the others are (but where top-p asks for the k largest's sum): its bin bounds the candidates, too
        int floor_bin = SR_BINS;
        if (min_p > 0.f && !(by_k && by_p)) floor_bin = (int)fminf(-__logf(min_p) * T * scale * 1.0001f, (float)SR_BINS) + 1;
        const bool floored = floor_bin <= last;
        last = min(last, floor_bin);
        const bool all = floored || last == SR_BINS - 1 || (clipped && last == SR_BINS - 2);     // every word that may be kept is a candidate
        SampleRowsShared* const first = cluster.map_shared_rank(&sh, 0);
        auto take = [&](int i, float v) {
            if (i < i1 && v >= -FLT_MAX && bin(v) <= last) {
                const unsigned n = atomicAdd(&first->n, 1u);
                if (n < SR_LIST) first->list[n] = sr_element(v, i);
            }
        };
        // the few threads that have some: their words again, a lane a group, four threads' loads under way
        for (unsigned m = __ballot_sync(0xffffffffu, mine >= -FLT_MAX && bin(mine) <= last); m; ) {
            int of[4];
#pragma unroll
            for (int q = 0; q < 4; ++q) { of[q] = m ? __ffs(m) - 1 : -1; m &= m - 1; }
            for (int j = lane; j < groups; j += 32) {
                float4 v[4];
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    if (of[q] >= 0) v[q] = fetch(j, of[q]);
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const int i = i0 + 128 * j + 4 * of[q];
                    if (of[q] >= 0) { take(i, v[q].x); take(i + 1, v[q].y); take(i + 2, v[q].z); take(i + 3, v[q].w); }
                }
            }
        }
        cluster.sync();
        // ---- 3. the first block: sort, cut, draw ----
        if (rank == 0 && sh.n <= SR_LIST) {
            const int n = (int)sh.n;
            const u64 e = sr_sort(sh, n);
            const float w = tid < n ? weight(sr_value((unsigned)(e >> 32)), vmax) : 0.f;
            const u64 units = sr_units(w), incl = sr_scan(sh, units);
            sh.weight[tid] = incl;
            if (tid == 0) sh.hit = SR_LIST;
            __syncthreads();
            // Are the words that are kept among the candidates?  The k largest are (or every word with a weight is); a nucleus is where it reaches p times the sum here;
            // by min-p alone where the last candidate is below it.
            bool enough = all || by_k;
            u64 sum = row_sum;
            int in_k = n;
            if (by_k) {
                const unsigned kth = n >= k ? (unsigned)(sh.list[k - 1] >> 32) : 0u;
                in_k = __syncthreads_count(tid < n && (unsigned)(e >> 32) >= kth);
                sum = sh.weight[in_k - 1];
            }
            const double reach = (double)p * (double)sum;
            if (by_p && !enough) enough = n > 0 && (double)sh.weight[n - 1] >= reach;
            if (!by_k && min_p > 0.f && !enough) enough = n > 0 && weight(sr_value((unsigned)(sh.list[n - 1] >> 32)), vmax) < min_p;
            if (enough) {
                // what is kept is the beginning of the sorted list
                const bool keep = tid < in_k && (tid == 0 || ((!by_p || (double)(incl - units) < reach) && w >= min_p));
                const int m = __syncthreads_count(keep);
                const u64 target = (u64)((double)u * (double)sh.weight[m - 1]);
                // ... by index
                __syncthreads();
                sh.weight[tid] = units;
                if (m <= SR_FEW) {
                    if (tid < SR_FEW) sh.place[tid] = 0ull;
                    __syncthreads();
                    sr_pairs(m, [&](int one, bool real, int j0, int j1) {
                        const unsigned own = (unsigned)sh.list[one];      // ~index
                        u64 before = 0ull;
                        for (int j = j0; j < j1; ++j) before += (unsigned)sh.list[j] > own ? sh.weight[j] : 0ull;
                        if (real && before) atomicAdd(&sh.place[one], before);
                    });
                    __syncthreads();
                    if (tid < m && sh.place[tid] + units > target && sh.place[tid] <= target) a.out[row_id] = (long long)(unsigned)~(unsigned)e;
                } else {
                    sh.list[tid] = (e << 32) | (unsigned)tid;             // ~index above the place: descending
                    __syncthreads();
                    const u64 x = sr_sort(sh, m);
                    const u64 wi = tid < m ? sh.weight[(unsigned)x & (SR_LIST - 1)] : 0ull, prefix = sr_scan(sh, wi);
                    if (tid < m && prefix > target && prefix - wi <= target) a.out[row_id] = (long long)(unsigned)~(unsigned)(x >> 32);
                }
                if (tid == 0) sh.verdict = 1u;
            }
        }
        cluster.sync();
        if (first->verdict) { cluster.sync(); return; }
        // ---- the cut by passes over the row ----
        // The smallest element that is kept when elements are taken in descending order until their count (of_count) or weight reaches `need`.
        auto search = [&](bool of_count, double need, u64 floor) -> u64 {
            auto reached = [&](unsigned c, u64 w) { return of_count ? (double)c >= need : (double)w >= need; };
            // Where the cut lies to within a bin: counts of all words, and their weights in 2^-31 of a bound of the sum.  Such sums are off by half a unit a word, so the bins
            // between which the cut lies are those with which it may be reached and with which it must be.
            const double unit = 2147483648.0 / ((double)row_sum > 0. ? (double)row_sum * 1.001 : 1099511627776.0 * vocab) * 1099511627776.0;
            unsigned* const mass = reinterpret_cast<unsigned*>(sh.weight);
            __syncthreads();
            for (int b = tid; b < SR_BINS; b += SR_THREADS) { sh.hist[b] = 0u; mass[b] = 0u; }
            if (tid == 0) { sh.sel = SR_BINS - 1; sh.n = SR_BINS - 1; }
            __syncthreads();
            {
                unsigned far_c = 0u, far_m = 0u;                  // the last bin's, which holds most words, stay with the thread
                each([&](int i, float v) {
                    if (v >= -FLT_MAX && sr_element(v, i) >= floor) {
                        const int b = bin(v);
                        const unsigned m = (unsigned)(weight(v, vmax) * (float)unit + 0.5f);
                        if (b == SR_BINS - 1) { ++far_c; far_m += m; }
                        else { atomicAdd(&sh.hist[b], 1u); if (m) atomicAdd(&mass[b], m); }
                    }
                });
                far_c = __reduce_add_sync(0xffffffffu, far_c); far_m = __reduce_add_sync(0xffffffffu, far_m);
                if (lane == 0) { atomicAdd(&sh.hist[SR_BINS - 1], far_c); atomicAdd(&mass[SR_BINS - 1], far_m); }
            }
            cluster.sync();
            {
                unsigned c = 0u;
                u64 m = 0ull;
                if (tid < SR_BINS)
                    for (int r = 0; r < C; ++r) {
                        SampleRowsShared* peer = cluster.map_shared_rank(&sh, r);
                        c += peer->hist[tid]; m += reinterpret_cast<unsigned*>(peer->weight)[tid];
                    }
                const u64 cc = sr_scan(sh, c), mm = sr_scan(sh, m);
                const double want = of_count ? need : need * (unit / 1099511627776.0), have = of_count ? (double)cc : (double)mm, err = of_count ? 0. : 0.51 * (double)cc + 1. + 1e-6 * want;
                if (tid < SR_BINS && have + err >= want) atomicMin(&sh.sel, (unsigned)tid);
                if (tid < SR_BINS && have - err >= want) atomicMin(&sh.n, (unsigned)tid);
            }
            __syncthreads();
            const int b1 = (int)sh.sel, b2 = (int)sh.n;
            // the smallest element whose word's bin is at most b
            auto bound = [&](int b) -> u64 {
                unsigned key = 0u;                                // the largest key of a bin beyond b: keys ascend, bins descend
                for (int bit = 31; bit >= 0; --bit) {
                    const unsigned trial = key | (1u << bit);
                    const float v = sr_value(trial);
                    if (trial <= sr_key(vmax) && (v != v || v < -FLT_MAX || bin(v) > b)) key = trial;
                }
                return (u64)(key + 1u) << 32;
            };
            u64 lo = b2 >= SR_BINS - 1 ? floor : max(floor, bound(b2)), hi = b1 == 0 ? ((u64)sr_key(vmax) + 1) << 32 : max(lo, bound(b1 - 1)), hi_w = 0ull;      // everything at or above hi is kept
            unsigned hi_c = 0u, lo_c = 0xffffffffu;
            {
                unsigned c = 0u;
                u64 w = 0ull;
                each([&](int i, float v) {
                    if (v >= -FLT_MAX && sr_element(v, i) >= hi) { ++c; w += sr_units(weight(v, vmax)); }
                });
                c = __reduce_add_sync(0xffffffffu, c); w = sr_warp_sum(w);
                if (lane == 0) { sh.wcutc[warp][0] = c; sh.wcutw[warp][0] = w; }
                __syncthreads();
                if (warp == 0) {
                    c = __reduce_add_sync(0xffffffffu, sh.wcutc[lane][0]); w = sr_warp_sum(sh.wcutw[lane][0]);
                    if (lane < C) {
                        SampleRowsShared* peer = cluster.map_shared_rank(&sh, lane);
                        peer->cutc[rank][0] = c; peer->cutw[rank][0] = w;
                    }
                }
                cluster.sync();
                for (int r = 0; r < C; ++r) { hi_c += sh.cutc[r][0]; hi_w += sh.cutw[r][0]; }
                cluster.sync();                                   // every block has read
                // (the count of a nucleus' bins and its exact sum may differ about a border: the words at or above hi reach it by themselves)
                if (hi_c > 0u && reached(hi_c, hi_w)) { hi = ((u64)sr_key(vmax) + 1) << 32; hi_c = 0u; hi_w = 0ull; }
            }
            for (;;) {
                const u64 step = (hi - lo) / (SR_CUTS + 1);
                if (lo_c != 0xffffffffu && (lo_c - hi_c <= SR_LIST || step == 0)) break;
                u64 cut[SR_CUTS];
#pragma unroll
                for (int j = 0; j < SR_CUTS; ++j) cut[j] = lo + step * j + (j ? (hi - lo) % (SR_CUTS + 1) * j / (SR_CUTS + 1) : 0);   // cut[0] = lo: is it reached at all?
                unsigned c[SR_CUTS] = {};
                u64 w[SR_CUTS] = {};
                each([&](int i, float v) {
                    const u64 e = sr_element(v, i);
                    if (v >= -FLT_MAX && e >= lo && e < hi) {
                        const u64 units = sr_units(weight(v, vmax));
#pragma unroll
                        for (int j = 0; j < SR_CUTS; ++j)
                            if (e >= cut[j]) { ++c[j]; w[j] += units; }
                    }
                });
                __syncthreads();
#pragma unroll
                for (int j = 0; j < SR_CUTS; ++j) {
                    const unsigned cj = __reduce_add_sync(0xffffffffu, c[j]);
                    const u64 wj = sr_warp_sum(w[j]);
                    if (lane == 0) { sh.wcutc[warp][j] = cj; sh.wcutw[warp][j] = wj; }
                }
                __syncthreads();
                if (warp < SR_CUTS) {
                    const unsigned cj = __reduce_add_sync(0xffffffffu, sh.wcutc[lane][warp]);
                    const u64 wj = sr_warp_sum(sh.wcutw[lane][warp]);
                    if (lane < C) {
                        SampleRowsShared* peer = cluster.map_shared_rank(&sh, lane);
                        peer->cutc[rank][warp] = cj; peer->cutw[rank][warp] = wj;
                    }
                }
                cluster.sync();
                u64 new_lo = lo, new_hi = hi, new_hw = hi_w;
                unsigned new_lc = 0u, new_hc = hi_c;
#pragma unroll
                for (int j = SR_CUTS - 1; j >= 0; --j) {          // from the highest cut down: the first one that is reached is the new lo
                    unsigned cj = hi_c;
                    u64 wj = hi_w;
                    for (int r = 0; r < C; ++r) { cj += sh.cutc[r][j]; wj += sh.cutw[r][j]; }
                    if (new_lc == 0u) {
                        if (reached(cj, wj) || j == 0) { new_lo = cut[j]; new_lc = cj; if (j == 0 && !reached(cj, wj)) { new_lc = 0xfffffffeu; new_hc = cj; new_hw = wj; } }
                        else { new_hi = cut[j]; new_hc = cj; new_hw = wj; }
                    }
                }
                cluster.sync();                                   // every block has read
                if (new_lc == 0xfffffffeu) {
                    if (lo == floor) return floor;                // all words together fall short: all are kept
                    hi = lo; hi_c = new_hc; hi_w = new_hw; lo = floor; lo_c = 0xffffffffu;
                    continue;
                }
                lo = new_lo; hi = new_hi; hi_w = new_hw; hi_c = new_hc; lo_c = new_lc;
            }
            // the bracket's words, sorted by the first block
            if (tid == 0) sh.n = 0u;
            cluster.sync();
            each([&](int i, float v) {
                const u64 e = sr_element(v, i);
                if (v >= -FLT_MAX && e >= lo && e < hi) {
                    const unsigned n = atomicAdd(&first->n, 1u);
                    if (n < SR_LIST) first->list[n] = e;
                }
            });
            cluster.sync();
            if (rank == 0) {
                const int n = (int)min(sh.n, (unsigned)SR_LIST);
                const u64 e = sr_sort(sh, n);
                const u64 units = tid < n ? sr_units(weight(sr_value((unsigned)(e >> 32)), vmax)) : 0ull, incl = sr_scan(sh, units);
                if (tid == 0) sh.found = lo;
                __syncthreads();
                // the first one with which `need` is reached
                if (tid < n && reached(hi_c + tid + 1, hi_w + incl) && !(tid > 0 && reached(hi_c + tid, hi_w + incl - units))) sh.found = e;
                __syncthreads();
            }
            cluster.sync();
            const u64 e = first->found;
            cluster.sync();
            return e;
        };
        if (by_k) least = search(true, (double)k, 0ull) & 0xffffffff00000000ull;      // ties at the k-th value are all kept
        if (by_p) {
            if (by_k) {
                u64 s = 0ull;
                each([&](int i, float v) { if (sr_element(v, i) >= least) s += sr_units(weight(v, vmax)); });
                exchange_sums(s);
            }
            least = search(false, (double)p * (double)row_sum, least);
        }
    }
    // ---- 4. the draw over the whole row ----
    auto kept = [&](int i, float v, float w) { return sr_element(v, i) >= least && w >= min_p; };
    if (filtered) {
        u64 s = 0ull;
        each([&](int i, float v) { const float w = weight(v, vmax); if (kept(i, v, w)) s += sr_units(w); });
        cluster.sync();                                           // (the sums of the exchange before have been read)
        exchange_sums(s);
    }
    const u64 target = (u64)((double)u * (double)row_sum);
    u64 base = 0ull, next = 0ull;
    for (int r = 0; r <= rank; ++r) { base = next; next += sh.bsum[r]; }
    if (base <= target && target < next) {
        u64 from = base;
        for (int w = 0; w < warp; ++w) from += sh.wsum[w];
        if (lane == 0 && from <= target && target < from + own_sum) { sh.sel = (unsigned)warp; sh.found = from; }
        if (tid == 0) { sh.hit = 0xffffffffu; sh.n = 0u; }
        __syncthreads();
        // exactly one warp's run holds the target; the block walks it, a word a thread
        const int r0 = run_start((int)sh.sel), r1 = run_start((int)sh.sel + 1);
        u64 run = sh.found;
        for (int f = r0; f < r1; f += SR_THREADS) {
            const int i = f + tid;
            const float v = i < r1 ? row[i] : -INFINITY, w = weight(v, vmax);
            const bool part = i < r1 && w > 0.f && kept(i, v, w);
            const u64 units = part ? sr_units(w) : 0ull, incl = sr_scan(sh, units);
            if (units && run + incl > target) atomicMin(&sh.hit, (unsigned)i);
            if (part) atomicMax(&sh.n, (unsigned)i + 1u);
            if (tid == SR_THREADS - 1) sh.weight[0] = incl;
            __syncthreads();
            run += sh.weight[0];
            const bool hit = sh.hit != 0xffffffffu;
            __syncthreads();
            if (hit) break;
        }
        // (a thread's sum is rounded to units once, its words one by one: the run may end short of the target, then its last word with a weight)
        if (tid == 0) a.out[row_id] = sh.hit != 0xffffffffu ? (long long)sh.hit : (long long)sh.n - 1;
    }
    cluster.sync();
}

}  // namespace q3

using namespace q3;

extern "C" int q3_sample_rows(const q3_sample_rows_args* p, void* stream) {
    auto bad = [&](const char* what) { return engine_fail(nullptr, Q3_ERR_INVALID, "q3_sample_rows: %s", what); };
    if (!p) return bad("null argument");
    if (!p->logits || !p->out_tokens || !p->uniform) return bad("logits, uniform and out_tokens are required");
    if (p->batch < 1 || p->batch > (1 << 20) || p->vocab < 1 || p->vocab > (1 << 22) || (p->row_stride < p->vocab && p->row_stride != 0))
        return engine_fail(nullptr, Q3_ERR_INVALID, "q3_sample_rows: batch=%d vocab=%d (1..2^22) row_stride=%lld out of range", p->batch, p->vocab, (long long)p->row_stride);
    if (!p->top_ks && p->top_k < 0) return bad("top_k must not be negative");
    if (!p->temperatures && p->temperature != p->temperature) return bad("temperature is not a number");
    if ((!p->top_ps && !(p->top_p >= 0.f)) || (!p->min_ps && !(p->min_p >= 0.f))) return bad("top_p and min_p must not be negative");
    const uintptr_t words = reinterpret_cast<uintptr_t>(p->logits) | reinterpret_cast<uintptr_t>(p->uniform) | reinterpret_cast<uintptr_t>(p->temperatures) |
                            reinterpret_cast<uintptr_t>(p->top_ks) | reinterpret_cast<uintptr_t>(p->top_ps) | reinterpret_cast<uintptr_t>(p->min_ps);
    if ((words & 3) || (reinterpret_cast<uintptr_t>(p->out_tokens) & 7)) return bad("logits and parameters must be 4-byte aligned, out_tokens 8-byte aligned");
    SampleRowsArgs a{};
    a.logits = p->logits; a.row_stride = p->row_stride; a.vocab = p->vocab;
    a.temperature = p->temperatures; a.top_p = p->top_ps; a.min_p = p->min_ps; a.top_k = p->top_ks;
    a.temperature1 = p->temperature; a.top_p1 = p->top_p; a.min_p1 = p->min_p; a.top_k1 = p->top_k;
    a.uniform = p->uniform; a.out = reinterpret_cast<long long*>(p->out_tokens);
    int cluster = p->batch <= 4 ? 16 : p->batch <= 14 ? 8 : p->batch <= 36 ? 4 : p->batch <= 74 ? 2 : 1;
    while (cluster > 1 && p->vocab < cluster * SR_THREADS) cluster /= 2;
    // N threads of which k hold words beyond a bound hold -N ln(1 - k/N) of them, if words are spread evenly: SR_NUCLEUS leaves the list of SR_LIST room for a bin more
    // (512 maxima whatever N: 27 mixed rows up to 210 us, where one has a nucleus of 500 words or more; now 45 at most over 200 draws, 20 in the middle)
    a.nucleus = (int)(cluster * SR_THREADS * (1. - exp(-(double)SR_NUCLEUS / (cluster * SR_THREADS))));
    cudaError_t e = cluster > 8 ? cudaFuncSetAttribute(sample_rows_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) : cudaSuccess;
    if (e == cudaSuccess) {
        cudaLaunchConfig_t cfg{};
        cfg.gridDim = dim3((unsigned)p->batch * (unsigned)cluster); cfg.blockDim = dim3(SR_THREADS); cfg.stream = (cudaStream_t)stream;
        cudaLaunchAttribute at[1];
        at[0].id = cudaLaunchAttributeClusterDimension;
        at[0].val.clusterDim.x = (unsigned)cluster; at[0].val.clusterDim.y = 1; at[0].val.clusterDim.z = 1;
        cfg.attrs = at; cfg.numAttrs = 1;
        e = cudaLaunchKernelEx(&cfg, sample_rows_kernel, a);
    }
    if (e != cudaSuccess) return engine_fail(nullptr, Q3_ERR_CUDA, "q3_sample_rows: %s", cudaGetErrorString(e));
    return Q3_OK;
}
