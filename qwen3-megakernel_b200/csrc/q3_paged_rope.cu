// The new tokens' q, k and v rows: head norm, rotary embedding, k and v into the pages of their sequences.
//
// A warp takes eight head rows of one token, a lane four neighbouring dims of each: all eight are requested before the first is used, the squares of a head
// meet in a warp's sum and RoPE's pairs in a shuffle (half layout: the lane rotary / 8 further; interleaved: the lane itself).  Bound by bytes for many tokens, by
// latency for few: one launch, three dependent loads (descriptors, page, rows and table meanwhile).
#include <cuda_fp16.h>

#include "q3_engine.h"
#include "q3_paged.h"

namespace q3 {

constexpr int RP_THREADS = 256, RP_ROWS = 8;          // head rows a warp takes

struct PagedRopeArgs {
    PagedView c;
    PgShape sh;
    const unsigned char *q, *k, *v;
    unsigned char* out;
    long long q_token, q_head, k_token, k_head, v_token, v_head, o_token, o_head;      // bytes
    const bf16_raw *q_gain, *k_gain;
    const float* rope;
    const int* positions;
    int q_heads, kv_rows;             // kv_rows: k and v rows of a token (0: q only)
    int rope_positions, rotary, interleaved;
    float eps;
};

template <int TYPE> __device__ __forceinline__ float4 rp_load(const unsigned char* p) {       // four elements
    if constexpr (TYPE == Q3_TYPE_FP32) return __ldg(reinterpret_cast<const float4*>(p));
    const uint2 u = __ldg(reinterpret_cast<const uint2*>(p));
    if constexpr (TYPE == Q3_TYPE_BF16) return make_float4(bf_lo(u.x), bf_hi(u.x), bf_lo(u.y), bf_hi(u.y));
    const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&u.x)), b = __half22float2(*reinterpret_cast<const __half2*>(&u.y));
    return make_float4(a.x, a.y, b.x, b.y);
}
template <bool BF> __device__ __forceinline__ uint2 rp_pack(float4 v) {
    uint2 u;
    if constexpr (BF) {
        asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(u.x) : "f"(v.y), "f"(v.x));
        asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(u.y) : "f"(v.w), "f"(v.z));
    } else {
        asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(u.x) : "f"(v.y), "f"(v.x));
        asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(u.y) : "f"(v.w), "f"(v.z));
    }
    return u;
}

template <int TYPE, bool BF>
__global__ void __launch_bounds__(RP_THREADS) paged_rope_kernel(const PagedRopeArgs a) {
    pdl_launch();
    pdl_wait();
    const int lane = threadIdx.x & 31, warps = (a.q_heads + a.kv_rows + RP_ROWS - 1) / RP_ROWS;
    const long long w = (long long)blockIdx.x * (RP_THREADS / 32) + uniform_warp();
    const long long t = w / warps;
    if (t >= a.sh.n_tokens) return;
    const int r0 = (int)(w - t * warps) * RP_ROWS;
    // the rows: q heads, then k heads, then v heads
    const int rows = a.q_heads + a.kv_rows, kv = a.sh.heads;
    float4 x[RP_ROWS];
#pragma unroll
    for (int i = 0; i < RP_ROWS; ++i) {
        const int r = min(r0 + i, rows - 1);
        const unsigned char* src = r < a.q_heads ? a.q + t * a.q_token + r * a.q_head : r < a.q_heads + kv ? a.k + t * a.k_token + (r - a.q_heads) * a.k_head
                                                                                      : a.v + t * a.v_token + (r - a.q_heads - kv) * a.v_head;
        x[i] = rp_load<TYPE>(src + lane * (TYPE == Q3_TYPE_FP32 ? 16 : 8));
    }
    // the token's sequence: as many as end at or before it come before
    int b = 0;
    for (int i = 0; i < a.sh.batch; i += 32)
        b += __popc(__ballot_sync(0xffffffffu, i + lane < a.sh.batch && a.c.q_start[min(i + lane, a.sh.batch - 1) + 1] <= t));
    if (b >= a.sh.batch) return;
    const PgSeq s = pg_seq(a.sh, a.c.q_start, a.c.kv_len, b);
    if (t < s.q0 || t >= s.q0 + s.q) return;          // (before the first sequence)
    const int place = s.kv - s.q + (int)(t - s.q0);
    const int page = place >= 0 && a.kv_rows ? pg_page(a.c, b, place) : -1;
    const int pos = a.positions ? a.positions[t] : place;
    const long long slot = page < 0 ? -1 : pg_offset(a.c, page, place & ((1 << a.c.page_log) - 1), 0);
    // this lane's cosines and sines; what is not rotated is multiplied by one
    const int half = a.rotary / 2, d = lane * 4;
    const bool turned = d < a.rotary;
    float c[4] = {1.f, 1.f, 1.f, 1.f}, sn[4] = {0.f, 0.f, 0.f, 0.f};
    if (turned) {
        const bool known = pos >= 0 && pos < a.rope_positions;
        const float* tab = a.rope + (size_t)(known ? pos : 0) * a.rotary;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int f = a.interleaved ? (d + i) >> 1 : d < half ? d + i : d + i - half;
            c[i] = known ? tab[f] : NAN;
            sn[i] = known ? tab[half + f] : NAN;
        }
    }
    const bool low = d < half;
    const int other = turned ? (low ? lane + half / 4 : lane - half / 4) : lane;
    const float q_g[4] = {a.q_gain ? bf_to_f(a.q_gain[d]) : 1.f, a.q_gain ? bf_to_f(a.q_gain[d + 1]) : 1.f, a.q_gain ? bf_to_f(a.q_gain[d + 2]) : 1.f, a.q_gain ? bf_to_f(a.q_gain[d + 3]) : 1.f};
    const float k_g[4] = {a.k_gain ? bf_to_f(a.k_gain[d]) : 1.f, a.k_gain ? bf_to_f(a.k_gain[d + 1]) : 1.f, a.k_gain ? bf_to_f(a.k_gain[d + 2]) : 1.f, a.k_gain ? bf_to_f(a.k_gain[d + 3]) : 1.f};
#pragma unroll
    for (int i = 0; i < RP_ROWS; ++i) {
        const int r = r0 + i;
        if (r >= rows) break;
        float v[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
        if (r < a.q_heads + kv) {
            const bool is_q = r < a.q_heads;
            if (is_q ? a.q_gain != nullptr : a.k_gain != nullptr) {
                const float n = rsqrtf(warp_sum(fmaf(v[0], v[0], fmaf(v[1], v[1], fmaf(v[2], v[2], v[3] * v[3])))) / (float)HEAD_DIM + a.eps);
#pragma unroll
                for (int j = 0; j < 4; ++j) v[j] = v[j] * n * (is_q ? q_g[j] : k_g[j]);
            }
            if (a.rotary) {
                float p[4];
                if (a.interleaved) { p[0] = -v[1]; p[1] = v[0]; p[2] = -v[3]; p[3] = v[2]; }
                else {
#pragma unroll
                    for (int j = 0; j < 4; ++j) { p[j] = __shfl_sync(0xffffffffu, v[j], other); if (low) p[j] = -p[j]; }
                }
                if (turned)
#pragma unroll
                    for (int j = 0; j < 4; ++j) v[j] = fmaf(p[j], sn[j], v[j] * c[j]);
            }
        }
        const uint2 u = rp_pack<BF>(make_float4(v[0], v[1], v[2], v[3]));
        if (r < a.q_heads) *reinterpret_cast<uint2*>(a.out + t * a.o_token + r * a.o_head + lane * 8) = u;
        else if (slot >= 0) {
            const int h = r - a.q_heads;
            *reinterpret_cast<uint2*>((h < kv ? a.c.k + h * a.c.head_bytes : a.c.v + (h - kv) * a.c.head_bytes) + slot + lane * 8) = u;
        }
    }
}

}  // namespace q3

using namespace q3;

extern "C" int q3_paged_rope(const q3_paged* c, const q3_paged_rope_args* p, void* stream) {
    const char* who = "q3_paged_rope";
    if (const int rc = paged_check(who, c)) return rc;
    auto bad = [&](const char* what) { return engine_fail(nullptr, Q3_ERR_INVALID, "%s: %s", who, what); };
    if (!p) return bad("null argument");
    if (c->n_tokens == 0) return Q3_OK;
    if (!p->k != !p->v) return bad("k and v come together");
    if (!p->q && !p->k) return bad("neither q nor k and v are given");
    if (p->q && (!p->q_out || p->q_heads < 1 || p->q_heads > 8192)) return bad("q needs q_out and 1 to 8192 heads");
    if (p->rows_type != Q3_TYPE_BF16 && p->rows_type != Q3_TYPE_FP16 && p->rows_type != Q3_TYPE_FP32) return bad("rows are fp32, bf16 or fp16");
    if (p->rotary_dim < 0 || p->rotary_dim > HEAD_DIM || p->rotary_dim % 8) return engine_fail(nullptr, Q3_ERR_INVALID, "%s: rotary_dim %d is not a multiple of 8 in 0..128", who, p->rotary_dim);
    if (p->rotary_dim && (!p->rope || p->rope_positions < 1)) return bad("a rotation needs a table");
    if (!(p->eps >= 0.f)) return bad("eps must not be negative");
    const int esize = p->rows_type == Q3_TYPE_FP32 ? 4 : 2;
    const uintptr_t in = reinterpret_cast<uintptr_t>(p->q) | reinterpret_cast<uintptr_t>(p->k) | reinterpret_cast<uintptr_t>(p->v);
    if (in & (esize == 4 ? 15 : 7)) return bad("fp32 rows must be 16-byte aligned, 16-bit rows 8-byte aligned");
    if (reinterpret_cast<uintptr_t>(p->q_out) & 7) return bad("q_out must be 8-byte aligned");
    if ((reinterpret_cast<uintptr_t>(p->rope) | reinterpret_cast<uintptr_t>(p->positions)) & 3) return bad("rope and positions must be 4-byte aligned");
    if ((reinterpret_cast<uintptr_t>(p->q_gain) | reinterpret_cast<uintptr_t>(p->k_gain)) & 1) return bad("gains must be 2-byte aligned");
    const int64_t most = 1ll << 38;
    for (int64_t s : {p->q_token, p->q_head, p->k_token, p->k_head, p->v_token, p->v_head, p->out_token, p->out_head})
        if (s < 0 || s > most || s % 4) return bad("strides must be multiples of 4 elements, not negative");
    PagedRopeArgs a{};
    a.c = paged_view(c);
    a.sh.heads = c->kv_heads; a.sh.batch = c->batch; a.sh.n_tokens = c->n_tokens; a.sh.most_keys = c->table_pages * c->page_size;
    a.q = static_cast<const unsigned char*>(p->q); a.k = static_cast<const unsigned char*>(p->k); a.v = static_cast<const unsigned char*>(p->v);
    a.out = static_cast<unsigned char*>(p->q_out);
    a.q_token = p->q_token * esize; a.q_head = p->q_head * esize; a.k_token = p->k_token * esize; a.k_head = p->k_head * esize;
    a.v_token = p->v_token * esize; a.v_head = p->v_head * esize; a.o_token = 2 * p->out_token; a.o_head = 2 * p->out_head;
    a.q_gain = static_cast<const bf16_raw*>(p->q_gain); a.k_gain = static_cast<const bf16_raw*>(p->k_gain);
    a.rope = p->rope; a.positions = p->positions;
    a.q_heads = p->q ? p->q_heads : 0; a.kv_rows = p->k ? 2 * c->kv_heads : 0;
    a.rope_positions = p->rope_positions; a.rotary = p->rotary_dim; a.interleaved = p->interleaved ? 1 : 0;
    a.eps = p->eps;
    const long long warps = (long long)c->n_tokens * ((a.q_heads + a.kv_rows + RP_ROWS - 1) / RP_ROWS), blocks = (warps + RP_THREADS / 32 - 1) / (RP_THREADS / 32);
    if (blocks > 0x7fffffffll) return bad("too many rows for a launch");
    auto* const kernel = c->type == Q3_TYPE_BF16
        ? (esize == 4 ? paged_rope_kernel<Q3_TYPE_FP32, true> : p->rows_type == Q3_TYPE_BF16 ? paged_rope_kernel<Q3_TYPE_BF16, true> : paged_rope_kernel<Q3_TYPE_FP16, true>)
        : (esize == 4 ? paged_rope_kernel<Q3_TYPE_FP32, false> : p->rows_type == Q3_TYPE_BF16 ? paged_rope_kernel<Q3_TYPE_BF16, false> : paged_rope_kernel<Q3_TYPE_FP16, false>);
    const cudaError_t err = launch_chain(kernel, dim3((unsigned)blocks), dim3(RP_THREADS), 0, (cudaStream_t)stream, a);
    if (err != cudaSuccess) return engine_fail(nullptr, Q3_ERR_CUDA, "%s: %s", who, cudaGetErrorString(err));
    return Q3_OK;
}
