// The new tokens' q, k and v rows: head norm, rotary embedding, k and v into the pages of their sequences.
//
// A warp takes four head rows of one token, two at a time: sixteen lanes a row, each with four dims and the four that they are rotated with (half layout; what is
// not rotated is dealt out in eights).  So a rotation stays within its lane and the squares of a head meet in four shuffles.  All rows are requested before the first is used.
// Bound by bytes for many tokens, by latency for few: one launch, three dependent loads (descriptors, page, table; the rows meanwhile).  2048 tokens of 16 + 8 + 8 fp32
// heads: 50 MB in 14.4 us, 3.5 TB/s of the 6.5 that a copy reaches, some 4 us of it the launch and the first loads' chain (a lane with four neighbouring dims of a whole
// row and its partner by shuffles: 20.1; sixteen lanes a row, 8 rows a warp in blocks of 256: 17.1, of 128: 14.9; 2 rows a warp: 17.0).
#include <cuda_fp16.h>

#include "q3_engine.h"
#include "q3_paged.h"
#include "q3_rows_meet.h"

namespace q3 {

constexpr int RP_THREADS = 128, RP_ROWS = 4;          // head rows a warp takes

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
    if constexpr (TYPE == Q3_TYPE_FP32) return *reinterpret_cast<const float4*>(p);       // (not by way of the read-only cache: q_out may be q)
    const uint2 u = *reinterpret_cast<const uint2*>(p);
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
    const int lane = threadIdx.x & 31, part = lane & 15, second = lane >> 4, rows = a.q_heads + a.kv_rows, kv = a.sh.heads, warps = (rows + RP_ROWS - 1) / RP_ROWS;
    const long long w = (long long)blockIdx.x * (RP_THREADS / 32) + uniform_warp();
    const long long t = w / warps;
    if (t >= a.sh.n_tokens) return;
    const int r0 = (int)(w - t * warps) * RP_ROWS + second;
    // this lane's dims: d0 .. d0 + 3 and d1 .. d1 + 3
    const int half = a.rotary / 2, d = part * 4;
    const bool turned = a.interleaved || d < half;
    const int d0 = turned ? d : a.rotary + (d - half) * 2, d1 = a.interleaved ? d + HEAD_DIM / 2 : turned ? d + half : d0 + 4;
    constexpr int SIZE = TYPE == Q3_TYPE_FP32 ? 4 : 2;
    float4 x[RP_ROWS / 2][2];
#pragma unroll
    for (int i = 0; i < RP_ROWS / 2; ++i) {
        const int r = min(r0 + 2 * i, rows - 1);      // the rows: q heads, then k heads, then v heads
        const unsigned char* src = r < a.q_heads ? a.q + t * a.q_token + r * a.q_head : r < a.q_heads + kv ? a.k + t * a.k_token + (r - a.q_heads) * a.k_head
                                                                                      : a.v + t * a.v_token + (r - a.q_heads - kv) * a.v_head;
        x[i][0] = rp_load<TYPE>(src + d0 * SIZE); x[i][1] = rp_load<TYPE>(src + d1 * SIZE);
    }
    // the token's sequence: as many as end at or before it come before
    int b = 0;
    for (int i = 0; i < a.sh.batch; i += 32)
        b += __popc(__ballot_sync(0xffffffffu, i + lane < a.sh.batch && a.c.q_start[min(i + lane, a.sh.batch - 1) + 1] <= t));
    if (b >= a.sh.batch) return;
    const PgSeq s = pg_seq(a.sh, a.c.q_start, a.c.kv_len, b);
    if (t < s.q0 || t >= s.q0 + s.q) return;          // (before the first sequence)
    // (by kv_len as it stands: a sequence that has outgrown its page table has no slot for its last tokens, and must not write over earlier ones)
    const long long stands = (long long)max(a.c.kv_len[b], 0) - s.q + (t - s.q0);
    const int place = (int)min(stands, 0x7fffffffll);
    const int page = place >= 0 && place < a.sh.most_keys && a.kv_rows ? pg_page(a.c, b, place) : -1;
    const int pos = a.positions ? a.positions[t] : place;
    const long long slot = page < 0 ? -1 : pg_offset(a.c, page, place & ((1 << a.c.page_log) - 1), 0);
    // this lane's cosines and sines: of d0 .. d0 + 3 and their partners d1 .., or of two pairs in each; what is not rotated is multiplied by one
    float4 c = make_float4(1.f, 1.f, 1.f, 1.f), sn = make_float4(0.f, 0.f, 0.f, 0.f);
    if (pos < 0 || pos >= a.rope_positions) {
        if (a.interleaved ? d0 < a.rotary : turned) c.x = c.y = c.z = c.w = sn.x = sn.y = sn.z = sn.w = NAN;
        if (a.interleaved && d1 >= a.rotary) { c.z = c.w = 1.f; sn.z = sn.w = 0.f; }
    } else {
        const float* const tab = a.rope + (size_t)pos * a.rotary;
        if (a.interleaved) {
            if (d0 < a.rotary) { c.x = tab[d0 / 2]; c.y = tab[d0 / 2 + 1]; sn.x = tab[half + d0 / 2]; sn.y = tab[half + d0 / 2 + 1]; }
            if (d1 < a.rotary) { c.z = tab[d1 / 2]; c.w = tab[d1 / 2 + 1]; sn.z = tab[half + d1 / 2]; sn.w = tab[half + d1 / 2 + 1]; }
        } else if (turned) {
            if ((reinterpret_cast<uintptr_t>(a.rope) & 15) == 0) {
                c = *reinterpret_cast<const float4*>(tab + d); sn = *reinterpret_cast<const float4*>(tab + half + d);
            } else {
                c = make_float4(tab[d], tab[d + 1], tab[d + 2], tab[d + 3]);
                sn = make_float4(tab[half + d], tab[half + d + 1], tab[half + d + 2], tab[half + d + 3]);
            }
        }
    }
    auto gains = [&](const bf16_raw* g, int at) {     // four of them, packed
        return g ? make_uint2(g[at] | (unsigned)g[at + 1] << 16, g[at + 2] | (unsigned)g[at + 3] << 16) : make_uint2(0x3f803f80u, 0x3f803f80u);
    };
    const uint2 gq0 = gains(a.q_gain, d0), gq1 = gains(a.q_gain, d1), gk0 = gains(a.k_gain, d0), gk1 = gains(a.k_gain, d1);
#pragma unroll
    for (int i = 0; i < RP_ROWS / 2; ++i) {
        const int r = r0 + 2 * i;
        float4 y = x[i][0], z = x[i][1];
        const bool is_q = r < a.q_heads;
        if (__any_sync(0xffffffffu, r < a.q_heads + kv)) {
            float n = fmaf(y.x, y.x, fmaf(y.y, y.y, fmaf(y.z, y.z, y.w * y.w))) + fmaf(z.x, z.x, fmaf(z.y, z.y, fmaf(z.z, z.z, z.w * z.w)));
#pragma unroll
            for (int o = 8; o > 0; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
            if (r < a.q_heads + kv) {
                if (is_q ? a.q_gain != nullptr : a.k_gain != nullptr) {
                    const uint2 g0 = is_q ? gq0 : gk0, g1 = is_q ? gq1 : gk1;
                    n = rsqrtf(n / (float)HEAD_DIM + a.eps);
                    y.x = y.x * n * bf_lo(g0.x); y.y = y.y * n * bf_hi(g0.x); y.z = y.z * n * bf_lo(g0.y); y.w = y.w * n * bf_hi(g0.y);
                    z.x = z.x * n * bf_lo(g1.x); z.y = z.y * n * bf_hi(g1.x); z.z = z.z * n * bf_lo(g1.y); z.w = z.w * n * bf_hi(g1.y);
                }
                const float4 p = y, q = z;
                if (a.interleaved) {
                    if (d0 < a.rotary) {
                        y.x = fmaf(-p.y, sn.x, p.x * c.x); y.y = fmaf(p.x, sn.x, p.y * c.x);
                        y.z = fmaf(-p.w, sn.y, p.z * c.y); y.w = fmaf(p.z, sn.y, p.w * c.y);
                    }
                    if (d1 < a.rotary) {
                        z.x = fmaf(-q.y, sn.z, q.x * c.z); z.y = fmaf(q.x, sn.z, q.y * c.z);
                        z.z = fmaf(-q.w, sn.w, q.z * c.w); z.w = fmaf(q.z, sn.w, q.w * c.w);
                    }
                } else if (turned) {
                    y.x = fmaf(-q.x, sn.x, p.x * c.x); y.y = fmaf(-q.y, sn.y, p.y * c.y); y.z = fmaf(-q.z, sn.z, p.z * c.z); y.w = fmaf(-q.w, sn.w, p.w * c.w);
                    z.x = fmaf(p.x, sn.x, q.x * c.x); z.y = fmaf(p.y, sn.y, q.y * c.y); z.z = fmaf(p.z, sn.z, q.z * c.z); z.w = fmaf(p.w, sn.w, q.w * c.w);
                }
            }
        }
        if (r >= rows) continue;
        unsigned char* to;
        if (is_q) to = a.out + t * a.o_token + r * a.o_head;
        else if (slot >= 0) {
            const int h = r - a.q_heads;
            to = (h < kv ? a.c.k + h * a.c.head_bytes : a.c.v + (h - kv) * a.c.head_bytes) + slot;
        } else continue;
        *reinterpret_cast<uint2*>(to + 2 * d0) = rp_pack<BF>(y);
        *reinterpret_cast<uint2*>(to + 2 * d1) = rp_pack<BF>(z);
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
    const int esize = p->rows_type == Q3_TYPE_FP32 ? 4 : 2;
    const uintptr_t in = reinterpret_cast<uintptr_t>(p->q) | reinterpret_cast<uintptr_t>(p->k) | reinterpret_cast<uintptr_t>(p->v);
    if (in & (esize == 4 ? 15 : 7)) return bad("fp32 rows must be 16-byte aligned, 16-bit rows 8-byte aligned");
    if (reinterpret_cast<uintptr_t>(p->q_out) & 7) return bad("q_out must be 8-byte aligned");
    if ((reinterpret_cast<uintptr_t>(p->rope) | reinterpret_cast<uintptr_t>(p->positions)) & 3) return bad("rope and positions must be 4-byte aligned");
    if ((reinterpret_cast<uintptr_t>(p->q_gain) | reinterpret_cast<uintptr_t>(p->k_gain)) & 1) return bad("gains must be 2-byte aligned");
    const int64_t most = 1ll << 38;
    for (int64_t s : {p->q_token, p->q_head, p->k_token, p->k_head, p->v_token, p->v_head, p->out_token, p->out_head})
        if (s < 0 || s > most || s % 4) return bad("strides must be multiples of 4 elements, not negative");
    if (p->q && ((c->n_tokens > 1 && p->out_token < HEAD_DIM) || (p->q_heads > 1 && p->out_head < HEAD_DIM))) return bad("rows of q_out must not overlap: strides of at least 128");
    if (p->q) {
        // a warp stores a token's rows while others still read theirs: q_out is q itself, row by row, or shares nothing with what is read
        const int width = HEAD_DIM * esize;
        auto rows = [&](const void* at, int64_t token, int64_t head, int heads) { return RowSet{reinterpret_cast<uintptr_t>(at), token * esize, head * esize, c->n_tokens, heads, width}; };
        const RowSet out{reinterpret_cast<uintptr_t>(p->q_out), 2 * p->out_token, 2 * p->out_head, c->n_tokens, p->q_heads, 2 * HEAD_DIM};
        if (rows_meet_themselves(out)) return bad("rows of q_out must not overlap");
        const bool in_place = p->q_out == p->q && p->rows_type == c->type && (c->n_tokens == 1 || p->out_token == p->q_token) && (p->q_heads == 1 || p->out_head == p->q_head);
        if ((!in_place && rows_meet(rows(p->q, p->q_token, p->q_head, p->q_heads), out) != Meet::No) ||
            (p->k && (rows_meet(rows(p->k, p->k_token, p->k_head, c->kv_heads), out) != Meet::No || rows_meet(rows(p->v, p->v_token, p->v_head, c->kv_heads), out) != Meet::No)))
            return bad("q_out must not overlap k, v or q, unless it is q itself in the pages' type (where address ranges meet, token strides must be the same)");
    }
    if (!(p->eps >= 0.f)) return bad("eps must not be negative");
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
