// New tokens of many sequences through the whole model over a pool of cache pages: q3_extend.
//
// Seven launches a layer: the q/k/v product without head norms (q3_prompt.h), the paged operators (head norms, RoPE, k and v into the pages; attention over them and its
// join), then the prompt's products that know no positions (Wo, gate/up, down, each finished in its epilogue).  The activations enter the products as one bf16 plane, like a
// prompt's; the last tokens' rows enter the LM head as three.  Up to 64 sequences nothing depends on an order of arrival: the same
// call gives the same bits.
#include <cuda.h>

#include "q3_engine.h"
#include "q3_gemm_tc.h"
#include "q3_paged.h"
#include "q3_prompt.h"

namespace q3 {

// The last new token's row of every sequence, zeros for one without: as it is, and (planes) times the final norm's gain as the three bf16 planes and 32 partial sums of squares
// that the LM head of up to 64 sequences reads (q3_gemm_tc.h).  Reports descriptors that do not fit what there is (the kernels cut them down), and clears the words
// of the row arg-max.
struct LastRowsArgs {
    const float* x;
    PgShape sh;
    const int *q_start, *kv_len;
    int rope_n;
    float* out;
    const bf16_raw* gain;
    bf16_raw* planes;                 // [3][plane_rows][1024], or nullptr
    float* ssq;                       // [32][plane_rows]
    int plane_rows;
    unsigned long long* keys;
    unsigned* tickets;
    uint32_t* status;
};
__global__ void __launch_bounds__(256) last_rows_kernel(const LastRowsArgs a) {
    pdl_launch();
    pdl_wait();
    const int b = blockIdx.x, i = threadIdx.x;
    const PgSeq s = pg_seq(a.sh, a.q_start, a.kv_len, b);
    if (i == 0) {
        if (a.q_start[b] != s.q0 || a.q_start[b + 1] != s.q0 + s.q || a.kv_len[b] != s.kv || (s.q > 0 && (s.kv < s.q || s.kv > a.rope_n)))
            report(a.status, ST_BAD_LEN, 1100, (uint32_t)a.kv_len[b]);
        a.keys[b] = 0ull; a.tickets[b] = 0u;
    }
    const float4 v = s.q > 0 ? reinterpret_cast<const float4*>(a.x + (size_t)(s.q0 + s.q - 1) * HIDDEN)[i] : make_float4(0.f, 0.f, 0.f, 0.f);
    reinterpret_cast<float4*>(a.out + (size_t)b * HIDDEN)[i] = v;
    if (a.planes == nullptr) return;
    float ss = fmaf(v.x, v.x, fmaf(v.y, v.y, fmaf(v.z, v.z, v.w * v.w)));
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);      // eight threads: 32 elements
    if ((i & 7) == 0) a.ssq[(size_t)(i >> 3) * a.plane_rows + b] = ss;
    const uint2 g = reinterpret_cast<const uint2*>(a.gain)[i];
    float r[4] = {v.x * bf_lo(g.x), v.y * bf_hi(g.x), v.z * bf_lo(g.y), v.w * bf_hi(g.y)};
#pragma unroll
    for (int p = 0; p < 3; ++p) {
        bf16_raw h[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) { h[j] = f_to_bf(r[j]); r[j] -= bf_to_f(h[j]); }
        reinterpret_cast<uint2*>(a.planes + ((size_t)p * a.plane_rows + b) * HIDDEN)[i] = make_uint2((uint32_t)h[0] | (uint32_t)h[1] << 16, (uint32_t)h[2] | (uint32_t)h[3] << 16);
    }
}

}  // namespace q3

using namespace q3;
#define fail q3::engine_fail

extern "C" int q3_extend(q3_engine* e, const q3_extend_args* a, void* stream) {
    if (!e || !a) return fail(e, Q3_ERR_INVALID, "q3_extend: null argument");
    if (!e->have_weights) return fail(e, Q3_ERR_INVALID, "q3_extend: call q3_set_weights first");
    if (!e->rope) return fail(e, Q3_ERR_INVALID, "q3_extend: call q3_set_rope first");
    if (paged_check("q3_extend", a->pages) != Q3_OK) return fail(e, Q3_ERR_INVALID, "%s", q3_last_error(nullptr));
    const q3_paged& pg = *a->pages;
    const int T = pg.n_tokens, B = pg.batch, L = e->cfg.n_layers, V = e->cfg.vocab;
    if (pg.kv_heads != KV_HEADS || pg.type != Q3_TYPE_BF16) return fail(e, Q3_ERR_INVALID, "q3_extend: this model's pages are bf16 with %d kv heads", KV_HEADS);
    if (a->layer_stride < 0 || a->layer_stride % 8 || (L > 1 && a->layer_stride < HEAD_DIM)) return fail(e, Q3_ERR_INVALID, "q3_extend: layer_stride must be a multiple of 8 elements");
    if (e->cap < Q3_TC_MIN_BATCH) return fail(e, Q3_ERR_UNSUPPORTED, "q3_extend: the engine needs max_tokens or max_batch of at least %d", Q3_TC_MIN_BATCH);
    if (T < 1 || T > e->cap) return fail(e, Q3_ERR_INVALID, "q3_extend: %d tokens outside 1..%d (the larger of max_tokens and max_batch)", T, e->cap);
    if (B > e->cfg.max_batch) return fail(e, Q3_ERR_INVALID, "q3_extend: %d sequences exceed max_batch %d", B, e->cfg.max_batch);
    if (!a->ids || !a->next_token) return fail(e, Q3_ERR_INVALID, "q3_extend: ids and next_token are required");
    const cudaError_t dev = cudaSetDevice(e->device);                 // (the workspace goes by this device's SMs)
    if (dev != cudaSuccess) return fail(e, Q3_ERR_CUDA, "q3_extend: %s", cudaGetErrorString(dev));
    const int64_t need = q3_paged_attn_workspace(&pg, Q_HEADS);
    if (need < 0) return fail(e, (int)need, "q3_extend: %s", q3_last_error(nullptr));
    if (!a->workspace || a->workspace_bytes < need || (reinterpret_cast<uintptr_t>(a->workspace) & 15))
        return fail(e, Q3_ERR_INVALID, "q3_extend: workspace holds %lld bytes, %lld needed, 16-byte aligned", (long long)a->workspace_bytes, (long long)need);
    cudaStream_t st = (cudaStream_t)stream;
#define LAUNCH(n, call)                                                                                \
    do {                                                                                               \
        cudaError_t err__ = (call);                                                                    \
        e->launches += (n);                                                                            \
        if (err__ != cudaSuccess) return fail(e, Q3_ERR_CUDA, "q3_extend: %s: %s", #call, cudaGetErrorString(err__)); \
    } while (0)
    const q3_weights& w = e->w;
    auto bf = [](const void* p) { return reinterpret_cast<const bf16_raw*>(p); };
    const size_t cap = (size_t)(e->cap + 127) / 128 * 128;
    // the activation planes' room: x * gain, hidden rows and the attention's output as a prompt has them, then q
    bf16_raw* const xn = reinterpret_cast<bf16_raw*>(e->planes);
    bf16_raw *const hid = xn + cap * HIDDEN, *const attn = hid + cap * INTER, *const q = attn + cap * Q_DIM;
    static_assert(HIDDEN + INTER + Q_DIM + Q_DIM <= 3 * INTER, "they fit");
    float* const ssq = e->gate;
    int parts = PR_SSQ_PARTS;
    CUtensorMap m_xn, m_hid, m_attn;
    const uint32_t box = (uint32_t)prompt_box_rows(T);
    if (!tc_make_map(&m_xn, xn, 0, T, HIDDEN, 1, box) || !tc_make_map(&m_hid, hid, 0, T, INTER, 1, box) || !tc_make_map(&m_attn, attn, 0, T, Q_DIM, 1, box))
        return fail(e, Q3_ERR_CUDA, "q3_extend: a tensor map could not be encoded");
    LAUNCH(1, launch_prompt_embed(reinterpret_cast<const long long*>(a->ids), bf(w.embed), V, e->x, bf(w.ln1), xn, ssq, T, e->status, T, st, pg.q_start, B));
    for (int l = 0; l < L; ++l) {
        PromptGemmCall c{};
        c.T = T; c.ssq = ssq; c.ssq_ld = T; c.parts = &parts; c.status = e->status;
        PromptGemmCall g = c;
        g.kind = PR_QKV; g.K = HIDDEN; g.in = &m_xn; g.qkv = e->qkv;
        g.w[0] = bf(w.wq) + (size_t)l * Q_DIM * HIDDEN; g.w[1] = bf(w.wk) + (size_t)l * KV_DIM * HIDDEN; g.w[2] = bf(w.wv) + (size_t)l * KV_DIM * HIDDEN;
        g.qn = bf(w.qn) + (size_t)l * HEAD_DIM; g.kn = bf(w.kn) + (size_t)l * HEAD_DIM; g.rope = e->up;
        LAUNCH(1, launch_prompt_gemm(g, st));

        q3_paged pl = pg;
        pl.k_pages = static_cast<bf16_raw*>(pg.k_pages) + (size_t)l * a->layer_stride;
        pl.v_pages = static_cast<bf16_raw*>(pg.v_pages) + (size_t)l * a->layer_stride;
        q3_paged_rope_args r{};
        r.q = e->qkv; r.k = e->qkv + Q_DIM; r.v = e->qkv + Q_DIM + KV_DIM; r.q_out = q;
        r.q_token = r.k_token = r.v_token = QKV_DIM; r.q_head = r.k_head = r.v_head = r.out_head = HEAD_DIM; r.out_token = Q_DIM;
        r.q_gain = bf(w.qn) + (size_t)l * HEAD_DIM; r.k_gain = bf(w.kn) + (size_t)l * HEAD_DIM;
        r.rope = e->rope; r.rope_positions = e->rope_n; r.rotary_dim = HEAD_DIM; r.q_heads = Q_HEADS; r.rows_type = Q3_TYPE_FP32; r.eps = EPS;
        int rc = q3_paged_rope(&pl, &r, stream);
        q3_paged_attn_args t{};
        t.q = q; t.out = attn; t.q_token = t.out_token = Q_DIM; t.q_head = t.out_head = HEAD_DIM; t.q_heads = Q_HEADS; t.scale = ATTN_SCALE;
        t.workspace = a->workspace; t.workspace_bytes = a->workspace_bytes; t.status = e->status;
        if (rc == Q3_OK) rc = q3_paged_attn_limited(&pl, &t, e->cfg.wait_limit_us, stream);
        if (rc != Q3_OK) return fail(e, rc, "q3_extend: %s", q3_last_error(nullptr));
        e->launches += 3;

        PromptGemmCall o = c;
        o.kind = PR_RESID; o.K = Q_DIM; o.in = &m_attn; o.x = e->x; o.xn = xn; o.gain = bf(w.ln2) + (size_t)l * HIDDEN;
        o.w[0] = bf(w.wo) + (size_t)l * HIDDEN * Q_DIM;
        LAUNCH(1, launch_prompt_gemm(o, st));
        PromptGemmCall u = c;
        u.kind = PR_SILU; u.K = HIDDEN; u.in = &m_xn; u.hid = hid;
        u.w[0] = bf(w.wg) + (size_t)l * INTER * HIDDEN; u.w[1] = bf(w.wu) + (size_t)l * INTER * HIDDEN;
        LAUNCH(1, launch_prompt_gemm(u, st));
        PromptGemmCall d = c;
        d.kind = PR_RESID; d.K = INTER; d.in = &m_hid; d.x = e->x; d.xn = xn;
        d.gain = l + 1 < L ? bf(w.ln1) + (size_t)(l + 1) * HIDDEN : bf(w.fnorm);
        d.w[0] = bf(w.wd) + (size_t)l * HIDDEN * INTER;
        LAUNCH(1, launch_prompt_gemm(d, st));
    }
    // the last tokens' logits
    float* const rows = e->up;
    unsigned long long* const keys = reinterpret_cast<unsigned long long*>(e->pval);
    unsigned* const tickets = reinterpret_cast<unsigned*>(e->pidx);
    float* const logits = a->logits ? a->logits : e->logits_tc;
    const bool tc = B >= Q3_TC_MIN_BATCH && V % 128 == 0 && logits, fixed = tc && B <= 64;      // fixed: sums in a fixed order
    const int lt = B <= 32 ? 32 : B <= 64 ? 64 : 128, lrow = (B + lt - 1) / lt * lt;
    LastRowsArgs r{};
    r.x = e->x; r.sh.batch = B; r.sh.n_tokens = T; r.sh.most_keys = pg.table_pages * pg.page_size; r.q_start = pg.q_start; r.kv_len = pg.kv_len; r.rope_n = e->rope_n;
    r.out = rows; r.gain = bf(w.fnorm); r.planes = fixed ? xn : nullptr; r.ssq = ssq; r.plane_rows = lrow; r.keys = keys; r.tickets = tickets; r.status = e->status;
    LAUNCH(1, launch_chain(last_rows_kernel, dim3(B), dim3(256), 0, st, r));
    if (tc) {
        if (fixed) {
            LAUNCH(1, launch_lm_head(LmHeadCall{w.embed, xn, lrow, B, V, ssq, lrow, logits, e->status}, st));
        } else {
            LAUNCH(1, launch_act_split(rows, HIDDEN, HIDDEN, bf(w.fnorm), xn, lrow, 3, B, st));
            GemmTcCall c{w.embed, xn, logits, nullptr, V, V, V, B, HIDDEN, 3, lrow, e->status};
            LAUNCH(1, launch_gemm_tc(c, st));
        }
        LAUNCH(1, launch_argmax_rows(logits, V, reinterpret_cast<long long*>(a->next_token), nullptr, 0, B, st, keys, tickets));
    } else {
        GemvArgs g{};
        g.seg[0] = {bf(w.embed), V};
        g.x = rows; g.ldx = HIDDEN; g.gain = bf(w.fnorm);
        g.out = a->logits; g.ldo = V; g.n_rows = V; g.batch = B; g.pval = e->pval; g.pidx = e->pidx;
        int lm_grid = (V + 15) / 16;
        if (lm_grid > e->lm_grid) lm_grid = e->lm_grid;
        LAUNCH(1, launch_gemv(1024, EPI_LOGITS, g, lm_grid, st));
        LAUNCH(1, launch_argmax_final(e->pval, e->pidx, lm_grid, reinterpret_cast<long long*>(a->next_token), nullptr, 0, B, st));
    }
#undef LAUNCH
    return Q3_OK;
}
