/*
 * q3mk.h — C ABI of the B200 (sm_100a) Qwen3-0.6B decode / prefill engine.
 *
 * This is the boundary a host language binds.  Plain pointers and sizes only; no C++ or
 * torch types.  Every function returns Q3_OK (0) or a negative error code and never throws.
 * All pointers named "device" are CUDA device addresses on the engine's GPU; the caller owns
 * every input and output buffer, the engine owns only its scratch (allocated in q3_create).
 *
 * It replaces the reference project's host->device boundary, which is a Python class driving
 * one NVRTC-compiled kernel through the CUDA driver API:
 *     qwen3mk/kernel.py:109-233   class Megakernel (step / bind / launch / _launch)
 *     csrc/qwen3_step.cu:382-394  extern "C" __global__ qwen3_step(25 pointers)
 * Tensor layouts are the reference's (qwen3mk/kernel.py:27-50): bf16 weights in Hugging Face
 * [out, in] row-major order stacked over layers, fp32 logits, int64 tokens, bf16 K/V rows.
 *
 * Model geometry is fixed to Qwen3-0.6B per head/row: hidden 1024, 16 query heads, 8 KV heads,
 * head dim 128, FFN 3072, RoPE theta 1e6, eps 1e-6.  The layer count and vocabulary size are
 * run-time values (28 and 151936 for the real model) so that small models can be tested.
 */
#ifndef Q3MK_H
#define Q3MK_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define Q3_OK                 0
#define Q3_ERR_INVALID       (-1)  /* bad argument (message in q3_last_error)               */
#define Q3_ERR_CUDA          (-2)  /* a CUDA runtime call failed                            */
#define Q3_ERR_NOT_RESIDENT  (-3)  /* the persistent grid cannot be co-resident on the GPU  */
#define Q3_ERR_DEVICE_WAIT   (-4)  /* a bounded device-side wait gave up (see q3_status)    */
#define Q3_ERR_UNSUPPORTED   (-5)  /* valid request this build cannot serve on that path    */

/* q3_decode_args.flags */
#define Q3_F_APPEND_KV    0x1u  /* write the new K/V rows into cache slot seq_len[b], then seq_len[b] += 1 */
#define Q3_F_PATH_AUTO    0x0u  /* engine picks: persistent kernel for up to three sequences it serves (sums in the order of arrival: logits
                                   differ from run to run by about 1e-6), layered otherwise (a fixed order up to 64 sequences) */
#define Q3_F_PATH_LAYERED 0x10u /* a chain of launches: five per layer up to 64 sequences, one per phase beyond */
#define Q3_F_PATH_FUSED   0x30u /* layered, but batches of 4..64 run two launches per layer: split attention + one persistent
                                   kernel for Wo, norm, gate/up, SiLU, down, norm and the next layer's q/k/v (opt-in: measured
                                   slower than the launch chain so far) */
#define Q3_F_PATH_PERSIST 0x20u /* one persistent cooperative launch per step                              */
#define Q3_F_PATH_MASK    0xf0u
#define Q3_F_GRAPH        0x100u /* layered path: capture the step's launches into a CUDA graph and replay it on later calls with the same arguments */

typedef struct q3_engine q3_engine; /* opaque */

typedef struct q3_config {
    int32_t n_layers;       /* 28 for Qwen3-0.6B                                                 */
    int32_t vocab;          /* 151936 for Qwen3-0.6B; must be >= 1                               */
    int32_t max_batch;      /* largest q3_decode_args.batch the scratch is sized for (>= 1)      */
    int32_t max_tokens;     /* largest q3_prefill_args.n_tokens the scratch is sized for (0: no prefill) */
    int32_t grid_limit;     /* 0 = one CTA per SM; otherwise cap the persistent grid (tests)     */
    int32_t wait_limit_us;  /* patience of the persistent and the layer kernel's waits, and of q3_extend's attention, in microseconds; 0 = the default (200 ms).  Tests set it low
                               to see a wait give up.  Waits inside the tensor-core products are fixed at 200 ms, at 400 for a cluster's partial tiles */
} q3_config;

/* The 13 weight tensors, device pointers to bf16.  Replaces slots 1..13 of the reference's
 * kernel argument list (qwen3mk/kernel.py:23-24, csrc/qwen3_step.cu:383-391). */
typedef struct q3_weights {
    const void* ln1;    /* [L, 1024]          */
    const void* wq;     /* [L, 2048, 1024]    */
    const void* wk;     /* [L, 1024, 1024]    */
    const void* wv;     /* [L, 1024, 1024]    */
    const void* qn;     /* [L, 128]           */
    const void* kn;     /* [L, 128]           */
    const void* wo;     /* [L, 1024, 2048]    */
    const void* ln2;    /* [L, 1024]          */
    const void* wg;     /* [L, 3072, 1024]    */
    const void* wu;     /* [L, 3072, 1024]    */
    const void* wd;     /* [L, 1024, 3072]    */
    const void* fnorm;  /* [1024]             */
    const void* embed;  /* [vocab, 1024], also the (tied) LM head */
} q3_weights;

/* One decode step for `batch` independent sequences.  Generalises the reference's fixed
 * batch-1 / position-128 launch (qwen3mk/kernel.py:180-191): sequence b decodes position
 * seq_len[b] against seq_len[b] cached positions.  The per-sequence descriptors live in device
 * memory so that back-to-back launches need no host work. */
typedef struct q3_decode_args {
    int32_t batch;                   /* 1..max_batch                                                   */
    int32_t max_len;                 /* host-side upper bound of seq_len[b] for this call (work split) */
    uint32_t flags;                  /* Q3_F_*                                                         */
    uint32_t reserved;
    const int64_t* token;            /* device [batch]  input token ids                                */
    const uint64_t* seq_k;           /* device [batch]  address of sequence b's K cache, bf16 [L][cap_b][8][128] */
    const uint64_t* seq_v;           /* device [batch]  same for V                                     */
    const int64_t* seq_layer_stride; /* device [batch]  elements between consecutive layers (cap_b * 1024) */
    int32_t* seq_len;                /* device [batch]  cached positions = position of this token; written only with Q3_F_APPEND_KV */
    float* logits;                   /* device [batch, vocab] fp32, or NULL                            */
    int64_t* next_token;             /* device [batch]  argmax, ties -> lowest index                   */
    void* k_write;                   /* device bf16 [batch, L, 8, 128] or NULL (K after head norm + RoPE) */
    void* v_write;                   /* device bf16 [batch, L, 8, 128] or NULL                         */
} q3_decode_args;

/* Causal prefill of one prompt: replaces qwen3mk/prefill.py:46-81 (fp32 torch loop) by GPU kernels. */
typedef struct q3_prefill_args {
    int32_t n_tokens;        /* 1..max_tokens                                        */
    int32_t cache_capacity;  /* positions per layer in kcache/vcache (>= n_tokens)   */
    const int64_t* ids;      /* device [n_tokens]                                    */
    void* kcache;            /* device bf16 [L, cache_capacity, 8, 128], slots [0, n_tokens) written */
    void* vcache;            /* device bf16 [L, cache_capacity, 8, 128]              */
    float* last_logits;      /* device [vocab] fp32, logits of the last position, or NULL */
    int64_t* next_token;     /* device [1] argmax of last_logits, or NULL            */
} q3_prefill_args;

/* Create an engine on CUDA device `device` (makes it current).  Replaces Megakernel.__init__
 * (qwen3mk/kernel.py:120-162): occupancy check, scratch, sync words. */
int q3_create(int device, const q3_config* cfg, q3_engine** out);

/* Free the engine's scratch.  Safe on NULL. */
void q3_destroy(q3_engine* e);

/* Record the weight pointers used by later calls (borrowed, never written).  Replaces the
 * pointer marshalling of Megakernel.step / bind (qwen3mk/kernel.py:185-188,203-206).  When a pointer of the seven
 * layer matrices differs from the last call's, the persistent kernel's packed copy is rebuilt: a kernel on the legacy
 * default stream between two cudaDeviceSynchronize (device-wide waits, once per weight set). */
int q3_set_weights(q3_engine* e, const q3_weights* w);

/* The persistent kernel streams an engine-owned re-layout of the seven layer matrices (built by
 * q3_set_weights, about 0.9 GB for the full model) and rebuilds it only when a weight POINTER
 * changes.  A caller that rewrites weights in place calls this before the next q3_set_weights.
 * No counterpart in the reference, which reads the caller's tensors directly. */
int q3_invalidate_weights(q3_engine* e);

/* Tensor parallelism over 2, 4 or 8 GPUs of one node, one process and one engine per GPU.  Rank r then owns query
 * heads [r 16/size, ..), kv heads [r 8/size, ..), FFN rows [r 3072/size, ..) and, for the LM head, words
 * [r vocab/size, ..); every rank keeps the whole residual stream.  The two per-layer sums over ranks (after the output
 * projection and after the down projection) are red instructions from every rank's CTAs straight into every rank's
 * accumulators over NVLink, fused into the phases that produce the partial sums; the grid barrier spans all ranks; the
 * arg-max is settled through per-rank mailboxes.  Peer memory is only ever written (red / st), never read.
 *   q3_tp_export: 64 bytes identifying this engine's state allocation (a CUDA IPC handle); the host exchanges them.
 *   q3_tp_attach: map the `size` handles (64 bytes each, in rank order; this rank's own entry is ignored) and switch
 *                 the engine to its share.  Call q3_set_weights afterwards (the FULL tensors: the engine packs its
 *                 share).  size = 1 switches tensor parallelism off again.
 * While attached, q3_decode serves batch 1 with up to 255 cached positions on the persistent path; every rank must
 * enqueue the same step (the kernels wait for one another, bounded by the wait limit).  Outputs: next_token on every
 * rank; logits only for the rank's words; k_write / v_write (and the appended cache rows) only for the rank's kv heads.
 * The reference is single-GPU (qwen3mk/kernel.py:120-131); no counterpart. */
int q3_tp_export(q3_engine* e, void* handle);
int q3_tp_attach(q3_engine* e, int32_t rank, int32_t size, const void* handles);

/* RoPE table: device fp32 [n_positions][128], row p = cos(p * f_0..f_63) then sin(p * f_0..f_63),
 * f_i = 1e6^(-2i/128).  Generalises the reference's single-position table
 * (qwen3mk/kernel.py:102-106).  Any address a float may have serves; the persistent kernel
 * only takes a 16-byte aligned table, its sequences take the launch chain otherwise.  Borrowed. */
int q3_set_rope(q3_engine* e, const float* table, int32_t n_positions);

/* Enqueue one decode step on `stream` (a cudaStream_t; NULL = default stream).  No host sync.
 * Replaces Megakernel._launch (qwen3mk/kernel.py:231-233). */
int q3_decode(q3_engine* e, const q3_decode_args* a, void* stream);

/* Enqueue a causal prefill on `stream`. */
int q3_prefill(q3_engine* e, const q3_prefill_args* a, void* stream);

/* One layered decode step WITHOUT an engine and without any device allocation, for callers that may
 * not call cudaMalloc where they decode (a plugin inside another runtime's memory budget, a process
 * whose device memory is fully pre-carved).  It has no counterpart in the reference.  The scratch is a
 * device array inside the library (about 0.4 MB per GPU, held until the process exits), which limits a
 * call to Q3_NOALLOC_MAX_BATCH sequences; larger batches are rejected with Q3_ERR_INVALID.  The first
 * call on a device looks up the array's address (make it before any stream capture).  All calls share
 * the array: do not let two calls overlap on the GPU, from one host thread or from several (the address
 * look-up itself is locked; the array is not).  `w`, `rope` and `a` are as for q3_set_weights,
 * q3_set_rope and q3_decode; only the layered path is available. */
#define Q3_NOALLOC_MAX_BATCH 2
int q3_decode_noalloc(const q3_weights* w, const float* rope, int32_t rope_positions, int32_t n_layers, int32_t vocab,
                      const q3_decode_args* a, void* stream);

/* Status of the last q3_decode_noalloc on the current device: synchronises `stream`, copies the status words
 * of the static array to `words` (up to `n`, may be NULL; same layout as q3_status) and returns Q3_OK or
 * Q3_ERR_DEVICE_WAIT (for example code 3: a token outside the vocabulary was replaced by token 0; code 5: a
 * cache longer than max_len).  Every q3_decode_noalloc clears the words when it starts, so read them before
 * the next call.  Allocates nothing.  No counterpart in the reference. */
int q3_noalloc_status(void* stream, uint32_t* words, int32_t n);

/* out[t, n] = (resid[t, n] +) sum_k w[n, k] * x[t, k] on the tensor cores (tcgen05 / TMEM / TMA): w bf16
 * [n_rows, K] row-major (n_rows a multiple of 128, K of 64), x fp32 [n_tok, K], out and resid fp32
 * [n_tok, n_rows] (resid may be NULL or alias out).  x is split into `nsplit` bf16 planes (1: rounded to
 * bf16, 3: exact to fp32) in the caller's `planes` buffer of at least nsplit * round_up(n_tok, tile) * K * 2
 * bytes, tile = 32 / 64 / 128 for n_tok <= 32 / <= 64 / more.  This is the dense product the reference's
 * prefill writes as `xn @ w.T` (qwen3mk/prefill.py:61-80), for callers with products of their own.  The engine uses the same
 * kernel for decode batches of more than 64 sequences; its prompts run on products that finish a layer's rows
 * themselves.  One plane and at least 256 tokens take a persistent kernel that nothing else uses.  Allocates nothing. */
int q3_linear_tc(const void* w, const float* x, float* out, const float* resid, int32_t n_rows, int32_t n_tok, int32_t K,
                 int32_t nsplit, void* planes, int64_t planes_bytes, void* stream);

/* Sample one token per row from fp32 logits [batch, vocab] on the device: keep the `top_k` largest logits of a row
 * (0 = all; ties at the k-th value are all kept), weigh them by exp((logit - max) / temperature) and return the first
 * index whose cumulative weight exceeds uniform[row] * total, in index order.  `uniform` is a device array of `batch`
 * numbers in [0, 1) drawn by the caller (so that a seed reproduces a run); temperature <= 0 or top_k == 1 returns the
 * arg-max (ties -> lowest index) and ignores `uniform`.  `out_tokens` (device int64 [batch]) may be the token buffer
 * of the next q3_decode, so that a sampled stream needs no host round trip.  Allocates nothing, no host sync.
 * The reference stops at greedy decoding and hands the fp32 logits to the caller for this step
 * (csrc/qwen3_step.cu:175, qwen3mk/kernel.py:44-50). */
int q3_sample(const float* logits, int32_t batch, int32_t vocab, float temperature, int32_t top_k,
              const float* uniform, int64_t* out_tokens, void* stream);

/* Sample one token per row with parameters of the row's own: weights w = exp((logit - max) / temperature); keep the top_k largest logits (0 or at least
 * vocab = all; ties at the k-th value are all kept); of these the most likely words until their weights reach top_p times the sum of the
 * kept ones (equal words: the lowest index first; 1 or more = all, 0 = the first); of these the words with w >= min_p (0 = all; the most
 * likely word is always kept); return the first index whose inclusive sum of kept weights exceeds uniform[row] * total, in index order.  The
 * arrays (device, [batch]) may be NULL: then the number beside them serves all rows.  temperature <= 0, top_k == 1 or min_p > 1, and rows that have no draw (a NaN
 * or an infinite maximum among the logits, a uniform number outside [0, 1)) give the arg-max (ties -> lowest index).  Logits of -inf are never
 * drawn; values that no parameter may have (a NaN, a negative top_k or min_p) switch that filter off, a negative top_p is 0, a temperature that is NaN gives the arg-max.  Row r begins at logits + r * row_stride.  The same
 * logits and numbers draw the same words on every run.  Allocates nothing, no host sync.  q3_sample, with one temperature and one top_k for all rows, sums in fp32. */
typedef struct q3_sample_rows_args {
    const float* logits;         /* device [batch][row_stride] fp32, vocab words a row */
    int64_t row_stride;          /* >= vocab, or 0: many draws from one row            */
    const float* temperatures;   /* device [batch] or NULL                             */
    const int32_t* top_ks;
    const float* top_ps;
    const float* min_ps;
    const float* uniform;        /* device [batch], in [0, 1)                          */
    int64_t* out_tokens;         /* device [batch]                                     */
    int32_t batch;               /* 1 .. 2^20                                          */
    int32_t vocab;               /* 1 .. 2^22                                          */
    float temperature;
    int32_t top_k;
    float top_p;
    float min_p;
} q3_sample_rows_args;
int q3_sample_rows(const q3_sample_rows_args* a, void* stream);

/* ---- a pool of cache pages -------------------------------------------------------------------------------------------
 * Many sequences whose K and V rows live in pages of `page_size` positions, in any order, each sequence with a row of a
 * page table: position p of sequence b is slot p % page_size of page page_table[b][p / page_size].  An entry outside
 * 0 .. n_pages - 1 is a page that is not there: nothing is written to it, its positions are not attended.  The new tokens of a call
 * are rows of q, k and v, sequence after sequence: sequence b's are rows q_start[b] .. q_start[b + 1] - 1 and its last
 * kv_len[b] - (kv_len[b] - new) positions, i.e. its token i stands at position kv_len[b] - new + i.  A sequence may have no new token; rows
 * behind q_start[batch] belong to nobody and are left as they were.  All descriptors lie in device memory and are read
 * when the call runs: a captured call may be replayed with others.  What they say is cut down to what there is
 * (n_tokens rows, table_pages * page_size positions: a longer sequence is attended as if it ended there, and its tokens behind that are not stored), so that no
 * value reads or writes out of bounds.
 * Strides are in elements; the 128 elements of a head are contiguous, pages 16-byte aligned and strides multiples of 8 that are at
 * least 128, the same for K and V. */
#define Q3_TYPE_BF16 0
#define Q3_TYPE_FP16 1
#define Q3_TYPE_FP32 2   /* rows of q3_paged_rope only */
#define Q3_PAGED_MAX_BATCH 1024
typedef struct q3_paged {
    void* k_pages;               /* device: element (page, slot, head, dim) at page * page_stride + slot * slot_stride + head * head_stride + dim */
    void* v_pages;
    const int32_t* page_table;   /* device [batch][table_stride], table_pages entries a row */
    const int32_t* q_start;      /* device [batch + 1], ascending                     */
    const int32_t* kv_len;       /* device [batch]: positions with the new tokens     */
    int64_t page_stride, slot_stride, head_stride;
    int64_t table_stride;
    int32_t table_pages;
    int32_t n_pages;
    int32_t page_size;           /* 16, 32, 64, 128 or 256                            */
    int32_t batch;               /* 1 .. Q3_PAGED_MAX_BATCH                           */
    int32_t n_tokens;            /* rows of q, k, v and out                           */
    int32_t max_new;             /* most new tokens of a sequence, as the host knows it: chooses the kernel, bounds nothing */
    int32_t kv_heads;            /* head dim is 128                                   */
    int32_t type;                /* Q3_TYPE_BF16 or Q3_TYPE_FP16: pages, q, out of the attention */
} q3_paged;

/* Attention of the new tokens over their sequences' pages: out[t][h] = sum_j softmax_j(scale q[t][h] . k_j) v_j over the
 * positions j of t's sequence up to t's own (the new tokens' k and v rows are in the pages, see q3_paged_rope).  q_heads is
 * kv_heads times 1, 2, 4 or 8; q head h reads kv head h / (q_heads / kv_heads).  A token that sees no position, or none with a weight (all
 * scores -inf), gets zeros; a row that it does not see does not touch its result, whatever it holds.  fp32 scores, maxima, sums and
 * accumulators; the probabilities enter the product with V in the pages' type.  q and out: element (token, head, dim) at token * _token + head * _head + dim, 16-byte
 * aligned, strides multiples of 8, at least 128; their rows must not overlap (where their address ranges meet, the token strides have to be the same).  `workspace`: device, at least q3_paged_attn_workspace bytes, 16-byte aligned, for this call alone.
 * `status`: device, 4 words that are 0, or NULL: a wait inside the kernel that gives up reports there as in q3_status (the first one since they were 0) and leaves NaN
 * in the rows it could not finish.  Allocates nothing, no host sync, the same bits on every run. */
typedef struct q3_paged_attn_args {
    const void* q;
    void* out;
    int64_t q_token, q_head, out_token, out_head;
    int32_t q_heads;
    float scale;                 /* > 0, at most 1e30, usually 128^-0.5 */
    void* workspace;
    int64_t workspace_bytes;
    uint32_t* status;
} q3_paged_attn_args;
int64_t q3_paged_attn_workspace(const q3_paged* c, int32_t q_heads);   /* bytes; depends on the device, the head counts and max_new alone, negative: an error code */
int q3_paged_attn(const q3_paged* c, const q3_paged_attn_args* a, void* stream);
/* The same with the patience of the kernel's waits in microseconds (0: the default, 200 ms), as q3_config has it for an engine.  Tests set it low to see a wait give up. */
int q3_paged_attn_limited(const q3_paged* c, const q3_paged_attn_args* a, int32_t wait_limit_us, void* stream);

/* The new tokens' q, k and v rows on their way to that attention: RMS norm of every q and k head (where a gain is given), rotary embedding of its
 * first rotary_dim dims by the table row of the token's position, and the k and v rows rounded once into the slots of their pages:
 *     n = x rsqrt(mean(x^2) + eps) gain
 *     half layout:  y[i] = n[i] c[i] - n[i + r/2] s[i],   y[i + r/2] = n[i + r/2] c[i] + n[i] s[i],      i < r/2 = rotary_dim / 2
 *     interleaved:  y[2i] = n[2i] c[i] - n[2i + 1] s[i],  y[2i + 1] = n[2i + 1] c[i] + n[2i] s[i]
 * in fp32.  q, k and v: element (token, head, dim) at token * _token + head * _head + dim (they may be slices of one row), 16-byte aligned fp32 or 8-byte
 * aligned bf16 / fp16, strides multiples of 4; q_out in the pages' type, 8-byte aligned, strides multiples of 4 and at least 128; it is q itself (address, strides and type) or shares no
 * memory with q, k and v (where address ranges meet, the token strides have to be the same).  `rope`: fp32 [rope_positions][rotary_dim], a row is the cosines and then the sines of
 * rotary_dim / 2 angles (any scaling of long contexts is in the table).  A token whose position has no row gets NaN (q, k); one without a slot (no page, a position
 * behind the page table's row, or kv_len below the number of new tokens) writes no k and v.  `positions`: device [n_tokens] or NULL: rotate by these instead of the tokens' places
 * in their sequences.  q may be NULL (k and v only), and k and v both (q only).  Allocates nothing, no host sync. */
typedef struct q3_paged_rope_args {
    const void *q, *k, *v;
    void* q_out;
    int64_t q_token, q_head, k_token, k_head, v_token, v_head, out_token, out_head;
    const void *q_gain, *k_gain; /* device bf16 [128] or NULL: no norm */
    const float* rope;           /* device; NULL when rotary_dim is 0  */
    const int32_t* positions;
    int32_t q_heads;
    int32_t rows_type;           /* Q3_TYPE_* of q, k and v            */
    int32_t rope_positions;
    int32_t rotary_dim;          /* a multiple of 8, 0 .. 128          */
    int32_t interleaved;
    float eps;
} q3_paged_rope_args;
int q3_paged_rope(const q3_paged* c, const q3_paged_rope_args* a, void* stream);

/* New tokens of many sequences through the whole model over a pool of pages: prompts, chunks of prompts, known turns and single tokens side by side in one
 * call.  `pages` describes layer 0 (8 kv heads, bf16; n_tokens up to the larger of the engine's max_tokens and max_batch, which must be at least 4; batch up to
 * max_batch), layer l's pages lie l * layer_stride elements further.  The tokens' K and V rows are written into their slots; kv_len counts them already, so the
 * caller adds a sequence's new tokens to kv_len before the call.  logits [batch][vocab] and next_token [batch] are those of every sequence's last new token (a
 * sequence without one gets zeros).  Positions reach to the RoPE table's end; descriptors that say more than there is are cut down and reported by q3_status (code 5, site 1100).
 * Activations enter the products rounded to bf16, as a prompt's do; up to 64 sequences the same call gives the same bits.  `workspace`: device, q3_paged_attn_workspace(pages, 16) bytes, for this call alone.
 * No host sync, allocates nothing on the device.  A captured call may be replayed with other descriptors and tokens. */
typedef struct q3_extend_args {
    const q3_paged* pages;
    int64_t layer_stride;
    const int64_t* ids;          /* device [n_tokens]; those of rows behind q_start[batch] may be anything */
    float* logits;               /* device [batch][vocab] fp32, or NULL */
    int64_t* next_token;         /* device [batch]                    */
    void* workspace;
    int64_t workspace_bytes;
} q3_extend_args;
int q3_extend(q3_engine* e, const q3_extend_args* a, void* stream);

/* Synchronise `stream`, read the device status words and clear them.  Returns Q3_OK or
 * Q3_ERR_DEVICE_WAIT; `words` (may be NULL) receives up to `n` raw status words:
 * [0] error code, [1] where (phase id), [2] CTA index, [3] observed counter value. */
int q3_status(q3_engine* e, void* stream, uint32_t* words, int32_t n);

/* Phase tracing of the persistent kernel (the reference's trace came from an external tool:
 * README.md:174-239).  `buf` is a device buffer of n_words 64-bit words, or NULL to switch tracing
 * off.  While set and large enough (grid * (4 + 12 * n_layers) words), every persistent launch makes
 * thread 0 of CTA c store %globaltimer (ns) at buf[c * (4 + 12 L) + ev].  ev 0 = start; for layer l,
 * base = 1 + 12 l: +0 Q activations staged, +1 Q done, +2 K/V rows requested, +3 F q/k/v prepared,
 * +4 F scores done, +5 F head output ready, +6 F done (attention delta sent), +7 attention delta complete,
 * +8 GD activations staged, +9 GD hid ready, +10 GD done (FFN delta sent), +11 FFN delta complete; then
 * 1 + 12 L = LM-head rows done, 2 + 12 L = end.
 * Borrowed. */
int q3_set_trace(q3_engine* e, uint64_t* buf, int64_t n_words);

/* Number of kernel launches this engine has enqueued since creation. */
int64_t q3_launch_count(const q3_engine* e);

/* Persistent-grid geometry chosen at creation: CTAs, threads per CTA, dynamic smem bytes. */
int q3_grid_info(const q3_engine* e, int32_t* ctas, int32_t* threads, int32_t* smem_bytes);

/* Engine-owned scratch for tools and tests: name in {"x","qkv","attn","hid","status","persist_acc"}; returns a
 * device pointer and its size in bytes, or Q3_ERR_INVALID.  Layered steps leave the residual rows in "x" and the last layer's
 * projections in "qkv"; "attn" is written by the fused path only, "hid" by its steps of fewer than four sequences.  "persist_acc" is the persistent kernel's four delta
 * accumulators (64-bit words: contributions << 56 | fixed-point sum), all zero between launches. */
int q3_scratch(const q3_engine* e, const char* name, void** ptr, int64_t* bytes);

/* Message of the last error on this engine (or of the last failed q3_create when e == NULL). */
const char* q3_last_error(const q3_engine* e);

/* Library version string, e.g. "q3mk-b200 0.1 sm_100a". */
const char* q3_version(void);

#ifdef __cplusplus
}
#endif
#endif /* Q3MK_H */
