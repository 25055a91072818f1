// Operators over a pool of cache pages: head norm + rotary rows into the pages (q3_paged_rope.cu), attention of new tokens over the pages (q3_paged_attn.cu).
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/q3mk.h"
#include "q3_paged_plan.h"

namespace q3 {

// what the kernels take of a q3_paged: one layer's pages and the descriptors of a batch
struct PagedView {
    unsigned char *k, *v;                             // page 0
    long long page_bytes, slot_bytes, head_bytes;     // from one to the next
    const int *table, *q_start, *kv_len;
    long long table_stride;
    int n_pages, page_log;
};

// the page that holds position p of sequence b, or -1: an entry outside the pool is a page that is not there
__device__ __forceinline__ int pg_page(const PagedView& c, int b, int p) {
    const int page = c.table[(long long)b * c.table_stride + (p >> c.page_log)];
    return (unsigned)page < (unsigned)c.n_pages ? page : -1;
}
__device__ __forceinline__ long long pg_offset(const PagedView& c, int page, int slot, int head) {
    return (long long)page * c.page_bytes + (long long)slot * c.slot_bytes + (long long)head * c.head_bytes;
}

// prefix[b] = units of the sequences before b, prefix[batch] = all.  Every thread of the block; ends with a barrier.
template <int THREADS>
__device__ __forceinline__ void pg_block_prefix(const PgShape& s, const int* q_start, const int* kv_len, long long* prefix, long long* warp_sum) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    long long carry = 0;
    if (tid == 0) prefix[0] = 0;
    for (int b0 = 0; b0 < s.batch; b0 += THREADS) {
        const int b = b0 + tid;
        const long long own = b < s.batch ? pg_seq_units(s, pg_seq(s, q_start, kv_len, b)) : 0;
        long long sum = own;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long v = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum += v;
        }
        if (b0 > 0) __syncthreads();                  // (warp_sum of the round before has been read)
        if (lane == 31) warp_sum[warp] = sum;
        __syncthreads();
        long long before = carry;
        for (int w = 0; w < THREADS / 32; ++w) {
            if (w < warp) before += warp_sum[w];
            carry += warp_sum[w];
        }
        if (b < s.batch) prefix[b + 1] = before + sum;
    }
    __syncthreads();
}

// checks of the arguments that both operators share; 0 or an error code (message in q3_last_error)
int paged_check(const char* who, const q3_paged* c);
PagedView paged_view(const q3_paged* c);

}  // namespace q3
