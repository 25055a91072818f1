// Whether two sets of rows share memory: a call that reads one while it writes the other is refused.  Plain host arithmetic, checked by brute force on the CPU.
#pragma once
#include <stdint.h>

namespace q3 {

// rows (token, head) of `width` bytes at address + token * token_stride + head * head_stride; strides not negative
struct RowSet {
    uintptr_t address;
    int64_t token_stride, head_stride;
    int tokens, heads, width;
};

enum class Meet { No, Yes, Unknown };      // Unknown: the ranges meet and the token strides differ, too much to look through

typedef __int128 WideInt;                  // (strides may be anything up to 2^40: products do not fit 64 bits)

// whether some m in lo .. hi has -below < m * step + at < above; `but_zero`: m = 0 does not count
inline bool rows_meet_step(WideInt at, WideInt step, int64_t lo, int64_t hi, int64_t below, int64_t above, bool but_zero) {
    if (step == 0) return (lo < hi || !but_zero) && at > -(WideInt)below && at < above;
    WideInt m = (-(WideInt)below - at) / step - 1;             // (at or before the first candidate: division rounds to zero)
    if (m < lo) m = lo;
    for (; m <= hi; ++m) {
        const WideInt d = m * step + at;
        if (d >= above) return false;
        if (d > -(WideInt)below && !(but_zero && m == 0)) return true;
    }
    return false;
}

inline Meet rows_meet(const RowSet& a, const RowSet& b) {
    if (a.tokens < 1 || b.tokens < 1 || a.heads < 1 || b.heads < 1) return Meet::No;
    const WideInt d = (WideInt)b.address - (WideInt)a.address;
    auto span = [](const RowSet& r) { return (WideInt)(r.tokens - 1) * r.token_stride + (WideInt)(r.heads - 1) * r.head_stride + r.width; };
    if (d >= span(a) || -d >= span(b)) return Meet::No;
    // a token stride that is not used may be anything
    const int64_t step = a.tokens > 1 ? a.token_stride : b.token_stride;
    if (a.tokens > 1 && b.tokens > 1 && a.token_stride != b.token_stride) return Meet::Unknown;
    const int64_t lo = -(int64_t)(b.tokens - 1), hi = a.tokens - 1;
    auto at = [&](WideInt heads_apart) { return rows_meet_step(heads_apart - d, step, lo, hi, a.width, b.width, false); };
    if (a.heads == 1 || b.heads == 1 || a.head_stride == b.head_stride) {
        const int64_t stride = a.heads > 1 ? a.head_stride : b.head_stride;
        for (int64_t h = -(int64_t)(b.heads - 1); h <= a.heads - 1; ++h)
            if (at((WideInt)h * stride)) return Meet::Yes;
        return Meet::No;
    }
    if ((int64_t)a.heads * b.heads > 1 << 16) return Meet::Unknown;
    for (int i = 0; i < a.heads; ++i)
        for (int j = 0; j < b.heads; ++j)
            if (at((WideInt)i * a.head_stride - (WideInt)j * b.head_stride)) return Meet::Yes;
    return Meet::No;
}

// whether rows of one set share memory with one another
inline bool rows_meet_themselves(const RowSet& r) {
    // the usual layouts: one of the dimensions within a step of the other
    auto nested = [&](int inner, int64_t step, int outer, int64_t stride) {
        return (inner <= 1 || step >= r.width) && (outer <= 1 || (WideInt)(inner - 1) * step + r.width <= stride);
    };
    if (nested(r.heads, r.head_stride, r.tokens, r.token_stride) || nested(r.tokens, r.token_stride, r.heads, r.head_stride)) return false;
    for (int64_t h = 0; h < r.heads; ++h)
        if (rows_meet_step((WideInt)h * r.head_stride, r.token_stride, -(int64_t)(r.tokens - 1), r.tokens - 1, r.width, r.width, h == 0)) return true;
    return false;
}

}  // namespace q3
