// How the attention over a paged cache is dealt out to blocks.  Plain arithmetic that compiles for host and device alike, so that it can be checked on the CPU.
//
// An ITEM is (sequence, kv head, tile of new tokens); its work is the keys that the tile's last token sees, in UNITS of a fixed number of keys.
// All items' units stand in one long row (sequence by sequence, within it head by head, tile by tile) that is cut into equal runs, one a block, wherever the cuts fall:
// uneven lengths leave no block idle.  A block takes its run as SEGMENTS, each a range of one item's units.  Only a run's first and last segment can be part
// of an item: two partial results a block at most, whatever the lengths are.
#pragma once
#include <stdint.h>

#ifdef __CUDACC__
#define PG_HD __host__ __device__ __forceinline__
#else
#define PG_HD inline
#endif

namespace q3 {

constexpr int PG_MAX_BATCH = 1024;    // sequences of a call: their prefix sums lie in shared memory

struct PgShape {
    int tile_log;     // a tile is 2^tile_log new tokens,
    int unit_log;     // a unit 2^unit_log keys, at least as many
    int heads;        // kv heads
    int batch;
    int n_tokens;     // rows of q: nothing behind them is read or written
    int most_keys;    // keys a row of the page table has room for
};

struct PgSeq { int q0, q, kv; };      // first row of q, new tokens, keys

// The descriptors lie in device memory and may hold anything: what they say is cut down to what there is.
PG_HD PgSeq pg_seq(const PgShape& s, const int* q_start, const int* kv_len, int b) {
    auto clip = [](int v, int lo, int hi) { return v < lo ? lo : v > hi ? hi : v; };
    PgSeq r;
    r.q0 = clip(q_start[b], 0, s.n_tokens);
    r.q = clip(q_start[b + 1], r.q0, s.n_tokens) - r.q0;
    r.kv = clip(kv_len[b], 0, s.most_keys);
    return r;
}

PG_HD int pg_tiles(const PgShape& s, const PgSeq& q) { return (int)(((long long)q.q + (1 << s.tile_log) - 1) >> s.tile_log); }

// Tile r sees the keys before position kv - q + min((r + 1) tile, q).  (Fewer keys than new tokens: counted as if the chunk began at position 0, so that
// an item has one unit at least; what its tokens see is looked up by position.)
PG_HD long long pg_tile_units(const PgShape& s, const PgSeq& q, int r) {
    const long long c0 = q.kv > q.q ? q.kv - q.q : 0, full = (long long)(r + 1) << s.tile_log, last = full < q.q ? full : q.q;
    return (c0 + last + (1 << s.unit_log) - 1) >> s.unit_log;
}

// sum of floor(i / 2^n) over i = 0 .. y
PG_HD long long pg_floor_sum(long long y, int n) {
    const long long q = (y + 1) >> n, rem = (y + 1) & ((1ll << n) - 1);
    return ((q * (q - 1) / 2) << n) + q * rem;
}

// Units of the tiles 0 .. x - 1, all of them but possibly the last tile of the sequence full: with c0 + tile + unit - 1 = tile * a + rest,
// tile r has floor((a + r) / (unit / tile)) units.
PG_HD long long pg_units_before(const PgShape& s, const PgSeq& q, int x) {
    const long long c0 = q.kv > q.q ? q.kv - q.q : 0, a = (c0 + (1 << s.tile_log) + (1 << s.unit_log) - 1) >> s.tile_log;
    const int n = s.unit_log - s.tile_log;
    return pg_floor_sum(a + x - 1, n) - pg_floor_sum(a - 1, n);
}

PG_HD long long pg_head_units(const PgShape& s, const PgSeq& q) {
    const int t = pg_tiles(s, q);
    return t ? pg_units_before(s, q, t - 1) + pg_tile_units(s, q, t - 1) : 0;
}
PG_HD long long pg_seq_units(const PgShape& s, const PgSeq& q) { return s.heads * pg_head_units(s, q); }

// blocks that share `total` units, at least `least` a block where there are that many
PG_HD int pg_blocks(long long total, int blocks, int least) {
    const long long n = (total + least - 1) / least;
    return (int)(n < blocks ? n : blocks);
}
PG_HD long long pg_run_start(long long total, int blocks, int i) { return total * i / blocks; }     // (total < 2^53: 2^31 keys a sequence, 2^10 sequences, 2^10 blocks)
// how many blocks begin before unit x: the one that holds unit x - 1 and all before it
PG_HD int pg_runs_before(long long total, int blocks, long long x) { return (int)((x * blocks + total - 1) / total); }

struct PgSegment {
    PgSeq seq;
    int b, h, r;               // the item
    int k0, k1, units;         // its units [k0, k1) of `units`
};

// The segments of the units [at, end) in order.  prefix[b]: units of the sequences before b; prefix[batch]: all.
struct PgWalk {
    long long at, end;
    PgSegment s;

    // the item that unit `at` belongs to; nothing is left to do where false
    PG_HD bool begin(const PgShape& sh, const long long* prefix, const int* q_start, const int* kv_len, long long from, long long to) {
        at = from; end = to;
        if (at >= end) return false;
        int lo = 0, hi = sh.batch - 1;                    // the last sequence that begins at or before `at` (empty ones share a start: the last of them has units)
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (prefix[mid] <= at) lo = mid; else hi = mid - 1;
        }
        s.b = lo;
        s.seq = pg_seq(sh, q_start, kv_len, lo);
        long long off = at - prefix[lo];
        const long long w = pg_head_units(sh, s.seq);
        s.h = (int)(off / w);
        off -= s.h * w;
        int r0 = 0, r1 = pg_tiles(sh, s.seq) - 1;
        while (r0 < r1) {
            const int mid = (r0 + r1 + 1) >> 1;
            if (pg_units_before(sh, s.seq, mid) <= off) r0 = mid; else r1 = mid - 1;
        }
        s.r = r0;
        s.k0 = (int)(off - pg_units_before(sh, s.seq, r0));
        fill(sh);
        return true;
    }
    PG_HD bool next(const PgShape& sh, const int* q_start, const int* kv_len) {
        at += s.k1 - s.k0;
        if (at >= end) return false;
        s.k0 = 0;
        if (++s.r >= pg_tiles(sh, s.seq)) {
            s.r = 0;
            if (++s.h >= sh.heads) {
                s.h = 0;
                do { ++s.b; s.seq = pg_seq(sh, q_start, kv_len, s.b); } while (s.seq.q == 0);     // (units are left, so there is one)
            }
        }
        fill(sh);
        return true;
    }
    PG_HD void fill(const PgShape& sh) {
        s.units = (int)pg_tile_units(sh, s.seq, s.r);
        const long long left = end - at;
        s.k1 = s.units - s.k0 > left ? s.k0 + (int)left : s.units;
    }
    PG_HD bool whole() const { return s.k0 == 0 && s.k1 == s.units; }
};

}  // namespace q3
