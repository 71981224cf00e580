// sa_paged_plan.h -- which rows and pages the operators over a paged KV cache
// touch, and how a batch's tiles are shared out, as plain arithmetic: included
// by the kernels and compiled with g++ by a CPU test that enumerates it.
#pragma once
#include <cmath>

#ifndef __CUDACC__
#define SA_HD
#else
#define SA_HD __host__ __device__
#endif

namespace sa {
namespace pg {

// Rows of a sequence that the block table can hold.
SA_HD inline int cut_len(int len, int max_pages, int page_log2) {
    const long long cap = (long long)max_pages << page_log2;
    return len < 0 ? 0 : (len > cap ? (int)cap : len);
}
SA_HD inline bool page_ok(int entry, int n_pages) { return (unsigned)entry < (unsigned)n_pages; }

// A query at position p sees row j when j <= p and (no window, or
// j > p - window, or j < sinks).  The first row of its window:
SA_HD inline int window_lo(int p, int window) { return (window > 0 && p >= window) ? p - window + 1 : 0; }

// The rows that ONE query over `len` rows sees, cut into tiles of `tk` rows
// that start at multiples of tk: tiles [0, ta) hold the first tokens, then
// tiles tb0.. hold the window; a tile that holds both is counted once.
struct Tiles {
    int len, lo, sinks, ta, tb0, n;
    SA_HD inline int row0(int i, int tk) const { return (i < ta ? i : i - ta + tb0) * tk; }
    SA_HD inline bool sees(int row) const { return row < len && (row >= lo || row < sinks); }
    // some row of [r0, r0 + n) is seen / every one is
    SA_HD inline bool any(int r0, int rows) const { return r0 < len && (r0 + rows > lo || r0 < sinks); }
    SA_HD inline bool all(int r0, int rows) const { return r0 + rows <= len && (r0 >= lo || r0 + rows <= sinks); }
};
SA_HD inline Tiles make_tiles(int len, int window, int sinks, int tk) {
    Tiles t;
    t.len = len;
    t.lo = window_lo(len - 1, window);
    if (sinks >= t.lo) t.lo = 0;                 // the first tokens reach the window: all rows are seen
    t.sinks = sinks < t.lo ? sinks : t.lo;
    t.ta = (t.sinks + tk - 1) / tk;
    t.tb0 = t.lo / tk > t.ta ? t.lo / tk : t.ta;
    const int tb1 = (int)(((long long)len + tk - 1) / tk);
    t.n = t.ta + (tb1 > t.tb0 ? tb1 - t.tb0 : 0);
    return t;
}

// The same for the query rows of one CTA of the tensor-core kernel: two slots
// of consecutive queries, the first query at position p0 and the slots' last
// ones at last[0] and last[1] (-1: the slot sees nothing).  Tiles hold every
// row that some query sees; slot x takes the first n[x] of them.
struct UnitTiles {
    Tiles t;          // t.n = max of n[]
    int n[2];
};
SA_HD inline UnitTiles make_unit(int p0, int last0, int last1, int window, int sinks, int tk) {
    UnitTiles u;
    const int last = last0 > last1 ? last0 : last1;
    u.t.len = last < 0 ? 0 : last + 1;
    u.t.lo = window_lo(p0 < 0 ? 0 : p0, window);
    if (sinks >= u.t.lo) u.t.lo = 0;
    u.t.sinks = sinks < u.t.lo ? sinks : u.t.lo;
    u.t.ta = (u.t.sinks + tk - 1) / tk;
    u.t.tb0 = u.t.lo / tk > u.t.ta ? u.t.lo / tk : u.t.ta;
    for (int x = 0; x < 2; ++x) {
        const int l = x ? last1 : last0;
        const int end = l < 0 ? 0 : l / tk + 1;
        u.n[x] = l < 0 ? 0 : u.t.ta + (end > u.t.tb0 ? end - u.t.tb0 : 0);
    }
    u.t.n = u.n[0] > u.n[1] ? u.n[0] : u.n[1];
    return u;
}

// A list of `total` tiles shared out over n CTAs (n <= total): the first tile
// of CTA c, and the CTA that a tile falls to.
SA_HD inline long long share_first(long long c, long long total, long long n) { return c * total / n; }
SA_HD inline int share_of(long long tile, long long total, long long n) {
    return (int)(((tile + 1) * n - 1) / total);
}

// Tokens [c0, c1) of a sequence, -1 for a range outside the n_tok of the token tensors;
// the units of up to `per` tokens that they are cut into.
SA_HD inline int token_count(int c0, int c1, int n_tok) { return c0 >= 0 && c1 <= n_tok && c1 >= c0 ? c1 - c0 : -1; }
SA_HD inline unsigned unit_count(int tokens, int per) { return tokens > 0 ? (unsigned)(tokens - 1) / per + 1u : 0u; }
// Adds to the units of a thread's run of sequences.  Ranges of a wrong cu_q may overlap,
// so a run counts for what keeps the block's sum in 32 bits; a right one's units, of rows
// that lie in memory, stay far below (some 2^23 at 180 GB).
SA_HD inline unsigned add_units(unsigned run, unsigned units, unsigned threads) {
    const unsigned cap = 0xffffffffu / threads;
    return run + units < cap ? run + units : cap;
}
// The sequence of [b0, b1), whose units begin at number `at`, that unit `want` >= at is in,
// and the number of that sequence's first unit; -1: none.
SA_HD inline int unit_sequence(const int* cu_q, int b0, int b1, int n_tok, int per, unsigned want, unsigned* at) {
    for (int b = b0; b < b1; ++b) {
        const unsigned u = unit_count(token_count(cu_q[b], cu_q[b + 1], n_tok), per);
        if (want - *at < u) return b;
        *at += u;
    }
    return -1;
}

// The row of token t (of n) of a sequence of `len` rows, -1 if the sequence has
// no such token (a wrong cu_q), the cache no such row or the angle table no such
// position.
SA_HD inline long long append_row(int len, int n, int t, int max_pages, int page_log2, long long pos0, long long n_pos) {
    const long long at = (long long)len - n + t;
    if (t < 0 || t >= n || at < 0 || (at >> page_log2) >= max_pages || pos0 + at >= n_pos) return -1;
    return at;
}

// A query row's softmax state: maximum (log2 units) and sum.  What a row's sums are
// multiplied by in the end: a row that sees nothing (sum 0) comes out as zeros.
struct RowState {
    float m, l;
};
SA_HD inline float row_factor(float l) { return l == 0.f ? 0.f : 1.f / l; }
// The state of a row that a kernel gave up on (an expired wait): the sum stays NaN
// through every join, whatever the weight of the state there, and so does the output.
SA_HD inline RowState given_up() { return {0.f, NAN}; }

}  // namespace pg
}  // namespace sa
