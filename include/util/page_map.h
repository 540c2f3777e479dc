// Where the tokens of a batch of sequences lie in a paged cache, shared by the kernels that write and read the cache and by
// the host-side check of this arithmetic.
//
// All of it comes from device memory that a serving program writes anew for every step, so no launcher can look at it: whatever
// the arrays hold, the functions below name only rows of `tokens`, entries of the table and pages of the pool.
#pragma once
#include "slice_map.h"

namespace gp {

struct SeqTokens {
    long row0;   // its first row of new tokens
    int rows;    // of them, those that are there (0 .. max_new)
    long first;  // position of row0: length - new tokens (may be negative: such a token has no place and sees nothing)
    long len;    // tokens in the cache, the new ones included
};

// r0, r1: its first row and the one behind its last; len: tokens in the cache
GP_HD SeqTokens seq_tokens_of(long r0, long r1, int len, long tokens, int max_new) {
    SeqTokens s;
    s.row0 = r0;
    s.len = len;
    s.first = s.len - (r1 - r0);
    long n = (r1 < tokens ? r1 : tokens) - r0;
    if (n > max_new) n = max_new;
    s.rows = r0 < 0 || n < 0 ? 0 : (int)n;
    return s;
}

// start: batch + 1 row numbers, or nullptr: one new token per sequence
GP_HD SeqTokens seq_tokens(const int *start, const int *kv_len, int b, long tokens, int max_new) {
    return seq_tokens_of(start ? start[b] : b, start ? start[b + 1] : (long)b + 1, kv_len[b], tokens, max_new);
}

// the first `bound` of a sequence's tokens lie in its table and in front of max_len
GP_HD long seq_bound(const SeqTokens &s, int max_len, int table_width, int page_size) {
    const long cap = (long)table_width * page_size;
    long n = s.len < max_len ? s.len : max_len;
    if (n > cap) n = cap;
    return n < 0 ? 0 : n;
}

// how many of `bound` keys the query at position `pos` sees
GP_HD long keys_seen(long bound, long pos, int causal) {
    if (!causal || pos + 1 >= bound) return bound;
    return pos < 0 ? 0 : pos + 1;
}

// the page of entry `idx` of a sequence, or -1: there is no such entry, or it names no page of the pool
GP_HD int page_of(const int *table, long table_width, int b, long idx, int pages) {
    if (idx < 0 || idx >= table_width) return -1;
    const int e = table[(long)b * table_width + idx];
    return e >= 0 && e < pages ? e : -1;
}

// pages that at most max_new tokens in a row touch
GP_HD int pages_touched(int max_new, int page_size) { return (int)(((long)max_new + page_size - 2) / page_size) + 1; }

// The slots of the j-th page that a sequence's new tokens touch: [lo, hi) of entry idx; lo >= hi: none.
struct PageSpan { long idx; int lo, hi; };
GP_HD PageSpan page_span(const SeqTokens &s, int j, int page_size) {
    const long pos0 = s.first > 0 ? s.first : 0, end = s.first + s.rows;
    PageSpan p;
    p.idx = pos0 / page_size + j;
    const long base = p.idx * page_size;
    p.lo = base < pos0 ? (int)(pos0 - base) : 0;
    const long hi = end - base;
    p.hi = hi < 0 ? 0 : hi < page_size ? (int)hi : page_size;
    return p;
}

// All sequences' keys in equal parts: sequence b has some number of units, one sequence behind the other, `total` of them in all, and part x of `shares` (at most
// as many as units) has the units [part_begin(x), part_begin(x + 1)).
GP_HD int part_begin(long x, long total, long shares) { return (int)(x * total / shares); }
// the part that unit x is in
GP_HD int part_of(long x, long total, long shares) {
    const long part = ((x + 1) * shares - 1) / total;
    return (int)(part < shares ? part : shares - 1);
}

// The sequences that a part [lo, hi) has units of, in their order.  `lanes` of them are looked at together, and looked at anew whenever they are needed, so the lengths that
// this walk meets need not be those that `total` was added up from if somebody writes to them meanwhile: it ends with the last sequence, whatever they are.
//   find(b0, lo, at, i)  looks at the sequences from b0 on, in front of which there are `at` units: whether unit lo is among theirs; then i is which of them has it and `at` the
//                        units in front of that one, else `at` goes behind them all
//   look(b0)             looks at the sequences from b0 on
//   visit(b, i, at)      sequence b, the i-th of those looked at last, in front of which there are `at` units: its units
template <class Find, class Look, class Visit>
GP_HD void walk_part(int batch, int lanes, int lo, int hi, Find &&find, Look &&look, Visit &&visit) {
    int at = 0, i = 0, b0 = 0;
    while (!find(b0, lo, at, i))
        if ((b0 += lanes) >= batch) return;
    for (int b = b0 + i; at < hi && b < batch; ++b) {
        if (b - b0 == lanes) look(b0 += lanes);
        at += visit(b, b - b0, at);
    }
}

}  // namespace gp
