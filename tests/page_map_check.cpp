// Where the tokens of a batch lie in a paged cache (include/util/page_map.h), against a walk over every token; and that nothing outside the
// arrays is named, whatever they hold.  Compiled and run by tests/test_serving_cpu.py.
#include <climits>
#include <cstdio>
#include <cstdlib>
#include <map>
#include <random>
#include <set>
#include <vector>
#include "util/page_map.h"
using namespace gp;

#define CHECK(c) do { if (!(c)) { printf("line %d: %s\n", __LINE__, #c); return 1; } } while (0)

int main() {
    std::mt19937 rng(1);
    auto pick = [&](long lo, long hi) { return lo + (long)(rng() % (unsigned long)(hi - lo + 1)); };
    const int wild[] = {INT_MIN, INT_MIN + 1, -1, 0, 1, INT_MAX - 1, INT_MAX};
    for (int round = 0; round < 20000; ++round) {
        const int P = 16 << pick(0, 3), batch = (int)pick(1, 4), width = (int)pick(1, 6), pages = (int)pick(1, 30), max_new = (int)pick(1, 200);
        const bool sane = round % 2 == 0;
        std::vector<int> start(batch + 1), len(batch), table(batch * width);
        long tokens = 0;
        for (int b = 0; b < batch; ++b) {
            const int n = (int)pick(0, 200);
            start[b] = (int)tokens;
            tokens += n;
            len[b] = (int)pick(0, 1) ? n + (int)pick(0, 300) : (int)pick(0, 400);
        }
        start[batch] = (int)tokens;
        tokens += pick(0, 3);
        for (int &e : table) e = (int)pick(-2, pages + 1);
        if (!sane) {
            for (int &v : start) if (rng() % 3 == 0) v = wild[rng() % 7];
            for (int &v : len) if (rng() % 3 == 0) v = wild[rng() % 7];
            for (int &v : table) if (rng() % 3 == 0) v = wild[rng() % 7];
            tokens = pick(1, 300);
        }
        const bool one = rng() % 4 == 0;
        if (one) tokens = batch + pick(0, 2);
        const int max_len = sane ? (int)pick(1, 600) : wild[rng() % 7];
        for (int b = 0; b < batch; ++b) {
            const SeqTokens s = seq_tokens(one ? nullptr : start.data(), len.data(), b, tokens, max_new);
            CHECK(s.rows >= 0 && s.rows <= max_new && (s.rows == 0 || (s.row0 >= 0 && s.row0 + s.rows <= tokens)));
            const long n = one ? 1 : (long)start[b + 1] - start[b], pos0 = (long)len[b] - n;
            CHECK(s.first == pos0 && s.len == len[b]);
            if (sane && !one) CHECK(s.row0 == start[b] && s.rows == (n < max_new ? n : max_new));
            const long bound = seq_bound(s, max_len, width, P);
            CHECK(bound >= 0 && bound <= (long)width * P);
            if (max_len > 0 && len[b] > 0) CHECK(bound <= max_len && bound <= len[b] && (bound == max_len || bound == len[b] || bound == (long)width * P));
            for (int causal = 0; causal < 2; ++causal)
                for (long pos : {pos0, pos0 + 1, pos0 + n - 1, bound - 1, bound, -1l}) {
                    const long seen = keys_seen(bound, pos, causal);
                    long want = bound;
                    if (causal && pos < bound) want = pos + 1 > 0 ? pos + 1 : 0;
                    CHECK(seen == (want < bound ? want : bound));
                }
            // the pages that the new tokens touch hold each of them once
            std::set<long> seen_pos;
            const int touched = pages_touched(max_new, P);
            for (int j = 0; j < touched; ++j) {
                const PageSpan p = page_span(s, j, P);
                if (p.lo >= p.hi) continue;
                CHECK(p.lo >= 0 && p.hi <= P && p.idx >= 0);
                for (int slot = p.lo; slot < p.hi; ++slot) {
                    const long pos = p.idx * P + slot;
                    CHECK(pos >= s.first && pos < s.first + s.rows && seen_pos.insert(pos).second);
                }
                CHECK(p.lo == 0 || j == 0);  // older tokens in the first one only
                const int page = page_of(table.data(), width, b, p.idx, pages);
                CHECK(page >= -1 && page < pages);
                CHECK(p.idx < width || page == -1);
                if (p.idx < width) CHECK(page == (table[b * width + p.idx] >= 0 && table[b * width + p.idx] < pages ? table[b * width + p.idx] : -1));
            }
            long places = 0;
            for (long i = 0; i < s.rows; ++i) places += s.first + i >= 0;
            CHECK((long)seen_pos.size() == places);
            for (long idx : {-1l, (long)width, LONG_MAX, LONG_MIN}) CHECK(page_of(table.data(), width, b, idx, pages) == -1);
        }
    }
    printf("ok\n");
    return 0;
}
