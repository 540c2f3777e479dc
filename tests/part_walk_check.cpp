// How the keys of a batch of sequences are dealt out in equal parts (include/util/page_map.h): every unit to one part, and every walk ends, also where the
// lengths are others than those that were added up.  Compiled and run by tests/test_serving_borders_cpu.py.
#include <cstdio>
#include <cstdlib>
#include <random>
#include <vector>
#include "util/page_map.h"
using namespace gp;

#define CHECK(c) do { if (!(c)) { printf("line %d: %s\n", __LINE__, #c); return 1; } } while (0)

int main() {
    std::mt19937 rng(1);
    auto pick = [&](int lo, int hi) { return lo + (int)(rng() % (unsigned)(hi - lo + 1)); };
    for (int round = 0; round < 4000; ++round) {
        const int batch = pick(1, 20), lanes = 1 << pick(0, 4);
        std::vector<int> added(batch), units;
        long total = 0;
        for (int &u : added) total += u = pick(0, 2) ? pick(0, 9) : 0;
        if (total == 0) continue;
        const int shares = pick(1, (int)total);
        // as they were added up; shorter; longer; others
        const int kind = round % 4;
        for (int u : added) units.push_back(kind == 0 ? u : kind == 1 ? pick(0, u) : kind == 2 ? u + pick(0, 5) : pick(0, 12));
        if (kind == 1 && pick(0, 1)) units.assign(batch, 0);
        std::vector<std::vector<int>> hits(batch);  // units that a part has visited
        for (int x = 0; x < shares; ++x) {
            const int lo = part_begin(x, total, shares), hi = part_begin(x + 1, total, shares);
            CHECK(lo < hi);
            for (int u = lo; u < hi; ++u) CHECK(part_of(u, total, shares) == x);
            int from = -1;  // the sequences that are looked at
            walk_part(batch, lanes, lo, hi, [&](int b0, int unit, int &at, int &i) {
                if (b0 < 0 || b0 >= batch) std::exit(2);
                from = b0;
                for (int b = b0; b < batch && b < b0 + lanes; ++b) {
                    if (at + units[b] > unit) { i = b - b0; return true; }
                    at += units[b];
                }
                return false;
            }, [&](int b0) { from = b0; if (b0 < 0 || b0 >= batch) std::exit(3); }, [&](int b, int i, int at) {
                if (b < 0 || b >= batch || b - from != i || i < 0 || i >= lanes) std::exit(4);
                const int u0 = lo > at ? lo - at : 0, u1 = hi - at < units[b] ? hi - at : units[b];
                for (int u = u0; u < u1; ++u) hits[b].push_back(u);
                if (units[b]) {
                    const int first = part_of(at, total, shares), last = part_of(at + units[b] - 1l, total, shares);
                    if (first < 0 || last < first || last >= shares) std::exit(5);
                    if (kind == 0 && (x < first || x > last)) std::exit(6);
                }
                return units[b];
            });
        }
        if (kind == 0)
            for (int b = 0; b < batch; ++b) {
                CHECK((int)hits[b].size() == units[b]);
                for (int u = 0; u < units[b]; ++u) CHECK(hits[b][u] == u);
            }
    }
    printf("ok\n");
    return 0;
}
