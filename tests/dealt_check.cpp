// dealt() of include/util/slice_map.h: a permutation, of each XCD's part by itself, in which every counter of an XCD gets its share of the heavy tiles that the part begins with, as nearly as whole
// tiles allow, and each counter's tiles stay in their order.
#include <cstdio>
#include <cstdlib>
#include <vector>
#include "util/slice_map.h"
using namespace gp;

int main() {
    long cases = 0;
    for (int groups : {1, 2, 8, 16, 32, 64})
        for (int total = 1; total <= 5000; total += total < 600 ? 1 : 97) {
            std::vector<char> seen(total, 0);
            for (int i = 0; i < total; ++i) {
                const int u = dealt(i, total, groups);
                if (u < 0 || u >= total || seen[u]) { printf("no permutation: %d of %d, %d groups -> %d\n", i, total, groups, u); return 1; }
                seen[u] = 1;
                const int q = total / kXcds, r = total % kXcds;
                auto xcd = [&](int x) { int k = 0; while (k + 1 < kXcds && x >= (k + 1) * q + (k + 1 < r ? k + 1 : r)) ++k; return k; };
                if (xcd(u) != xcd(i)) { printf("%d of %d leaves its XCD\n", i, total); return 1; }
                if (groups <= 8 && u != i) { printf("one counter to an XCD: %d of %d -> %d\n", i, total, u); return 1; }
            }
            ++cases;
        }
    // the tiles of a launch as prefix_attention.hip has them (an eighth of both kinds each, the heavy ones first), claimed by 512 workgroups through 32 counters
    for (int heavy : {8, 32, 33, 63}) for (int light : {40, 100, 256, 777}) {
        const int slice = heavy + light, total = 8 * slice, groups = 32, grid = 512;
        int least = total, most = 0;
        for (int g = 0; g < groups; ++g) {
            int n = 0, last = -1;
            for (int i = group_slice_begin(total, g, groups, grid); i < group_slice_begin(total, g + 1, groups, grid); ++i) {
                const int j = dealt(i, total, groups) % slice;
                if (j < heavy) ++n;
                if (last >= 0 && j < last && j >= heavy + 4) { printf("out of order\n"); return 1; }
                last = j;
            }
            least = n < least ? n : least;
            most = n > most ? n : most;
        }
        if (most - least > 2) { printf("%d heavy tiles of %d: %d to %d for a counter\n", heavy, slice, least, most); return 1; }
        ++cases;
    }
    printf("ok %ld\n", cases);
}
