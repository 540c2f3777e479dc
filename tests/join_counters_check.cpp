// The counters in front of a workspace (include/util/join_counters.h), for any number of compute units: room for each kind, none in another's, none behind the end.  Compiled and run by tests/test_decoders_cpu.py.
#include <cstdio>
#include "util/join_counters.h"
using namespace gp;

#define CHECK(c) do { if (!(c)) { printf("%d compute units, line %d: %s\n", cus, __LINE__, #c); return 1; } } while (0)

int main() {
    for (int cus = 1; cus <= 2048; ++cus) {
        const PrefixCounters c = prefix_counters(cus);
        const size_t two = 2 * (size_t)cus * sizeof(int);
        CHECK(c.parts == 0 && c.parts + two <= c.arrived);
        CHECK(c.arrived + PREFIX_UNITS * sizeof(int) <= c.met);
        CHECK(c.met + two <= c.bytes);
        CHECK(c.arrived % JOIN_ALIGN == 0 && c.met % JOIN_ALIGN == 0 && c.bytes % JOIN_ALIGN == 0);
        CHECK(c.bytes < c.met + two + JOIN_ALIGN);
    }
    puts("ok");
}
