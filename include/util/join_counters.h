// Where the counters lie in front of a workspace in which parts of a result are joined behind a shared beginning (prefix_attention.hip): in one place whatever the launch and whatever the number of
// compute units, so that launches of either kind leave each other's counters alone.  Shared by the launcher and its check on the host.
#pragma once
#include <cstddef>

namespace gp {

constexpr size_t JOIN_ALIGN = 256;
constexpr size_t join_aligned(size_t bytes) { return (bytes + JOIN_ALIGN - 1) / JOIN_ALIGN * JOIN_ALIGN; }

constexpr int PREFIX_UNITS = 16384;  // sequences times blocks of their rows times heads, at most

struct PrefixCounters {
    size_t parts;    // of the parts of own keys, and of launches for each sequence: two for every compute unit
    size_t arrived;  // ... of blocks of rows: PREFIX_UNITS
    size_t met;      // ... of the parts of shared keys: two for every compute unit
    size_t bytes;    // of all: what lies behind them is nobody's counter
};
constexpr PrefixCounters prefix_counters(int cus) {
    PrefixCounters c{};
    c.parts = 0;
    c.arrived = c.parts + join_aligned(2 * (size_t)cus * sizeof(int));
    c.met = c.arrived + join_aligned(PREFIX_UNITS * sizeof(int));
    c.bytes = c.met + join_aligned(2 * (size_t)cus * sizeof(int));
    return c;
}

}  // namespace gp
