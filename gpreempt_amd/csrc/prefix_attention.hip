// Attention of a batch of sequences that begin with the same tokens, in the same pages of the cache.
//
// What they share is read once for the rows of all sequences: a tile takes a head of the cache, the rows of as many whole sequences as 128 rows hold, and one of `shares` parts of the shared
// keys (many_keys in paged_many.hpp).  What a sequence has of its own is attended to as in a step without anything shared (attend_few in paged_few.hpp, behind the first shared_len
// keys).  A sequence with a row that does not see all of the shared keys attends to everything for itself: behind what it sees may lie NaN, and a probability of 0 times that is no 0.
// Both are tiles of one launch, the shared ones first, and leave a reference, a sum and a weighted sum per row.  The parts of the shared keys are joined two by two, and whoever comes second to a
// sequence's rows, with what its own or what the shared keys come to, joins both; in one order whoever that is.
//
// Measured, on different days (32 heads of queries over 8 of 128; each sequence for itself in brackets): 64 sequences behind 8192 tokens, up to 2048 of their own, e4m3: 61 to 64 us (152) for 169 MB; 5 with 4 new
// tokens behind 131072, bf16: 143 to 146 us (397), some 100 us of it tiles of which 80 of 128 rows are there, and some 30 us in which 63 parts meet over six levels; 256 behind 16384, fp16: 124 to 134 us (1879), 520 to
// 560 TFLOP/s.  A part's result, 66 KB, is written in 2 us and read in 3.  16 sequences with up to 8 new tokens, which are 32 rows to a head, behind 16384: bf16 79 us, e4m3 68, 31 and 65 registers of a lane in scratch
// memory.  Preemptible, with nothing to stop for: 68 us (65 plain, calls one by one), 148 (147), 181 (139: more tiles than workgroups, which claim them, and 70 registers in scratch memory).
#include <algorithm>
#include "paged_few.hpp"
#include "paged_many.hpp"
#include "launch_tiles.hpp"
#include "../../include/util/join_counters.h"

namespace gp {

constexpr int PREFIX_ROWS = 64;  // of a sequence and a head of the cache, at most

struct PrefixArgs {
    FewArgs few;              // of the sequences' own keys
    const int *table;
    int shared_len;
    int rows, per_block;      // rows of a sequence; sequences of a shared tile
    int blocks, shares;
    int shared_tiles, own_x;  // tiles; parts or sequences of the own keys
    int shared_slice, own_slice;  // tiles of an XCD
    int *arrived;             // workspace: a counter for every block of rows of a sequence and head, 0 between launches
    int *met;                 // ... and one for every part of the shared keys
    float *own, *shared;      // ... what the own keys come to, for each of these; what the parts of the shared keys come to
};

// Four floats at a time of what another workgroup reads or has written within the launch: what put_shared and get_shared do, in 16 bytes (sc1: past this XCD's cache)
constexpr int PAST_XCD = 16;
__device__ __forceinline__ __amdgpu_buffer_rsrc_t shared_buffer(const float *p) { return __builtin_amdgcn_make_buffer_rsrc((void *)p, 0, 0x7FFFFFFF, 0x00020000); }
__device__ __forceinline__ void put_shared4(__amdgpu_buffer_rsrc_t to, int at, f32x4 v) { __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, v), to, at * 4, 0, PAST_XCD); }
__device__ __forceinline__ f32x4 get_shared4(__amdgpu_buffer_rsrc_t from, int at) { return __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(from, at * 4, 0, PAST_XCD)); }

// What a part of the shared keys comes to, as the threads of many_keys have it: values d .. d + 3 (d a multiple of 4) of row r, and its reference and sum
template <int D> __device__ __forceinline__ int shared_value_at(int r, int d) { return (d / 32 * 4 + d % 32 / 8) * 4 * MANY_NT + 4 * (r / 32 * 64 + d / 4 % 2 * 32 + r % 32); }
template <int D> __device__ __forceinline__ int shared_sum_at(int r) { return D / 8 * 4 * MANY_NT + 2 * (r / 32 * 64 + r % 32); }

// Joins, for `rows` rows of a block of sequences from its row row0 on, what the own keys and what the shared keys come to.  complete: (nullptr: all) which of the block's (sequence, block of
// its rows) have both.
template <typename T, int D, int NT>
__device__ __forceinline__ void join_prefix(const PrefixArgs &a, int block, int kvh, int row0, int rows, const int *complete, float *lds) {
#pragma clang fp contract(off)  // (as in attend_stretch)
    constexpr int ROWS = 16 * NT, COLS = D / 4, ITEMS = 8;  // values of a thread at a time, in fours
    const gp_paged_attention_params &p = a.few.p;
    const int tid = threadIdx.x, row_blocks = a.few.row_blocks;
    const float *shared = a.shared + ((long)block * p.cache.kv_heads + kvh) * a.shares * many_partial_floats<D>();
    const float *own = a.own + ((long)kvh * row_blocks * p.batch + block * a.per_block) * few_partial_floats<NT, D>();
    const int mates = p.batch - block * a.per_block < a.per_block ? p.batch - block * a.per_block : a.per_block;
    auto own_at = [&](int row) {  // (rows that are not there are looked up somewhere in what is: nobody uses what comes back)
        const int mate = row / a.rows, in = row - mate * a.rows;
        return (in / ROWS * p.batch + (mate < mates ? mate : 0)) * few_partial_floats<NT, D>();
    };
    f32x2 *factors = (f32x2 *)lds;                  // of the own and of the shared keys' values
    long *place = (long *)(lds + 2 * MANY_ROWS);    // where the result goes, or -1
    __syncthreads();
    for (int u = tid; u < rows; u += FEW_NT) {
        const int row = row0 + u, mate = row / a.rows, in = row - mate * a.rows, b = block * a.per_block + mate, token = in / a.few.group;
        const f32x2 x = get_shared(own + own_at(row) + ROWS * D + 2 * (in % ROWS)), y = get_shared(shared + shared_sum_at<D>(row));
        long at = -1;
        if (mate < mates && (!complete || complete[mate * row_blocks + in / ROWS])) {
            const SeqTokens s = seq_tokens(p.start, p.kv_len, b, p.tokens, p.max_new);
            if (token < s.rows) at = (s.row0 + token) * p.ld_out + ((long)kvh * a.few.group + in - token * a.few.group) * D;
        }
        place[u] = at;
        const float top = fmaxf(x[0], y[0]), base = top == -INFINITY ? 0.f : top;
        const float f = __builtin_amdgcn_exp2f(x[0] - base), g = __builtin_amdgcn_exp2f(y[0] - base), sum = fmaf(g, y[1], f * x[1]), inv = sum == 0.f ? 0.f : 1.f / sum;
        factors[u] = f32x2{f * inv, y[1] == 0.f ? -1.f : g * inv};  // (-1: none of the shared keys counts, and their sum may be NaN)
    }
    __syncthreads();
    const auto own_buffer = shared_buffer(own), shared_result = shared_buffer(shared);
    const int d = tid % COLS * 4;  // (FEW_NT is a multiple of COLS)
#pragma unroll 1
    for (int u0 = tid; u0 < rows * COLS; u0 += ITEMS * FEW_NT) {
        f32x4 x[ITEMS], y[ITEMS];
#pragma unroll
        for (int k = 0; k < ITEMS; ++k) {
            const int r = (u0 + k * FEW_NT) / COLS, row = row0 + (r < rows ? r : 0);
            x[k] = get_shared4(own_buffer, own_at(row) + row % a.rows % ROWS * D + d);
            y[k] = get_shared4(shared_result, shared_value_at<D>(row, d));
        }
#pragma unroll
        for (int k = 0; k < ITEMS; ++k) {
            const int r = (u0 + k * FEW_NT) / COLS;
            if (r >= rows || place[r] < 0) continue;
            const f32x2 f = factors[r];
            typedef T tx4 __attribute__((ext_vector_type(4)));
            tx4 out;
#pragma unroll
            for (int e = 0; e < 4; ++e) out[e] = Elem<T>::from_f(rounded(f[1] < 0.f ? f[0] * x[k][e] : fmaf(f[1], y[k][e], f[0] * x[k][e])));
            *(tx4 *)((T *)p.out + place[r] + d) = out;
        }
    }
}

// a sequence's own keys: the result waits for those of the shared keys, or joins them
template <typename T, int D, int NT> struct PrefixOut {
    static constexpr bool SKIPS = true;
    const PrefixArgs &a;
    float *lds;
    __device__ __forceinline__ void put(const FewSequence &, int b, int hr, int r, int d, f32x4 v, float top, float sum) const {
        float *slot = a.own + ((long)hr * a.few.p.batch + b) * few_partial_floats<NT, D>();
        put_shared4(shared_buffer(slot), r * D + d, v);
        if (d == 0) put_shared(slot + 16 * NT * D + 2 * r, f32x2{top, sum});
    }
    __device__ __forceinline__ void done(const FewSequence &f, int b, int hr) const {
        __shared__ int before;
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the stores above have reached the memory that all XCDs see
        __syncthreads();
        int *arrived = a.arrived + (long)hr * a.few.p.batch + b;
        if (threadIdx.x == 0) before = __hip_atomic_fetch_add(arrived, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __syncthreads();
        if (before != 1) return;
        if (threadIdx.x == 0) __hip_atomic_store(arrived, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        const int rb = hr % a.few.row_blocks, rows = f.nrows < 16 * NT ? f.nrows : 16 * NT;
        join_prefix<T, D, NT>(a, b / a.per_block, hr / a.few.row_blocks, b % a.per_block * a.rows + rb * 16 * NT, rows, nullptr, lds);
    }
};

template <typename T, int D, bool E8, int NT>
__device__ __forceinline__ void attend_shared(const PrefixArgs &a, int at, char *lds) {
#pragma clang fp contract(off)  // (as in attend_stretch)
    const gp_paged_attention_params &p = a.few.p;
    constexpr int DB = D / 32, ROWS = 16 * NT;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), l32 = lane & 31;
    const int kvh = at % p.cache.kv_heads, block = at / p.cache.kv_heads % a.blocks, share = at / p.cache.kv_heads / a.blocks;
    // ---- this lane's query ----
    const int r = wave * 32 + l32, b = block * a.per_block + r / a.rows, in = r % a.rows, token = in / a.few.group, hg = in - token * a.few.group;
    bool there = r < a.per_block * a.rows && b < p.batch;
    const SeqTokens s = seq_tokens(p.start, p.kv_len, there ? b : 0, p.tokens, p.max_new);
    // (all shared keys or none: few_sequence)
    there = there && token < s.rows && keys_seen(seq_bound(s, p.max_len, p.table_width, p.cache.page_size), s.first, p.causal) >= a.shared_len;
    const int seen = there ? a.shared_len : 0;
    const T *q = (const T *)p.q + (there ? s.row0 + token : 0) * p.ld_q + ((long)kvh * a.few.group + (there ? hg : 0)) * D;
    const int tiles = (a.shared_len + MANY_KEYS - 1) / MANY_KEYS;
    f32x16 o[DB];
    float m, l;
    many_keys<T, D, E8>(PagedKeys{p.cache, a.table, a.shared_len / p.cache.page_size, 0, kvh}, ManyRow{there, seen, q}, p.scale, a.shared_len, a.shared_len,
                        part_begin(share, tiles, a.shares), part_begin(share + 1, tiles, a.shares), lds, o, m, l);
    l += __shfl_xor(l, 32, 64);
    if (!there) { m = -INFINITY; l = 0.f; }  // (what has come together here is of no row)
    // ---- the parts' results meet two by two: whoever of a pair comes second goes on with both, in their order ----
    const long unit = (long)block * p.cache.kv_heads + kvh;
    float *slots = a.shared + unit * a.shares * many_partial_floats<D>();
    auto put = [&](int part) {
        float *to = slots + (long)part * many_partial_floats<D>();
        const auto buffer = shared_buffer(to);
#pragma unroll
        for (int i = 0; i < DB; ++i)
#pragma unroll
            for (int v = 0; v < 16; v += 4) put_shared4(buffer, (4 * i + v / 4) * 4 * MANY_NT + 4 * tid, f32x4{o[i][v], o[i][v + 1], o[i][v + 2], o[i][v + 3]});
        put_shared(to + D / 8 * 4 * MANY_NT + 2 * tid, f32x2{m, l});
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the stores have reached the memory that all XCDs see
    };
    __shared__ int before;
    int at_level = share, parts = a.shares;  // (a result's place is that of its first part)
    for (int level = 0; parts > 1; ++level, at_level /= 2, parts = (parts + 1) / 2) {
        if ((at_level ^ 1) >= parts) continue;  // (nobody to meet)
        put(at_level << level);
        __syncthreads();
        int *met = a.met + unit * a.shares + (at_level / 2 << (level + 1)) + (1 << level);  // (the place of the pair's second part: each is second once)
        if (tid == 0) before = __hip_atomic_fetch_add(met, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __syncthreads();
        if (before == 0) return;
        if (tid == 0) __hip_atomic_store(met, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        const float *other = slots + ((long)(at_level ^ 1) << level) * many_partial_floats<D>();
        const auto buffer = shared_buffer(other);
        f32x4 x[D / 8];
#pragma unroll
        for (int i = 0; i < D / 8; ++i) x[i] = get_shared4(buffer, i * 4 * MANY_NT + 4 * tid);
        const f32x2 y = get_shared(other + D / 8 * 4 * MANY_NT + 2 * tid);
        const float top = fmaxf(m, y[0]), base = top == -INFINITY ? 0.f : top;
        const float f = __builtin_amdgcn_exp2f(m - base), g = __builtin_amdgcn_exp2f(y[0] - base);
        const bool first = at_level % 2 == 0;
        m = top;
        // (a sum of two products, the second's rounded first)
        l = first ? fmaf(f, l, g * y[1]) : fmaf(g, y[1], f * l);
#pragma unroll
        for (int i = 0; i < DB; ++i)
#pragma unroll
            for (int v = 0; v < 16; ++v) {
                const float mine = o[i][v], theirs = x[4 * i + v / 4][v % 4];
                o[i][v] = first ? fmaf(f, mine, g * theirs) : fmaf(g, theirs, f * mine);
            }
        __syncthreads();  // (`before` has been read)
    }
    put(0);
    // ---- the blocks of rows of which this was the last result ----
    __shared__ int complete[MANY_ROWS];
    __syncthreads();
    const int row_blocks = a.few.row_blocks, mates = a.per_block * row_blocks;  // (at most MANY_ROWS)
    bool last = false;
    if (tid < mates) {
        const int mate = block * a.per_block + tid / row_blocks, rb = tid % row_blocks;
        if (mate < p.batch && seq_tokens(p.start, p.kv_len, mate, p.tokens, p.max_new).rows * a.few.group > rb * ROWS) {
            int *arrived = a.arrived + (long)(kvh * row_blocks + rb) * p.batch + mate;
            last = __hip_atomic_fetch_add(arrived, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == 1;
            if (last) __hip_atomic_store(arrived, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
        complete[tid] = last;
    }
    if (__syncthreads_or(last)) join_prefix<T, D, NT>(a, block, kvh, 0, a.per_block * a.rows, complete, (float *)lds);
}

template <int D, int NT> constexpr size_t prefix_lds_bytes() { return std::max(many_lds_bytes<D>(), few_lds_floats<NT, D>() * sizeof(float)); }

template <typename T, int D, bool E8, int NT, int LOOP = LOOP_ANY>
__global__ __launch_bounds__(FEW_NT, 2) void prefix_kernel(PrefixArgs a, BlpArgs blp) {
    static_assert(FEW_NT == MANY_NT, "tiles of both kinds in one launch");
    extern __shared__ __attribute__((aligned(16))) unsigned char prefix_lds[];
    tiles<LOOP>(blp, [&](TileIdx claimed) {
        const TileIdx t = dealt_tile<LOOP>(blp, claimed);
        // (an XCD has neighbouring tiles: an eighth of both kinds each, the shared ones first; through counters they are dealt out, or one of an XCD's would have all the shared ones: 256 sequences behind
        // 16384, fp16, preemptible, 337 -> 181 us)
        const int slice = a.shared_slice + a.own_slice, xcd = t.x / slice, j = t.x - xcd * slice;
        if (j < a.shared_slice) {
            if (j * 8 + xcd < a.shared_tiles) attend_shared<T, D, E8, NT>(a, j * 8 + xcd, (char *)prefix_lds);
            return;
        }
        const int heads = a.few.row_blocks * a.few.p.cache.kv_heads, at = (j - a.shared_slice) * 8 + xcd;
        if (at >= heads * a.own_x) return;
        attend_few<T, D, E8, NT>(a.few, TileIdx{at / heads, at % heads, 0}, (float *)prefix_lds, PrefixOut<T, D, NT>{a, (float *)prefix_lds});
    });
}

// in front of everything else, whatever the launch: so one workspace serves launches of any sizes
static size_t prefix_counter_bytes() { return prefix_counters(device_cus()).bytes; }

struct PrefixPlan {
    PrefixArgs a;
    bool shared;  // or as if nothing were
    int nt;
    long tiles;
    size_t work_bytes;
};

static int plan_prefix(const gp_prefix_attention_params *p, PrefixPlan *pl) {
    GP_REQUIRE(p, "null prefix_attention params");
    *pl = PrefixPlan{};
    const gp_paged_attention_params &q = p->attention;
    if (int rc = paged_work_bytes(&q, prefix_counter_bytes(), &pl->work_bytes)) return rc;
    GP_REQUIRE(p->shared_len >= 0 && p->shared_len % q.cache.page_size == 0, "prefix_attention: shared_len must be whole pages");
    GP_REQUIRE(p->shared_len == 0 || p->shared_table, "prefix_attention: where are the shared pages?");
    PrefixArgs &a = pl->a;
    FewArgs &few = a.few;
    few.p = q;
    few.group = q.heads / q.cache.kv_heads;
    if (!q.start) few.p.max_new = 1;
    if (few.p.scale == 0.f) few.p.scale = 1.f;
    const long rows = (long)few.p.max_new * few.group;
    pl->nt = rows <= 16 ? 1 : 2;
    few.row_blocks = (int)((rows + 16 * pl->nt - 1) / (16 * pl->nt));
    const long heads = (long)few.row_blocks * q.cache.kv_heads;
    // Once for all, or for each sequence as if nothing were shared: the first has some 10 to 30 us of parts that meet in front of it, more for more keys, the second reads (batch - 1) times what is shared once more,
    // from caches where it is small.  Us, once / each (up to 100 own tokens, one new), around the border of 8 heads of 128 (32 of queries), e4m3, 1024 shared tokens: 64 sequences 25.5 / 25.3, 96 26 / 36; 4096: 16
    // sequences 30 / 23, 24 31 / 32, 32 32 / 33, 48 34 / 49; 16384: 8 sequences 40 / 36, 12 40 / 53; fp16, 1024: 32 sequences 26 / 17, 48 26 / 26, 64 27 / 29; 16384: 4 sequences 42 / 35, 6 42 / 54; 2 heads of 128 (32 of
    // queries), fp16, 4096: 48 sequences 34 / 32, 64 34 / 33, 96 38 / 45; 12 heads of 64, bf16, where the second is slower for the same bytes: 1024: 16 sequences 17.0 / 15.4, 24 17.4 / 18.7; 4096: 8 22.8 / 23.3.
    // Of 225 measured pairs the choice costs 0.5 % on average and 15 % at most.
    GP_REQUIRE(p->shared_len <= (1 << 30), "prefix_attention: shared_len must be at most 2^30");
    GP_REQUIRE(p->variant >= GP_PREFIX_AUTO && p->variant <= GP_PREFIX_EACH, "prefix_attention: variant %d", p->variant);
    const bool can = p->shared_len > 0 && rows <= PREFIX_ROWS && heads * q.batch <= PREFIX_UNITS;
    const long reach = std::min((long)q.max_len, (long)q.table_width * q.cache.page_size);  // (what is shared behind it nobody sees)
    GP_REQUIRE(can || p->variant != GP_PREFIX_TOGETHER, "prefix_attention: together only behind shared tokens, up to %d query rows of a sequence to a head of the cache and %d blocks of 16 or 32 of them", PREFIX_ROWS, PREFIX_UNITS);
    const double megabytes = 0x1p-19 * p->shared_len * q.cache.kv_heads * q.cache.head_dim * (q.cache.dtype == GP_E4M3 ? 1 : 2) * (q.cache.head_dim == 64 ? 2.5 : 1);
    pl->shared = can && reach >= p->shared_len && (p->variant == GP_PREFIX_AUTO ? (q.batch - 1) * megabytes >= std::min(150 + 10 * megabytes, 280.) : p->variant == GP_PREFIX_TOGETHER);
    if (!pl->shared) return GP_SUCC;
    a.table = p->shared_table;
    a.shared_len = few.skip = p->shared_len;
    a.rows = (int)rows;
    a.per_block = MANY_ROWS / a.rows;
    a.blocks = (q.batch + a.per_block - 1) / a.per_block;
    const long units = (long)a.blocks * q.cache.kv_heads, key_tiles = (p->shared_len + MANY_KEYS - 1l) / MANY_KEYS;
    // Own keys: a tile for each sequence, or in equal parts, two per compute unit, where there are few sequences or long ones.  Us, a tile each / parts (8 heads of 128, 512 of a sequence's tiles fill the chip
    // once), up to 2048 own keys behind 8192 shared ones, e4m3: 16 sequences 39 / 38, 32 47 / 43, 48 55 / 53, 63 60 / 61, 64 63 / 69, 80 62 / 76; behind 4096 63 65 / 65; up to 4096 own keys 63 sequences 101 / 88,
    // 64 88 / 86; behind 4096 up to 512 own keys 48 sequences 35.8 / 35.
    // A sequence that does not see all of what is shared has keys of its own from the first on: where that may be more than a tile of the others has, its keys are dealt out in parts, one for each compute unit,
    // behind the others' tiles.  (A tile is not stopped half-way, and reads 25 to 30 GB/s.  Us, in one tile / in parts (8 heads of 128), of which
    // none / one / eight end 100 to 1000 tokens within what is shared: 64 sequences behind 8192, e4m3, 71 / 103 / 141 and 71 / 68 / 74; 64 behind 32768 79 / 244 / 478 and 76 / 84 / 179; 8 behind 131072, bf16, one: 1623
    // and 229)
    const int unit = q.cache.dtype == GP_E4M3 ? few_unit<true>() : few_unit<false>();
    const long most = std::max(1l, (reach - p->shared_len + unit - 1) / unit), whole = heads * q.batch < 2l * device_cus() ? 4 : 16;
    const long all = std::max(most, (std::min(reach, p->shared_len + few.p.max_new - 1l) + unit - 1) / unit);  // of a sequence that ends within what is shared, or begins there
    a.own_x = q.batch;
    if (most > whole) a.own_x = few.shares = (int)std::min(std::max(1l, 2l * device_cus() / heads), all * q.batch);
    else if (all > whole) {
        few.whole = (int)whole;
        few.shares = (int)std::min(std::max(1l, device_cus() / heads), all * q.batch);
        a.own_x += few.shares;
    }
    // Shared tiles: one to a compute unit, beside the sequences' own, whose loads then have their arithmetic to hide behind, or two where the shared keys are most of the work.  Us, one / two (8 heads of 128), with
    // 4, 8, 16 and 32 tiles of shared keys to a tile of own ones, or to half a compute unit: 63 sequences of up to 100 own keys, e4m3, 39 / 46, 51 / 53, 73 / 71; 256 of up to 316 78 / 89, 119 / 117, 203 / 183,
    // 385 / 322; 64 of up to 2048 63 / 72, 62 / 75, 80 / 91, 125 / 120; fp16 96 / 104, 86 / 107, 108 / 127, 149 / 157; 256 of up to 1000 141 / 167, 171 / 206, 265 / 270, 471 / 417.
    const long own_tiles = std::max(heads * (few.whole ? q.batch : a.own_x), 2l * device_cus()), per_unit = units * key_tiles <= (9 + most) * own_tiles ? 1 : 2;
    // (two to a compute unit: a place is left for the workgroup that reads the flag, or a part would wait for it: 5 sequences with 4 new tokens behind 131072, bf16, preemptible, 176 -> 148 us, plain 144 level)
    a.shares = (int)std::max(1l, std::min((per_unit * device_cus() - (per_unit == 2 ? kXcds : 0)) / units, key_tiles / 4));
    a.shared_tiles = (int)(units * a.shares);
    a.shared_slice = (a.shared_tiles + 7) / 8;
    a.own_slice = (int)((heads * a.own_x + 7) / 8);
    pl->tiles = 8l * a.shared_slice + 8l * a.own_slice;
    GP_REQUIRE(pl->tiles < (1L << 31), "prefix_attention: too large");
    const size_t part = (size_t)16 * pl->nt * (q.cache.head_dim + 2) * sizeof(float), many = (size_t)(q.cache.head_dim / 2 + 2) * MANY_NT * sizeof(float);
    char *at = (char *)q.work;
    auto take = [&](size_t bytes) { char *x = at + pl->work_bytes; pl->work_bytes += join_aligned(bytes); return x; };
    const PrefixCounters counters = prefix_counters(device_cus());
    few.arrived = (int *)(at + counters.parts);  // (parts of the own keys, and of the shared ones: at most two to a compute unit where there are any)
    a.arrived = (int *)(at + counters.arrived);
    a.met = (int *)(at + counters.met);
    pl->work_bytes = counters.bytes;
    a.own = (float *)take(heads * q.batch * part);
    a.shared = (float *)take((size_t)a.shared_tiles * many);
    few.partial = (float *)take(few.shares > 1 ? (size_t)heads * few.shares * 2 * part : 0);
    return GP_SUCC;
}

}  // namespace gp

using namespace gp;

extern "C" int gp_prefix_attention_work_bytes(const gp_prefix_attention_params *p, size_t *bytes) {
    PrefixPlan pl;
    if (int rc = plan_prefix(p, &pl)) return rc;
    GP_REQUIRE(bytes, "prefix_attention: no place for the size");
    *bytes = pl.work_bytes;
    return GP_SUCC;
}

extern "C" int gp_launch_prefix_attention(const gp_prefix_attention_params *p, const gp_preempt_ctx *ctx, gp_stream s, gp_launch_info *info) {
    PrefixPlan pl;
    if (int rc = plan_prefix(p, &pl)) return rc;
    if (!pl.shared) return launch_paged(&p->attention, prefix_counter_bytes(), ctx, s, info);
    const gp_paged_attention_params &q = p->attention;
    GP_REQUIRE(q.work && aligned16(q.work) && q.work_bytes >= pl.work_bytes, "prefix_attention: needs a workspace of %zu bytes, 16-byte aligned", pl.work_bytes);
    switch (q.cache.head_dim * 8 + (q.cache.dtype == GP_E4M3) * 4 + (q.dtype == GP_F16) * 2 + (pl.nt == 2)) {
#define GP_PREFIX(T, F16, D, E8, NT) case D * 8 + E8 * 4 + F16 * 2 + (NT == 2): return launch_tiles(GP_KSET(prefix_kernel<T, D, E8, NT), (int)pl.tiles, 1, ctx, s, info, pl.a, prefix_lds_bytes<D, NT>(), 1, FEW_NT);
#define GP_PREFIX_BOTH(D, E8, NT) GP_PREFIX(_Float16, 1, D, E8, NT) GP_PREFIX(__bf16, 0, D, E8, NT)
        GP_PREFIX_BOTH(64, 0, 1) GP_PREFIX_BOTH(64, 0, 2) GP_PREFIX_BOTH(64, 1, 1) GP_PREFIX_BOTH(64, 1, 2)
        GP_PREFIX_BOTH(128, 0, 1) GP_PREFIX_BOTH(128, 0, 2) GP_PREFIX_BOTH(128, 1, 1) GP_PREFIX_BOTH(128, 1, 2)
#undef GP_PREFIX_BOTH
#undef GP_PREFIX
    }
    return GP_OUTOFRANGE;
}
