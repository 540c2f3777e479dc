// New keys and values into a paged cache, rotated by their position on the way, in 16 bits or in 8 with a scale per page and head.
//
// A tile of the first kind is one page of one head that a sequence's new tokens touch, of the keys or of the values: whoever
// sets the scale of a page has to see all of its new tokens, and nobody else writes there.  A tile of the second kind is a few tokens'
// queries.  Bound by memory: a row is read once and written once, 16 bytes per lane.
//
// Measured (32 query heads, 8 cached of 128): 8192 tokens, bf16, pages of 32: 45.5 us, 4.4 TB/s read and written (a large copy: 4.8); 6785 tokens of five sequences, fp16 into e4m3,
// pages of 64: 42 us, 3.6 TB/s, behind the barriers at which a page's threads agree on its scale; 64 sequences' single tokens, e4m3: 7.9 us, of which
// a launch is 4.5 and the rest the chain length, table, row, scale, older values.  Non-temporal loads: 40.7 us for the e4m3 prompts, but 51 for the bf16 one.
#include <algorithm>
#include "kv_cache.hpp"
#include "lanes.hpp"
#include "launch_tiles.hpp"

namespace gp {

constexpr int APPEND_NT = 256;
constexpr float LOWEST_SCALE = 0x1p-40f;

struct AppendArgs {
    gp_kv_append_params p;
    int touched;    // pages per sequence
    int head_block, head_blocks;  // heads of a tile of the first kind, and how many such blocks there are
    int kv_tiles;   // the tiles of the first kind come first
    int q_block;    // tokens of a tile of the second kind
    int q_blocks;   // ... per sequence
};

// A thread's share of a row: two runs of eight values, half of the rotated values (or half of what is behind them) apart.  In pairs of halves the runs
// are each other's partners, neighbours are in a run; either way eight angles serve sixteen values, and a row of D values is D / 16 threads' work.
struct Share {
    int at[2];
    bool rotated;
};
__device__ __forceinline__ Share share_of_row(int u, int rot, int dim) {
    Share s;
    s.rotated = 16 * u < rot;
    s.at[0] = s.rotated ? 8 * u : rot / 2 + 8 * u;
    s.at[1] = s.at[0] + (s.rotated ? rot : dim - rot) / 2;
    return s;
}
// Cosines and sines of position * inv_freq[j].  The angle is taken in turns, in 64 bits (a position of 10^6 has 20 bits in front of the point), and
// its fraction goes to the hardware's functions, which take turns: good to about 10^-6, a hundredth of half a unit of fp16.
struct Turns {
    double per_token[8];
    __device__ __forceinline__ Turns(const float *inv_freq, const Share &s, int pairs) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int j = pairs == GP_ROT_HALVES ? s.at[0] + i : s.at[i / 4] / 2 + i % 4;
            per_token[i] = s.rotated ? (double)inv_freq[j] * 0.15915494309189533577 : 0.0;
        }
    }
    __device__ __forceinline__ void at(long pos, f32x2 (&cs)[8]) const {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float f = (float)__builtin_amdgcn_fract((double)pos * per_token[i]);
            cs[i] = f32x2{__builtin_amdgcn_cosf(f), __builtin_amdgcn_sinf(f)};
        }
    }
};

template <typename T> struct Runs {
    typedef T tx8 __attribute__((ext_vector_type(8)));
    tx8 raw[2];
    __device__ __forceinline__ void load(const T *row, const Share &s) { raw[0] = *(const tx8 *)(row + s.at[0]); raw[1] = *(const tx8 *)(row + s.at[1]); }
    __device__ __forceinline__ void widen(float (&x)[16]) const {
#pragma unroll
        for (int i = 0; i < 16; ++i) x[i] = Elem<T>::to_f(raw[i / 8][i % 8]);
    }
};
__device__ __forceinline__ void rotate(float (&x)[16], const f32x2 (&cs)[8], int pairs) {
    if (pairs == GP_ROT_HALVES) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float a = x[i], b = x[8 + i];
            x[i] = rounded(fmaf(a, cs[i][0], -(b * cs[i][1])));
            x[8 + i] = rounded(fmaf(b, cs[i][0], a * cs[i][1]));
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float a = x[2 * i], b = x[2 * i + 1];
            x[2 * i] = rounded(fmaf(a, cs[i][0], -(b * cs[i][1])));
            x[2 * i + 1] = rounded(fmaf(b, cs[i][0], a * cs[i][1]));
        }
    }
}

template <typename T>
__device__ __forceinline__ void store_runs(T *row, const Share &s, const float (&x)[16]) {
    typedef T tx8 __attribute__((ext_vector_type(8)));
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        tx8 y;
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = Elem<T>::from_f(x[8 * h + i]);
        *(tx8 *)(row + s.at[h]) = y;
    }
}

// the smallest power of two that a magnitude is at most 448 = 1.75 * 2^8 times, from its exponent and mantissa, as far as pages' scales go
__device__ __forceinline__ float scale_for(float most) {
    const unsigned bits = __builtin_bit_cast(unsigned, most);
    const int k = (int)(bits >> 23) - 127 - 8 + ((bits & 0x7FFFFFu) > 0x600000u);
    return k < -40 ? LOWEST_SCALE : fminf(__builtin_bit_cast(float, (unsigned)(k + 127) << 23), MOST_SCALE);
}

// The new values of one page and head in 8 bits: the scale that they need, what the page holds on a new one, and the values.
template <int D, int PASSES>
__device__ __forceinline__ void append_e4m3(const AppendArgs &a, const PageSpan &span, int j, int page, int head, bool values, const Share &share, const float (&x)[PASSES][16], float *lds_most) {
    const gp_kv_append_params &p = a.p;
    constexpr int LANES = D / 16, ROWS = APPEND_NT / LANES;
    const int P = p.cache.page_size, n = span.hi - span.lo, r = threadIdx.x / LANES;
    const long block = ((long)page * p.cache.kv_heads + head) * P * D;
    float most = 0.f;
#pragma unroll
    for (int q = 0; q < PASSES; ++q)  // (a row that is there twice changes nothing)
        if (q * ROWS + r < n) {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const float m = fabsf(x[q][i]);
                if (m < INFINITY && m > most) most = m;
            }
        }
    // the largest magnitude of the page's new tokens
    most = max_of_wave(most);
    __syncthreads();  // (the previous tile's is still being read)
    if ((threadIdx.x & 63) == 0) lds_most[threadIdx.x >> 6] = most;
    __syncthreads();
    most = fmaxf(fmaxf(lds_most[0], lds_most[1]), fmaxf(lds_most[2], lds_most[3]));
    float *scale_at = (values ? p.cache.v_scale : p.cache.k_scale) + (long)page * p.cache.kv_heads + head;
    const float stored = span.lo ? *scale_at : 0.f;
    const float before = stored > 0.f ? within_scales(stored) : 0.f;  // (0: a scale that nobody has set)
    const float scale = most > 448.f * before || before == 0.f ? scale_for(most) : before;
    const float inv = 1.f / scale;
    unsigned char *dst = (unsigned char *)(values ? p.cache.v : p.cache.k) + block;
    __syncthreads();  // everybody has read the scale
    if (threadIdx.x == 0 && scale != stored) *scale_at = scale;
    if (scale != before) {
        // what else the page holds, on the new scale (in the first page that the sequence writes to: the others begin here)
        if (j == 0) {
            const float ratio = before * inv;
            // Loads of a thread in flight.  A few new tokens: a page of 64 times 128 in one go (64 sequences' single tokens 7.9 us, one at a time 8.3).  For more
            // rows of new tokens the registers that it takes cost more (the prompts named above 46.4 us, 42.4).
            constexpr int U = PASSES == 1 ? 4 : 1;
            const int chunks = (P - n) * (D / 8);
            for (int i0 = threadIdx.x; i0 < chunks; i0 += U * APPEND_NT) {
                u32x2 *at[U], raw[U];
#pragma unroll
                for (int k = 0; k < U; ++k) {
                    const int i = i0 + k * APPEND_NT < chunks ? i0 + k * APPEND_NT : i0, slot = i / (D / 8);
                    at[k] = (u32x2 *)(dst + (slot < span.lo ? slot : slot + n) * D + i % (D / 8) * 8);
                    raw[k] = *at[k];
                }
#pragma unroll
                for (int k = 0; k < U; ++k) {
                    if (i0 + k * APPEND_NT >= chunks) break;
                    float old[8];
                    unpack_e4m3(raw[k], old);
#pragma unroll
                    for (int e = 0; e < 8; ++e) old[e] *= ratio;
                    *at[k] = pack_e4m3(old);
                }
            }
        }
    }
#pragma unroll
    for (int q = 0; q < PASSES; ++q)
        if (q * ROWS + r < n) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float y[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) y[i] = x[q][8 * h + i] * inv;
                *(u32x2 *)(dst + (span.lo + q * ROWS + r) * D + share.at[h]) = pack_e4m3(y);
            }
        }
}

template <typename T, int D, bool E8, int PASSES>
__device__ __forceinline__ void append_page(const AppendArgs &a, int tile, float *lds_most) {
    const gp_kv_append_params &p = a.p;
    constexpr int LANES = D / 16, ROWS = APPEND_NT / LANES;  // threads to a row, rows at a time; a page is PASSES times as many at most
    const int P = p.cache.page_size;
    const bool values = tile & 1;
    int u = tile >> 1;
    const int head0 = u % a.head_blocks * a.head_block, head1 = head0 + a.head_block < p.cache.kv_heads ? head0 + a.head_block : p.cache.kv_heads;
    u /= a.head_blocks;
    const int j = u % a.touched, b = u / a.touched;
    const SeqTokens s = seq_tokens(p.start, p.kv_len, b, p.tokens, p.max_new);
    const PageSpan span = page_span(s, j, P);
    if (span.lo >= span.hi) return;
    const int r = threadIdx.x / LANES, n = span.hi - span.lo;
    const long pos0 = span.idx * P + span.lo, row0 = s.row0 + (pos0 - s.first);
    const T *src = (const T *)(values ? p.v : p.k) + row0 * p.ld_qkv;
    const int rot = values ? 0 : p.rot_dim, first = __builtin_amdgcn_readfirstlane(r);  // (of the wavefront's rows)
    const Share share = share_of_row(threadIdx.x % LANES, rot, D);
    Runs<T> raw[PASSES];
    auto load = [&](int head) {
#pragma unroll
        for (int q = 0; q < PASSES; ++q) raw[q].load(src + (long)(q * ROWS + r < n ? q * ROWS + r : n - 1) * p.ld_qkv + (long)head * D, share);
    };
    load(head0);
    const int page = page_of(p.page_table, p.table_width, b, span.idx, p.cache.pages);  // (the rows are on their way meanwhile)
    if (page < 0) return;
    f32x2 cs[PASSES][8];
    if (rot) {
        const Turns turns(p.inv_freq, share, p.rot_pairs);
#pragma unroll
        for (int q = 0; q < PASSES; ++q)
            if (q * ROWS + first < n) turns.at(pos0 + q * ROWS + r, cs[q]);
    }
    for (int head = head0; head < head1; ++head) {
        float x[PASSES][16];
#pragma unroll
        for (int q = 0; q < PASSES; ++q) raw[q].widen(x[q]);
        if (head + 1 < head1) load(head + 1);
        if (rot && share.rotated) {
#pragma unroll
            for (int q = 0; q < PASSES; ++q)
                if (q * ROWS + first < n) rotate(x[q], cs[q], p.rot_pairs);
        }
        const long block = ((long)page * p.cache.kv_heads + head) * P * D;
        if constexpr (!E8) {
            T *dst = (T *)(values ? p.cache.v : p.cache.k) + block + (long)span.lo * D;
#pragma unroll
            for (int q = 0; q < PASSES; ++q)
                if (q * ROWS + r < n) store_runs(dst + (q * ROWS + r) * D, share, x[q]);
        } else {
            append_e4m3<D, PASSES>(a, span, j, page, head, values, share, x, lds_most);
        }
    }
}

// A thread keeps its token and its place in a head, and with them its cosines and sines, over the heads.
template <typename T, int D>
__device__ __forceinline__ void rotate_queries(const AppendArgs &a, int tile) {
    const gp_kv_append_params &p = a.p;
    constexpr int LANES = D / 16, SLOTS = APPEND_NT / LANES;
    const int b = tile / a.q_blocks, i = (tile - b * a.q_blocks) * a.q_block + (int)threadIdx.x / LANES / (SLOTS / a.q_block);
    const SeqTokens s = seq_tokens(p.start, p.kv_len, b, p.tokens, p.max_new);
    if (i >= s.rows) return;
    const Share share = share_of_row(threadIdx.x % LANES, p.rot_dim, D);
    const T *src = (const T *)p.q + (s.row0 + i) * p.ld_qkv;
    T *dst = (T *)p.q_out + (s.row0 + i) * p.ld_q_out;
    f32x2 cs[8];
    if (p.rot_dim) Turns(p.inv_freq, share, p.rot_pairs).at(s.first + i, cs);
    const int step = SLOTS / a.q_block;
    constexpr int U = 4;  // heads on their way at a time
    for (int h0 = (int)threadIdx.x / LANES % step; h0 < p.heads; h0 += U * step) {
        Runs<T> raw[U];
#pragma unroll
        for (int k = 0; k < U; ++k) raw[k].load(src + (long)(h0 + k * step < p.heads ? h0 + k * step : h0) * D, share);
#pragma unroll
        for (int k = 0; k < U; ++k)
            if (h0 + k * step < p.heads) {
                float x[16];
                raw[k].widen(x);
                if (share.rotated) rotate(x, cs, p.rot_pairs);
                store_runs(dst + (long)(h0 + k * step) * D, share, x);
            }
    }
}

template <typename T, int D, bool E8, int PASSES, int LOOP = LOOP_ANY>
__global__ __launch_bounds__(APPEND_NT) void kv_append_kernel(AppendArgs a, BlpArgs blp) {
    __shared__ float lds_most[APPEND_NT / 64];
    tiles<LOOP>(blp, [&](TileIdx t) {
        if (t.x < a.kv_tiles) append_page<T, D, E8, PASSES>(a, t.x, lds_most);
        else rotate_queries<T, D>(a, t.x - a.kv_tiles);
    });
}

}  // namespace gp

using namespace gp;

extern "C" int gp_launch_kv_append(const gp_kv_append_params *p, const gp_preempt_ctx *ctx, gp_stream s, gp_launch_info *info) {
    GP_REQUIRE(p && p->kv_len && p->page_table && p->k && p->v, "null kv_append params");
    if (int rc = check_kv_cache(p->cache, p->dtype, "kv_append")) return rc;
    GP_REQUIRE(p->batch > 0 && p->tokens > 0 && p->max_new > 0 && p->table_width > 0, "kv_append: batch, tokens, max_new and table_width must be positive");
    GP_REQUIRE(p->start || p->tokens >= p->batch, "kv_append: one new token per sequence needs a row for each");
    GP_REQUIRE(!p->q || (p->q_out && p->heads > 0), "kv_append: queries need a place to go to, and heads");
    const long head_cols = (long)p->cache.kv_heads * p->cache.head_dim, q_cols = (long)p->heads * p->cache.head_dim;
    GP_REQUIRE(p->ld_qkv % 8 == 0 && p->ld_qkv >= head_cols && (!p->q || (p->ld_qkv >= q_cols && p->ld_q_out % 8 == 0 && p->ld_q_out >= q_cols)),
               "kv_append: row strides must be multiples of 8 elements that hold the heads");
    GP_REQUIRE(aligned16(p->k) && aligned16(p->v) && aligned16(p->q) && (!p->q || aligned16(p->q_out)), "kv_append: 16-byte alignment");
    GP_REQUIRE(p->q != p->q_out || !p->q || p->ld_qkv == p->ld_q_out, "kv_append: queries that are rotated in place keep their row stride");
    GP_REQUIRE(p->rot_dim >= 0 && p->rot_dim % 16 == 0 && p->rot_dim <= p->cache.head_dim && (p->rot_dim == 0 || p->inv_freq),
               "kv_append: rot_dim must be a multiple of 16 within the head, with its frequencies");
    GP_REQUIRE(p->rot_pairs == GP_ROT_HALVES || p->rot_pairs == GP_ROT_NEIGHBOURS, "kv_append: rot_pairs %d", p->rot_pairs);
    AppendArgs a{*p};
    const int max_new = p->start ? p->max_new : 1;
    a.touched = pages_touched(max_new, p->cache.page_size);
    // A tile of 16 KB of rows is long enough for what stands in front of it: smaller pages go several heads to a tile, whose cosines and sines are the
    // same, where four tiles per compute unit are left.  (8192 tokens in pages of 32, 8 heads of 128, with 32 heads of queries: 60 us with one head, 47 with two, 49 with
    // four; 6785 tokens in pages of 64, e4m3: 43 with one, 48 with two.)
    const long pages = 2l * p->batch * a.touched, page_bytes = 2l * std::min(p->cache.page_size, max_new) * p->cache.head_dim;
    for (a.head_block = 1; a.head_block < p->cache.kv_heads && page_bytes * a.head_block < 16384 && pages * p->cache.kv_heads >= 8l * a.head_block * device_cus(); a.head_block *= 2) {}
    a.head_blocks = (p->cache.kv_heads + a.head_block - 1) / a.head_block;
    const long kv_tiles = pages * a.head_blocks;
    a.q_block = max_new >= 4 ? 4 : max_new >= 2 ? 2 : 1;
    a.q_blocks = (max_new + a.q_block - 1) / a.q_block;
    const long tiles = kv_tiles + (p->q ? (long)p->batch * a.q_blocks : 0);
    GP_REQUIRE(tiles < (1L << 31), "kv_append: too large");
    a.kv_tiles = (int)kv_tiles;
    const bool e8 = p->cache.dtype == GP_E4M3, f16 = p->dtype == GP_F16;
    const int rows = APPEND_NT / (p->cache.head_dim / 16), need = (std::min(p->cache.page_size, max_new) + rows - 1) / rows, passes = need <= 2 ? need : 4;
    switch (p->cache.head_dim * 32 + passes * 4 + e8 * 2 + f16) {
#define GP_APPEND(T, F16, D, E8, N) case D * 32 + N * 4 + E8 * 2 + F16: return launch_tiles(GP_KSET(kv_append_kernel<T, D, E8, N), (int)tiles, 1, ctx, s, info, a, 0, 4, APPEND_NT);
#define GP_APPEND4(D, N) GP_APPEND(_Float16, 1, D, 0, N) GP_APPEND(__bf16, 0, D, 0, N) GP_APPEND(_Float16, 1, D, 1, N) GP_APPEND(__bf16, 0, D, 1, N)
        GP_APPEND4(64, 1) GP_APPEND4(64, 2) GP_APPEND4(128, 1) GP_APPEND4(128, 2) GP_APPEND4(128, 4)
#undef GP_APPEND4
#undef GP_APPEND
    }
    return GP_OUTOFRANGE;
}
