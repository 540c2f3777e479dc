// New keys and values into a paged cache, rotated by their position on the way, in 16 bits or in 8 with a scale per page and head.
//
// A tile of the first kind is one page of one head that a sequence's new tokens touch, of the keys or of the values: whoever
// sets the scale of a page has to see all of its new tokens, and nobody else writes there.  A tile of the second kind is a few tokens'
// queries.  Bound by memory: a row is read once and written once, 16 bytes per lane.
#include <algorithm>
#include "kv_cache.hpp"
#include "launch_tiles.hpp"

namespace gp {

constexpr int APPEND_NT = 256;
constexpr float LOWEST_SCALE = 0x1p-40f;

struct AppendArgs {
    gp_kv_append_params p;
    int touched;    // pages per sequence
    int kv_tiles;   // the tiles of the first kind come first
    int q_block;    // tokens of a tile of the second kind
    int q_blocks;   // ... per sequence
};

// cosine and sine of position * inv_freq[j].  The angle is taken in turns, in 64 bits (a position of 10^6 has 20 bits in front of the point), and
// its fraction goes to the hardware's functions, which take turns: good to about 10^-6, a hundredth of half a unit of fp16.
__device__ __forceinline__ f32x2 turn(long pos, float inv_freq) {
    const double turns = (double)pos * ((double)inv_freq * 0.15915494309189533577);
    const float f = (float)__builtin_amdgcn_fract(turns);
    return f32x2{__builtin_amdgcn_cosf(f), __builtin_amdgcn_sinf(f)};
}

// eight values of a head, from `at` on, in fp32, rotated.  cs(j): cosine and sine of pair j of this row
template <typename T, class CS>
__device__ __forceinline__ void load_rotated(const T *row, int at, int rot, int pairs, CS &&cs, float (&x)[8]) {
    typedef T tx8 __attribute__((ext_vector_type(8)));
    const tx8 own = *(const tx8 *)(row + at);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = Elem<T>::to_f(own[i]);
    if (at >= rot) return;
    if (pairs == GP_ROT_HALVES) {
        const int half = rot / 2;
        const bool first = at < half;
        const tx8 other = *(const tx8 *)(row + (first ? at + half : at - half));
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const f32x2 c = cs((first ? at : at - half) + i);
            const float y = Elem<T>::to_f(other[i]);
            x[i] = first ? x[i] * c[0] - y * c[1] : x[i] * c[0] + y * c[1];
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const f32x2 c = cs(at / 2 + i);
            const float a = x[2 * i], b = x[2 * i + 1];
            x[2 * i] = a * c[0] - b * c[1];
            x[2 * i + 1] = b * c[0] + a * c[1];
        }
    }
}

template <typename T>
__device__ __forceinline__ void store8(T *to, const float (&x)[8]) {
    typedef T tx8 __attribute__((ext_vector_type(8)));
    tx8 y;
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = Elem<T>::from_f(x[i]);
    *(tx8 *)to = y;
}

// the smallest power of two that a magnitude is at most 448 = 1.75 * 2^8 times, from its exponent and mantissa
__device__ __forceinline__ float scale_for(float most) {
    const unsigned bits = __builtin_bit_cast(unsigned, most);
    const int k = (int)(bits >> 23) - 127 - 8 + ((bits & 0x7FFFFFu) > 0x600000u);
    return k < -40 ? LOWEST_SCALE : __builtin_bit_cast(float, (unsigned)(k + 127) << 23);
}

template <typename T, int D, bool E8>
__device__ __forceinline__ void append_page(const AppendArgs &a, int tile, float *lds_most) {
    const gp_kv_append_params &p = a.p;
    constexpr int LANES = D / 8, ROWS = APPEND_NT / LANES, PASSES = 128 / ROWS;  // lanes to a row, rows at a time, at most so many times
    const int P = p.cache.page_size;
    const bool values = tile & 1;
    int u = tile >> 1;
    const int head = u % p.cache.kv_heads;
    u /= p.cache.kv_heads;
    const int j = u % a.touched, b = u / a.touched;
    const SeqTokens s = seq_tokens(p.start, p.kv_len, b, p.tokens, p.max_new);
    const PageSpan span = page_span(s, j, P);
    if (span.lo >= span.hi) return;
    const int page = page_of(p.page_table, p.table_width, b, span.idx, p.cache.pages);
    if (page < 0) return;
    const int lane = threadIdx.x % LANES, r = threadIdx.x / LANES, n = span.hi - span.lo;
    const long pos0 = span.idx * P + span.lo, row0 = s.row0 + (pos0 - s.first);
    const T *src = (const T *)(values ? p.v : p.k) + row0 * p.ld_qkv + (long)head * D;
    const long block = ((long)page * p.cache.kv_heads + head) * P * D;
    const int rot = values ? 0 : p.rot_dim;
    float x[PASSES][8];
    float most = 0.f;
#pragma unroll
    for (int q = 0; q < PASSES; ++q) {
        const int t = q * ROWS + r;
        if (t < n) {
            const long pos = pos0 + t;
            load_rotated(src + t * p.ld_qkv, lane * 8, rot, p.rot_pairs, [&](int i) { return turn(pos, p.inv_freq[i]); }, x[q]);
            if constexpr (E8) {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float m = fabsf(x[q][i]);
                    if (m < INFINITY && m > most) most = m;
                }
            }
        }
    }
    if constexpr (!E8) {
        T *dst = (T *)(values ? p.cache.v : p.cache.k) + block + (long)span.lo * D + lane * 8;
#pragma unroll
        for (int q = 0; q < PASSES; ++q)
            if (q * ROWS + r < n) store8(dst + (q * ROWS + r) * D, x[q]);
    } else {
        // the largest magnitude of the page's new tokens
#pragma unroll
        for (int d = 1; d < 64; d *= 2) most = fmaxf(most, __shfl_xor(most, d, 64));
        __syncthreads();  // (the previous tile's is still being read)
        if ((threadIdx.x & 63) == 0) lds_most[threadIdx.x >> 6] = most;
        __syncthreads();
        most = fmaxf(fmaxf(lds_most[0], lds_most[1]), fmaxf(lds_most[2], lds_most[3]));
        float *scale_at = (values ? p.cache.v_scale : p.cache.k_scale) + (long)page * p.cache.kv_heads + head;
        float before = span.lo ? *scale_at : 0.f;
        if (!(before > 0.f && before < INFINITY)) before = 0.f;  // (a scale that nobody has set)
        const float scale = most > 448.f * before || before == 0.f ? scale_for(most) : before;
        const float inv = 1.f / scale;
        unsigned char *dst = (unsigned char *)(values ? p.cache.v : p.cache.k) + block;
        __syncthreads();  // everybody has read the scale
        if (scale != before) {
            if (threadIdx.x == 0) *scale_at = scale;
            // what else the page holds, on the new scale (in the first page that the sequence writes to: the others begin here)
            if (j == 0) {
                const float ratio = before * inv;
                for (int i = threadIdx.x; i < (P - n) * LANES; i += APPEND_NT) {
                    const int slot = i / LANES;
                    u32x2 *at = (u32x2 *)(dst + (slot < span.lo ? slot : slot + n) * D + i % LANES * 8);
                    float old[8];
                    unpack_e4m3(*at, old);
#pragma unroll
                    for (int e = 0; e < 8; ++e) old[e] *= ratio;
                    *at = pack_e4m3(old);
                }
            }
        }
#pragma unroll
        for (int q = 0; q < PASSES; ++q)
            if (q * ROWS + r < n) {
#pragma unroll
                for (int i = 0; i < 8; ++i) x[q][i] *= inv;
                *(u32x2 *)(dst + (span.lo + q * ROWS + r) * D + lane * 8) = pack_e4m3(x[q]);
            }
    }
}

template <typename T, int D>
__device__ __forceinline__ void rotate_queries(const AppendArgs &a, int tile) {
    const gp_kv_append_params &p = a.p;
    const int b = tile / a.q_blocks, i0 = (tile - b * a.q_blocks) * a.q_block;
    const SeqTokens s = seq_tokens(p.start, p.kv_len, b, p.tokens, p.max_new);
    const int n = s.rows - i0 < a.q_block ? s.rows - i0 : a.q_block;
    constexpr int LANES = D / 8;
    // (a row's lanes are in one wavefront, which has loaded all of it before it stores: q_out may be q)
    for (int u = threadIdx.x; u < n * p.heads * LANES; u += APPEND_NT) {
        const int lane = u % LANES, head = u / LANES % p.heads, i = u / LANES / p.heads + i0;
        const long row = s.row0 + i, pos = s.first + i;
        float x[8];
        load_rotated((const T *)p.q + row * p.ld_qkv + (long)head * D, lane * 8, p.rot_dim, p.rot_pairs, [&](int j) { return turn(pos, p.inv_freq[j]); }, x);
        store8((T *)p.q_out + row * p.ld_q_out + (long)head * D + lane * 8, x);
    }
}

template <typename T, int D, bool E8, int LOOP = LOOP_ANY>
__global__ __launch_bounds__(APPEND_NT) void kv_append_kernel(AppendArgs a, BlpArgs blp) {
    __shared__ float lds_most[APPEND_NT / 64];
    tiles<LOOP>(blp, [&](TileIdx t) {
        if (t.x < a.kv_tiles) append_page<T, D, E8>(a, t.x, lds_most);
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
    const long kv_tiles = 2l * p->batch * a.touched * p->cache.kv_heads;
    a.q_block = std::min(8, max_new);
    a.q_blocks = (max_new + a.q_block - 1) / a.q_block;
    const long tiles = kv_tiles + (p->q ? (long)p->batch * a.q_blocks : 0);
    GP_REQUIRE(tiles < (1L << 31), "kv_append: too large");
    a.kv_tiles = (int)kv_tiles;
    const bool e8 = p->cache.dtype == GP_E4M3, f16 = p->dtype == GP_F16;
#define GP_APPEND(T, D, E8) return launch_tiles(GP_KSET(kv_append_kernel<T, D, E8), (int)tiles, 1, ctx, s, info, a, 0, 4, APPEND_NT)
    if (p->cache.head_dim == 128) {
        if (f16) { if (e8) GP_APPEND(_Float16, 128, true); GP_APPEND(_Float16, 128, false); }
        if (e8) GP_APPEND(__bf16, 128, true);
        GP_APPEND(__bf16, 128, false);
    }
    if (f16) { if (e8) GP_APPEND(_Float16, 64, true); GP_APPEND(_Float16, 64, false); }
    if (e8) GP_APPEND(__bf16, 64, true);
    GP_APPEND(__bf16, 64, false);
#undef GP_APPEND
}
