// Attention over a paged cache for many query rows: prompts, where the matrix products are most of the work.
//
// A tile is one head of the cache and 128 query rows of a sequence that share it (its new tokens times the query heads of the head), 32 to a wavefront.
// Keys and values come 64 at a time through LDS, two buffers of them, in 16 bits whatever the cache's type:
//   S^T = K Q^T    v_mfma_f32_32x32x16 with K as A: a lane has 16 scores of every 32 keys, of one query (column l % 32): keys
//                  8 (v / 4) + 4 (l / 32) + v % 4 in register v.  The softmax is a reduction over a lane's own registers and one exchange.
//   O^T = V^T P^T  with the probabilities as B where they are: registers 8 j .. 8 j + 7 stand for keys 16 j + 4 (l / 32) + {0..3} and those 8 behind.
//                  V is turned on its way into LDS, four keys by eight values in a thread's registers, its keys in that order, so that an operand is 16
//                  bytes of a row.
// Rows of LDS are 16-byte chunks whose place is changed by the row's number, so that eight neighbouring rows' chunks lie in different banks.
// Bound by the vector instructions of the softmax and the matrix instructions alike (32 of each lane's values cost about 900 cycles, the
// products of 64 keys 1024), so two workgroups share a compute unit and fill each other's gaps.
//
// Measured: four sequences of 2900 to 5000 keys, 1358 to 4096 of them new, 32 heads, 8 cached of 128, e4m3: 587 to 593 us, 920 TFLOP/s (a large matrix product: 1200).  The matrix
// instructions are busy 41 % of the cycles and vector instructions 58 %, and they seldom overlap; LDS is in conflict for a quarter of the cycles it is active.
#pragma once
#include "paged_few.hpp"

namespace gp {

constexpr int MANY_NT = 256, MANY_ROWS = 128, MANY_KEYS = 64;

struct ManyArgs {
    gp_paged_attention_params p;
    int group;       // query heads to a head of the cache
    int row_blocks;  // of MANY_ROWS rows
    int shares;      // parts of a block's keys, at most
    int *arrived;    // workspace: a counter for every (head, sequence, row block), 0 between launches
    float *partial;  // ... and many_partial_floats for every part
};
// Parts of a block's `tiles` tiles of keys, at most: joining a part costs as much as a few tiles.
__host__ __device__ inline int many_shares(long tiles, long most) {
    int n = 1;
    while (n < most && 3l * (n + 1) * (n + 1) <= tiles) ++n;
    return n;
}

template <int D> constexpr int many_partial_floats() { return (D / 32 * 16 + 2) * MANY_NT; }  // every thread's sums as they are, its maximum and its sum
template <int D> constexpr size_t many_lds_bytes() { return 2 * 2 * (size_t)MANY_KEYS * D * 2; }

// Where the keys and values of one head lie: in the pages that row `b` of a table names, or (packed) in rows one behind the other
struct PagedKeys {
    static constexpr bool PAGED = true;
    const gp_kv_cache &cache;
    const int *table;
    int width, b, kvh;
};
struct PackedKeys {
    static constexpr bool PAGED = false;
    const char *k, *v;  // of the first key
    long ld;            // bytes from one to the next
    int last;           // the last that there is
};

// A lane's query, and how many keys it sees (`there`: 0 .. kend; a lane without a query: nothing is asked of it)
struct ManyRow { bool there; int seen; const void *q; };

// The tiles [first_tile, tiles) of keys for 128 rows: adds up a lane's part of sum_j 2^(x_j - m) v_j in o (o[i][v] belongs to the lane's query and value
// 32 i + 8 (v / 4) + 4 half + v % 4), sum_j 2^(x_j - m) over the lane's half of the keys in l, the reference in m.  kend: keys that some row of the block sees; the values from
// `bound` on are taken as zeros.
template <typename T, int D, bool E8, class Keys>
__device__ __forceinline__ void many_keys(const Keys &keys, const ManyRow &row_of_lane, float score_scale, int kend, int bound, int first_tile, int tiles, char *lds, f32x16 (&o)[D / 32], float &m, float &l) {
#pragma clang fp contract(off)  // (as in attend_stretch)
    constexpr int ES = E8 ? 1 : 2, DB = D / 32, KSTEPS = D / 16;
    constexpr float ROOM = Reference<T>::room(8.f);
    constexpr int KCH = D / 8;                              // 16-byte chunks of a key's row in LDS
    constexpr int TILE_BYTES = MANY_KEYS * D * 2;           // of keys; values behind them
    constexpr bool PAGED = Keys::PAGED;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), l32 = lane & 31, half = lane >> 5;
    const bool there = row_of_lane.there;
    const int seen = row_of_lane.seen;
    int kmin = there ? seen : kend;  // what all rows of the wavefront see
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
        const int o = __shfl_xor(kmin, d, 64);
        kmin = o < kmin ? o : kmin;
    }
    kmin = __builtin_amdgcn_readfirstlane(kmin);
    u32x4 q[KSTEPS];
    {
        const T *row = (const T *)row_of_lane.q;
        const unsigned flip = score_scale < 0.f ? 0x80008000u : 0u;  // (so that the scale is positive from here on)
#pragma unroll
        for (int k = 0; k < KSTEPS; ++k) {
            q[k] = *(const u32x4 *)(row + 16 * k + 8 * half);
#pragma unroll
            for (int e = 0; e < 4; ++e) q[k][e] = there ? q[k][e] ^ flip : 0u;
        }
    }
    const float scale2 = fmaxf(fabsf(score_scale) * 1.44269504088896340736f, 0x1p-100f);
#pragma unroll
    for (int i = 0; i < DB; ++i)
#pragma unroll
        for (int v = 0; v < 16; ++v) o[i][v] = 0.f;
    m = -INFINITY;
    l = 0.f;

    // ---- pages: lane i has that of the i-th 16 keys of the sixteen tiles from `window` on; what a tile needs is read from there when it is needed (kept in
    // scalar registers over three steps there were too many of them: 608 us for the sequences named above, 593 so) ----
    int page_l = -1, window = first_tile;
    float ks_l = scale2, lv_l = 0.f, iv_l = 1.f;
    auto look_up = [&]() {
        if constexpr (PAGED) {
            const int key = window * MANY_KEYS + lane * 16;
            page_l = key < kend ? page_of(keys.table, keys.width, keys.b, key / keys.cache.page_size, keys.cache.pages) : -1;
            if constexpr (E8) {
                const long at = (long)(page_l < 0 ? 0 : page_l) * keys.cache.kv_heads + keys.kvh;
                const float vs = page_scale(keys.cache.v_scale, at);
                ks_l = fmaxf(scale2 * page_scale(keys.cache.k_scale, at), 0x1p-100f);  // (-infinity times it is that)
                lv_l = __builtin_amdgcn_logf(vs);
                iv_l = 1.f / vs;
            }
        }
    };
    auto scalar = [](float v, int at) { return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), at)); };
    // ---- from the pages to registers: thread (tid % 16, tid / 16).  Keys: 16 keys at a time, a row's 16 (8) chunks side by side.  Values: four keys of the
    // wavefront's 16, eight (four) values ----
    constexpr int KLOADS = E8 ? 2 * D / 128 : 4 * D / 128;  // 16-byte loads of a thread for the keys
    constexpr int KROWS = MANY_NT / (D * ES / 16);          // keys at a time
    constexpr int VV = D / 16;                              // values of a thread
    typedef unsigned int VRow __attribute__((ext_vector_type(VV * ES / 4)));
    static_assert(KROWS * KLOADS == MANY_KEYS, "the loads of a tile's keys");
    u32x4 kr[KLOADS];
    VRow vr[4];
    // (packed: a lane's rows of a tile as offsets of 32 bits from the tile's first, which the wavefront shares; in the tile where the sequence ends they stop at its last row.  A multiplication of 64 bits
    // for each load instead: 1540 us for 1520)
    unsigned krow[KLOADS], vrow[4];
    auto look_at_rows = [&](int last) {
        if constexpr (!PAGED) {
            auto row = [&](int r) { return (unsigned)(r < last ? r : last) * (unsigned)keys.ld; };
#pragma unroll
            for (int i = 0; i < KLOADS; ++i) krow[i] = row(i * KROWS + tid / (D * ES / 16)) + tid % (D * ES / 16) * 16;
#pragma unroll
            for (int e = 0; e < 4; ++e) vrow[e] = row(wave * 16 + lane / 16 * 4 + e) + lane % 16 * (VV * ES);
        }
    };
    look_at_rows(MANY_KEYS);
    auto fetch = [&](int tile) {
        if constexpr (!PAGED) {
            if (tile * MANY_KEYS + MANY_KEYS > keys.last) look_at_rows(keys.last - tile * MANY_KEYS);
            const char *k = keys.k + tile * MANY_KEYS * keys.ld, *v = keys.v + tile * MANY_KEYS * keys.ld;
#pragma unroll
            for (int i = 0; i < KLOADS; ++i) kr[i] = *(const u32x4 *)(k + krow[i]);
#pragma unroll
            for (int e = 0; e < 4; ++e) vr[e] = *(const VRow *)(v + vrow[e]);
        } else {
            auto block_at = [&](int page, int key) -> long { return (((long)(page < 0 ? 0 : page) * keys.cache.kv_heads + keys.kvh) * keys.cache.page_size + (key & (keys.cache.page_size - 1))) * D * ES; };
            const int sub = (tile - window) * 4;
#pragma unroll
            for (int i = 0; i < KLOADS; ++i) {
                const int row = i * KROWS + tid / (D * ES / 16), chunk = tid % (D * ES / 16);
                const int page = __builtin_amdgcn_readlane(page_l, sub + (i * KROWS + wave * (64 / (D * ES / 16))) / 16);  // (a wavefront's rows are 16 or part of them)
                kr[i] = *(const u32x4 *)((const char *)keys.cache.k + block_at(page, tile * MANY_KEYS + row) + chunk * 16);
            }
            const int page = __builtin_amdgcn_readlane(page_l, sub + wave), key0 = tile * MANY_KEYS + wave * 16 + lane / 16 * 4;
            const char *at = (const char *)keys.cache.v + block_at(page, key0) + lane % 16 * (VV * ES);
#pragma unroll
            for (int e = 0; e < 4; ++e) vr[e] = *(const VRow *)(at + e * D * ES);
        }
    };
    // ---- ... and on to LDS ----
    auto kslot = [&](int row, int chunk) { return row * (D * 2) + (chunk ^ (row & (KCH - 1))) * 16; };
    auto vslot = [&](int d, int chunk) { return TILE_BYTES + d * (MANY_KEYS * 2) + (chunk ^ ((d ^ (d >> 3)) & 7)) * 16; };
    // (what a lane reads, once for all tiles: 32 keys on, or 64 values on, and in the other buffer are constants away)
    int kat[KSTEPS], vat[2][4];
#pragma unroll
    for (int k = 0; k < KSTEPS; ++k) kat[k] = kslot(l32, 2 * k + half);
#pragma unroll
    for (int u = 0; u < 4; ++u) { vat[0][u] = vslot(l32, 2 * u + half); vat[1][u] = vslot(32 + l32, 2 * u + half); }
    auto stage = [&](char *buf, int tile) {
#pragma unroll
        for (int i = 0; i < KLOADS; ++i) {
            const int row = i * KROWS + tid / (D * ES / 16), chunk = tid % (D * ES / 16);
            if constexpr (E8) {
                const u32x4 x = kr[i];
                *(u32x4 *)(buf + kslot(row, 2 * chunk)) = u32x4{widen<false>(x[0], T()), widen<true>(x[0], T()), widen<false>(x[1], T()), widen<true>(x[1], T())};
                *(u32x4 *)(buf + kslot(row, 2 * chunk + 1)) = u32x4{widen<false>(x[2], T()), widen<true>(x[2], T()), widen<false>(x[3], T()), widen<true>(x[3], T())};
            } else {
                *(u32x4 *)(buf + kslot(row, chunk)) = kr[i];
            }
        }
        const int vbound = !PAGED || __builtin_amdgcn_readlane(page_l, (tile - window) * 4 + wave) >= 0 ? bound : 0;
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (tile * MANY_KEYS + wave * 16 + lane / 16 * 4 + e >= vbound) vr[e] = VRow(0);
        // keys 4 g .. 4 g + 3 of the wavefront's 16: half g % 2, and there the first four or the second
        const int g = lane / 16, chunk = 2 * wave + g % 2, d0 = lane % 16 * VV;
#pragma unroll
        for (int j = 0; j < VV; j += 2) {
            u32x2 v0, v1;
#pragma unroll
            for (int kp = 0; kp < 2; ++kp) {
                if constexpr (E8) {
                    const unsigned two = __builtin_amdgcn_perm(vr[2 * kp + 1][j / 4], vr[2 * kp][j / 4], j % 4 == 0 ? 0x05010400u : 0x07030602u);
                    v0[kp] = widen<false>(two, T());
                    v1[kp] = widen<true>(two, T());
                } else {
                    v0[kp] = __builtin_amdgcn_perm(vr[2 * kp + 1][j / 2], vr[2 * kp][j / 2], 0x05040100u);
                    v1[kp] = __builtin_amdgcn_perm(vr[2 * kp + 1][j / 2], vr[2 * kp][j / 2], 0x07060302u);
                }
            }
            *(u32x2 *)(buf + vslot(d0 + j, chunk) + g / 2 * 8) = v0;
            *(u32x2 *)(buf + vslot(d0 + j + 1, chunk) + g / 2 * 8) = v1;
        }
    };

    // A tile's way: fetched two steps ahead, put into LDS one step ahead, between the matrix instructions of the scores
    __syncthreads();  // (the previous tile's buffers are still being read)
    if (tiles > first_tile) {
        look_up();
        fetch(first_tile);
        stage(lds, first_tile);
        if (first_tile + 1 < tiles) fetch(first_tile + 1);
    }
    __syncthreads();
    // one tile of keys, in buffer BUF
    auto step = [&](int tile, auto buffer) {
        constexpr int BUF = decltype(buffer)::value;
        const char *buf = lds + BUF * 2 * TILE_BYTES;
        const int key0 = tile * MANY_KEYS;
        if (PAGED && tile + 2 - window >= 16) { window = tile; look_up(); }  // (this tile, the one that is staged and the one that is fetched)
        const int sub = (tile - window) * 4;
        int pages[4];
        float ks[4], lv[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            pages[u] = PAGED ? __builtin_amdgcn_readlane(page_l, sub + u) : 0;
            ks[u] = E8 ? scalar(ks_l, sub + u) : scale2;
            lv[u] = E8 ? scalar(lv_l, sub + u) : 0.f;
        }
        const bool whole = key0 + MANY_KEYS <= kmin && (pages[0] | pages[1] | pages[2] | pages[3]) >= 0;
        // ---- scores ----
        f32x16 x[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
#pragma unroll
            for (int v = 0; v < 16; ++v) x[i][v] = 0.f;
#pragma unroll
            for (int k = 0; k < KSTEPS; ++k) Elem<T>::mma(*(const u32x4 *)(buf + kat[k] + i * 32 * D * 2), q[k], x[i]);
        }
        stage(lds + (1 - BUF) * 2 * TILE_BYTES, tile + 1);  // (behind the last tile: the last one again, which nobody reads)
        // (the order that the compiler is asked for: operands four ahead, a few of the other instructions behind every matrix instruction; four prompts of 2600 to 4096 tokens,
        // 32 heads of 128, bf16: 708 us without, 681 with)
        __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);  // reads of LDS
#pragma unroll
        for (int k = 0; k < 2 * KSTEPS; ++k) {
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);  // matrix instructions
            __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x002, 5, 0);  // vector instructions
        }
        if (tile + 2 < tiles) fetch(tile + 2);
        if (!whole) {
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int v = 0; v < 16; ++v)
                    if (pages[2 * i + v / 8] < 0 || key0 + i * 32 + 8 * (v / 4) + 4 * half + v % 4 >= seen) x[i][v] = -INFINITY;
        }
        // ---- running reference (raised only when it is exceeded 2^ROOM-fold, which the types and the sums have room for) and sum.  8 bits: the logarithm of the
        // values' scale is part of the exponent, so that what is rounded to 16 bits is the probability times that scale; the sum takes it back out ----
        float top = -INFINITY;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            float most = x[u / 2][8 * (u % 2)];
#pragma unroll
            for (int v = 1; v < 8; ++v) most = fmaxf(most, x[u / 2][8 * (u % 2) + v]);
            top = fmaxf(top, fmaf(most, ks[u], lv[u]));
        }
        top = fmaxf(top, __shfl_xor(top, 32, 64));
        if (__any(top > m + ROOM)) {
            const float high = fmaxf(m, Reference<T>::below(top)), f = high == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - high);
            m = high;
            l *= f;
#pragma unroll
            for (int i = 0; i < DB; ++i)
#pragma unroll
                for (int v = 0; v < 16; ++v) o[i][v] *= f;
        }
        const float base = m == -INFINITY ? 0.f : m;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const float off = lv[u] - base;
            float part = 0.f;
            typedef T tx8 __attribute__((ext_vector_type(8)));
            tx8 pb;
#pragma unroll
            for (int v = 0; v < 8; ++v) {
                const float y = __builtin_amdgcn_exp2f(fmaf(x[u / 2][8 * (u % 2) + v], ks[u], off));
                part += y;
                pb[v] = Elem<T>::from_f(y);
            }
            l = E8 ? fmaf(part, scalar(iv_l, sub + u), l) : l + part;
            // ---- O^T += V^T P^T, 16 keys ----
#pragma unroll
            for (int i = 0; i < DB; ++i) Elem<T>::mma(*(const u32x4 *)(buf + vat[i % 2][u] + i / 2 * 64 * MANY_KEYS * 2), __builtin_bit_cast(u32x4, pb), o[i]);
        }
        __syncthreads();
    };
    for (int tile = first_tile; tile < tiles; tile += 2) {
        step(tile, IntC<0>());
        if (tile + 1 < tiles) step(tile + 1, IntC<1>());
    }
}

template <typename T, int D, bool E8>
__device__ __forceinline__ void attend_many(const ManyArgs &a, TileIdx t, char *lds) {
#pragma clang fp contract(off)  // (as in attend_stretch)
    const gp_paged_attention_params &p = a.p;
    constexpr int DB = D / 32;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), l32 = lane & 31, half = lane >> 5, P = p.cache.page_size;
    const int rb = a.row_blocks - 1 - t.x / a.shares, share = t.x % a.shares, b = t.y % p.batch, kvh = t.y / p.batch;  // (the last rows see most keys: they come first)
    const SeqTokens s = seq_tokens(p.start, p.kv_len, b, p.tokens, p.max_new);
    const int nrows = s.rows * a.group - rb * MANY_ROWS;
    if (nrows <= 0) return;
    const int bound = (int)seq_bound(s, p.max_len, p.table_width, P);
    const int last_token = (rb * MANY_ROWS + (nrows < MANY_ROWS ? nrows : MANY_ROWS) - 1) / a.group;
    const int kend = (int)keys_seen(bound, s.first + last_token, p.causal), all_tiles = (kend + MANY_KEYS - 1) / MANY_KEYS;
    const int shares = a.shares == 1 ? 1 : many_shares(all_tiles, a.shares);
    if (share >= shares) return;
    const int first_tile = (int)((long)share * all_tiles / shares), tiles = (int)((share + 1l) * all_tiles / shares);

    // ---- this lane's query ----
    const int r = wave * 32 + l32, token = (rb * MANY_ROWS + r) / a.group, hg = rb * MANY_ROWS + r - token * a.group;
    const bool there = r < nrows;
    const int seen = there ? (int)keys_seen(bound, s.first + token, p.causal) : 0;
    const T *q = (const T *)p.q + (s.row0 + (there ? token : 0)) * p.ld_q + ((long)kvh * a.group + (there ? hg : 0)) * D;
    f32x16 o[DB];
    float m, l;
    many_keys<T, D, E8>(PagedKeys{p.cache, p.page_table, p.table_width, b, kvh}, ManyRow{there, seen, q}, p.scale, kend, bound, first_tile, tiles, lds, o, m, l);
    l += __shfl_xor(l, 32, 64);
    if (shares > 1) {
        // a part: every thread leaves what it has; the threads of whoever comes last take the parts, in their order, from where they left them
        const long unit = (long)t.y * a.row_blocks + rb;
        float *mine = a.partial + (unit * a.shares + share) * many_partial_floats<D>() + 2 * tid;
#pragma unroll
        for (int i = 0; i < DB; ++i)
#pragma unroll
            for (int v = 0; v < 16; v += 2) put_shared(mine + (8 * i + v / 2) * 2 * MANY_NT, f32x2{o[i][v], o[i][v + 1]});
        put_shared(mine + 8 * DB * 2 * MANY_NT, f32x2{m, l});
        __shared__ int came;
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the stores above have reached the memory that all XCDs see
        __syncthreads();
        if (tid == 0) came = __hip_atomic_fetch_add(a.arrived + unit, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __syncthreads();
        if (came != shares - 1) return;
        if (tid == 0) __hip_atomic_store(a.arrived + unit, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        m = -INFINITY;
        l = 0.f;
#pragma unroll
        for (int i = 0; i < DB; ++i)
#pragma unroll
            for (int v = 0; v < 16; ++v) o[i][v] = 0.f;
        for (int k = 0; k < shares; ++k) {
            const float *from = a.partial + (unit * a.shares + k) * many_partial_floats<D>() + 2 * tid;
            f32x2 y[8 * DB + 1];
#pragma unroll
            for (int i = 0; i <= 8 * DB; ++i) y[i] = get_shared(from + i * 2 * MANY_NT);
            const float mk = y[8 * DB][0], now = fmaxf(m, mk), base = now == -INFINITY ? 0.f : now;
            const float f = __builtin_amdgcn_exp2f(m - base), fk = __builtin_amdgcn_exp2f(mk - base);
            m = now;
            l = fmaf(l, f, y[8 * DB][1] * fk);
#pragma unroll
            for (int i = 0; i < DB; ++i)
#pragma unroll
                for (int v = 0; v < 16; ++v) o[i][v] = fmaf(o[i][v], f, y[8 * i + v / 2][v % 2] * fk);
        }
    }
    if (!there) return;
    const float inv = l == 0.f ? 0.f : 1.f / l;
    T *out = (T *)p.out + (s.row0 + token) * p.ld_out + ((long)kvh * a.group + hg) * D + 4 * half;
#pragma unroll
    for (int i = 0; i < DB; ++i)
#pragma unroll
        for (int v = 0; v < 16; v += 4) {
            typedef T tx4 __attribute__((ext_vector_type(4)));
            tx4 y;
#pragma unroll
            for (int e = 0; e < 4; ++e) y[e] = Elem<T>::from_f(rounded(o[i][v + e] * inv));
            *(tx4 *)(out + 32 * i + 2 * v) = y;
        }
}

template <typename T, int D, bool E8, int LOOP = LOOP_ANY>
__global__ __launch_bounds__(MANY_NT, 2) void paged_many_kernel(ManyArgs a, BlpArgs blp) {
    extern __shared__ __attribute__((aligned(16))) unsigned char many_lds[];
    tiles<LOOP>(blp, [&](TileIdx t) { attend_many<T, D, E8>(a, t, (char *)many_lds); });
}

}  // namespace gp
