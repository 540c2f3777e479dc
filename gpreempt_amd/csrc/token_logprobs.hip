// Log probabilities of given tokens, entropy and largest alternatives of rows of logits, in one pass over the row.
//
// With m the largest logit so far, y = scale * (x - m), S = sum 2^(y log2 e) and W = sum y 2^(..): log p = y - log S, entropy = log S - W / S, and a
// larger m' turns them into f S and f (W + d S), f = 2^(d log2 e), d = scale * (m - m').  Every thread keeps m, S and W of what it has seen.
// Many rows: a workgroup takes a row, 16384 logits at a time, 32 to a thread, the next ones on their way while these are worked on.
// A few long rows are cut into parts, joined by whoever comes last.
// Measured: 500 rows of 131001 bf16 logits, 20 alternatives: 35 us, 3.8 TB/s (a kernel that only reads: 7.1), bound by vector instructions:
// a wavefront takes some 62 cycles of them per 64 logits (16 of these the exponential) for the maximum, the two sums and their exponents.  One row of 30522: 7.5 us, of which a launch is 4.5.
// Rows that are walked once more for every alternative, since more logits are candidates than the list holds (below): the 500 rows with all logits equal 1980 us.
//
// The alternatives: every group of eight threads leaves the largest logit of each tile in LDS.  Of the 64 lanes' largest logits, all wavefronts together, the
// top-th largest is a bound that at least `top` logits reach; the few groups and tiles that reach it are looked at again, what reaches it goes to a list
// in LDS, and the largest are picked from there by their rank.
#include <algorithm>
#include "mma.hpp"
#include "lanes.hpp"
#include "launch_tiles.hpp"

namespace gp {

constexpr int LP_NT = 512, LP_WAVES = LP_NT / 64, LP_TOP = 32;
constexpr int LP_EACH = 32;                 // logits of a thread at a time
constexpr int LP_TILE = LP_NT * LP_EACH;
constexpr int LP_LIST = 1024;               // places for candidates
constexpr int LP_GROUPS = LP_NT / 8;          // of eight threads
constexpr int LP_KEPT = 32;                 // tiles whose groups' largest logits are kept apart (tile t and t + 32 together)
static_assert(LP_GROUPS == 64, "a lane for each group");
constexpr int LP_PARTS = 16;                // of a row, at most
constexpr int LP_PART_WORDS = 2 + LP_TOP;   // 64-bit words of a part's result

struct LogprobsArgs {
    gp_token_logprobs_params p;
    int parts, tiles_per_part;
    int *arrived;                 // workspace: a counter per row, 0 between launches
    unsigned long long *partial;  // ... and LP_PART_WORDS for every part
};

struct LogprobsLds {
    float groups[LP_KEPT][LP_GROUPS], lanes[LP_WAVES][64];
    int count, hits, came;
    float red[3][LP_WAVES];
    unsigned long long list[2][LP_LIST];
    unsigned short hit[LP_KEPT * LP_GROUPS];
};

// Order of the alternatives in one number: the larger logit first, then the lower token.  0: no alternative (NaN, -infinity).
__device__ __forceinline__ unsigned long long rank_key(float x, int id) {
    if (!(x > -INFINITY)) return 0;
    const unsigned bits = __builtin_bit_cast(unsigned, x == 0.f ? 0.f : x);  // (one zero)
    return (unsigned long long)(bits & 0x80000000u ? ~bits : bits | 0x80000000u) << 32 | (0xFFFFFFFFu - (unsigned)id);
}
__device__ __forceinline__ float key_value(unsigned long long key) {
    const unsigned u = (unsigned)(key >> 32);
    return key ? __builtin_bit_cast(float, u & 0x80000000u ? u & 0x7FFFFFFFu : ~u) : -INFINITY;
}
__device__ __forceinline__ int key_id(unsigned long long key) { return key ? (int)(0xFFFFFFFFu - (unsigned)key) : -1; }

// A value that at least `top` of the 64 lanes' values reach, the largest with its 16 leading bits (-infinity: fewer than that are above it).  Bit by bit, in
// scalar registers: a rank by 64 comparisons takes a wavefront ten times as many vector instructions.
__device__ __forceinline__ float reached_by(float v, int top) {
    const unsigned bits = __builtin_bit_cast(unsigned, v), order = v > -INFINITY ? (bits & 0x80000000u ? ~bits : bits | 0x80000000u) : 0u;
    unsigned t = 0;
#pragma unroll
    for (int bit = 31; bit >= 16; --bit)
        if (__popcll(__ballot(order >= (t | 1u << bit))) >= top) t |= 1u << bit;
    return t == 0 ? -INFINITY : __builtin_bit_cast(float, t & 0x80000000u ? t & 0x7FFFFFFFu : ~t);
}
// A thread's logits of one tile: LOADS times VEC neighbours.  The chunk in which the row ends is fetched so that it ends there, whoever comes behind it fetches
// the same; what is in front of a thread's own place counts as -infinity.
template <typename T> struct Logits {
    static constexpr int VEC = 16 / sizeof(T), LOADS = LP_EACH / VEC;
    typedef T Raw __attribute__((ext_vector_type(VEC), aligned(sizeof(T))));  // (rows start anywhere)
    typedef T Chunk __attribute__((ext_vector_type(VEC)));
    static __device__ __forceinline__ int own(int thread, int tile, int load) { return tile * LP_TILE + load * (LP_NT * VEC) + thread * VEC; }
    static __device__ __forceinline__ int at(int own, int vocab) { return own + VEC <= vocab || vocab < VEC ? own : vocab - VEC; }  // where it is fetched from
    Chunk raw[LOADS];
    static __device__ __forceinline__ void mask(Chunk &c, int vocab, int own) {
#pragma unroll
        for (int e = 0; e < VEC; ++e)
            if (e < own - at(own, vocab)) c[e] = Elem<T>::from_f(-INFINITY);
    }
    // a row shorter than a chunk
    static __device__ __forceinline__ Chunk tiny(const T *row, int vocab, int own) {
        Chunk c;
#pragma unroll
        for (int e = 0; e < VEC; ++e) c[e] = own == 0 && e < vocab ? row[e < vocab ? e : 0] : Elem<T>::from_f(-INFINITY);
        return c;
    }
    // (the same loads whatever the tile, so that the compiler knows at every wait how many are younger; the row's last tile is masked when it is there)
    __device__ __forceinline__ void fetch(const T *row, int vocab, int tile) {
#pragma unroll
        for (int k = 0; k < LOADS; ++k) raw[k] = *(const Raw *)(row + at(own((int)threadIdx.x, tile, k), vocab));
    }
    __device__ __forceinline__ float operator()(int k, int e) const { return Elem<T>::to_f(raw[k][e]); }
};

// the largest `top` of a list of keys (no 0 among them), of which there may be fewer: put(rank, key)
template <class Put>
__device__ __forceinline__ void pick(LogprobsLds &l, int which, int count, int top, Put &&put) {
    const int tid = threadIdx.x;
    float bound = -INFINITY;
    while (count > 256) {  // (of a long list, those that reach a bound: as for the logits)
        float most = -INFINITY;
        for (int i = tid; i < count; i += LP_NT) most = fmaxf(most, key_value(l.list[which][i]));
        most = max_of_8_lanes(most);
        __syncthreads();
        if ((tid & 7) == 0) l.groups[0][tid >> 3] = most;
        if (tid == 0) l.count = 0;
        __syncthreads();
        const float next = reached_by(l.groups[0][tid & 63], top);
        if (!(next > bound)) break;
        bound = next;
        for (int i = tid; i < count; i += LP_NT) {
            const unsigned long long key = l.list[which][i];
            if (key_value(key) >= bound) l.list[!which][atomicAdd(&l.count, 1)] = key;
        }
        __syncthreads();
        count = l.count;
        which = !which;
    }
    for (int i = tid; i < count; i += LP_NT) {
        const unsigned long long key = l.list[which][i];
        int rank = 0;
#pragma unroll 8
        for (int j = 0; j < count; ++j) rank += l.list[which][j] > key;
        if (rank < top) put(rank, key);
    }
    for (int i = count + tid; i < top; i += LP_NT) put(i, 0ull);
}

template <typename T>
__device__ __forceinline__ void logprobs_tile(const LogprobsArgs &a, TileIdx t, LogprobsLds &l) {
#pragma clang fp contract(off)  // (contracted where the code says so and nowhere else: the plain and the preemptible kernels give the same bits)
    const gp_token_logprobs_params &p = a.p;
    const int tid = threadIdx.x, wave = tid >> 6, top = p.top, vocab = p.vocab;
    const long r = t.y;
    const T *row = (const T *)p.logits + r * p.ld;
    const float c = p.scale * 1.44269504088896340736f;
    const int tiles = (vocab + LP_TILE - 1) / LP_TILE, first = t.x * a.tiles_per_part, last = first + a.tiles_per_part < tiles ? first + a.tiles_per_part : tiles;
    Logits<T> x;
    const bool tiny = vocab < Logits<T>::VEC;
    if (!tiny) x.fetch(row, vocab, first);
    // the given token's logit (needed last)
    const long token = p.logprob ? p.tokens[r] : -1;
    const T said_raw = token >= 0 && token < vocab ? row[token] : Elem<T>::from_f(0.f);
    __syncthreads();  // (the previous row's lists are still being read)
    if (tid == 0) l.count = l.hits = 0;

    float m = -INFINITY, s = 0.f, w = 0.f;
    auto add = [&](const Logits<T> &x, int tile) {
        float most = -INFINITY;
#pragma unroll
        for (int k = 0; k < Logits<T>::LOADS; ++k)
#pragma unroll
            for (int e = 0; e < Logits<T>::VEC; e += 2) most = max3(most, x(k, e), x(k, e + 1));
        if (most > m) {
            if (m > -INFINITY) {
                const float d = (m - most) * c, f = __builtin_amdgcn_exp2f(d);
                w = f == 0.f ? 0.f : f * fmaf(d, s, w);
                s *= f;
            }
            m = most;
        }
        const float base = m > -INFINITY ? m : 0.f;  // (nothing but -infinity so far; or NaN, whose sum is NaN all the same)
#pragma unroll
        for (int k = 0; k < Logits<T>::LOADS; ++k)
#pragma unroll
            for (int e = 0; e < Logits<T>::VEC; ++e) {
                const float y = (x(k, e) - base) * c, z = __builtin_amdgcn_exp2f(y);
                s += z;
                w = fmaf(z, max3(y, -150.f, -150.f), w);  // (where 2^y is 0, y may be -infinity)
            }
        if (top) {
            const float group = max_of_8_lanes(most);
            if ((tid & 7) == 0) {
                float *at = &l.groups[(tile - first) % LP_KEPT][tid >> 3];
                *at = tile - first < LP_KEPT ? group : max3(*at, group, group);
            }
        }
    };
    for (int tile = first; tile + 1 < last; ++tile) {
        Logits<T> next;
        next.fetch(row, vocab, tile + 1);
        add(x, tile);
        x = next;
    }
    if (last * LP_TILE > vocab) {
#pragma unroll
        for (int k = 0; k < Logits<T>::LOADS; ++k) {
            const int own = Logits<T>::own(tid, last - 1, k);
            if (tiny) x.raw[k] = Logits<T>::tiny(row, vocab, own);
            else Logits<T>::mask(x.raw[k], vocab, own);
        }
    }
    add(x, last - 1);

    // ---- the threads' sums ----
    const int kept = last - first < LP_KEPT ? last - first : LP_KEPT;
    // A signalling NaN has made the instruction above forget the largest logit so far (making it a quiet one first is an instruction more for every logit of every row).  A thread that has
    // seen one, whose sum is NaN then, has its group looked at again whatever that left.  (A bound that is too low only lets more candidates through)
    if (top && s != s)
        for (int i = 0; i < kept; ++i) l.groups[i][tid >> 3] = INFINITY;
    float M = max_of_wave(m);
    l.lanes[wave][tid & 63] = m;
    if ((tid & 63) == 0) l.red[0][wave] = M;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < LP_WAVES; ++i) M = fmaxf(M, l.red[0][i]);
    if (m > -INFINITY) {
        const float d = (m - M) * c, f = __builtin_amdgcn_exp2f(d);
        w = f == 0.f ? 0.f : f * fmaf(d, s, w);
        s *= f;
    } else w = 0.f;  // (s is 0, or NaN)
    s = sum_of_wave(s);
    w = sum_of_wave(w);
    if ((tid & 63) == 0) { l.red[1][wave] = s; l.red[2][wave] = w; }
    // ---- candidates ----
    float bound = -INFINITY;
    if (top) {
        float lane = l.lanes[0][tid & 63];
#pragma unroll
        for (int i = 1; i < LP_WAVES; ++i) lane = fmaxf(lane, l.lanes[i][tid & 63]);
        bound = reached_by(lane, top);
        for (int i = tid; i < kept * LP_GROUPS; i += LP_NT) {
            const float g = l.groups[i / LP_GROUPS][i % LP_GROUPS];
            if (g >= bound && g > -INFINITY) l.hit[atomicAdd(&l.hits, 1)] = (unsigned short)i;
        }
    }
    __syncthreads();
    s = w = 0.f;
#pragma unroll
    for (int i = 0; i < LP_WAVES; ++i) { s += l.red[1][i]; w += l.red[2][i]; }
    constexpr int LOOKS = 8 * Logits<T>::LOADS;  // chunks of a group and tile
    const int looks = l.hits * LOOKS;
    for (int i = tid; i < looks; i += LP_NT) {
        const int hit = l.hit[i / LOOKS], thread = hit % LP_GROUPS * 8 + i % 8, load = i / 8 % Logits<T>::LOADS;
        for (int tile = first + hit / LP_GROUPS; tile < last; tile += LP_KEPT) {
            const int own = Logits<T>::own(thread, tile, load);
            typename Logits<T>::Chunk chunk;
            if (tiny) chunk = Logits<T>::tiny(row, vocab, own);
            else {
                chunk = *(const typename Logits<T>::Raw *)(row + Logits<T>::at(own, vocab));
                Logits<T>::mask(chunk, vocab, own);
            }
#pragma unroll
            for (int e = 0; e < Logits<T>::VEC; ++e) {
                const float v = Elem<T>::to_f(chunk[e]);
                if (v >= bound && v > -INFINITY) {
                    const int at = atomicAdd(&l.count, 1);
                    if (at < LP_LIST) l.list[0][at] = rank_key(v, Logits<T>::at(own, vocab) + e);
                }
            }
        }
    }
    __syncthreads();
    int count = l.count;

    auto finish = [&](float M, float s, float w, int which, int count) {
        const float log_sum = __builtin_amdgcn_logf(s) * 0.69314718055994530942f, said = Elem<T>::to_f(said_raw);
        if (tid == 0) {
            if (p.logprob) p.logprob[r] = token < 0 || token >= vocab ? 0.f : s == 0.f || (said == -INFINITY && s == s) ? -INFINITY : (said - M) * p.scale - log_sum;
            if (p.entropy) p.entropy[r] = s == 0.f ? 0.f : log_sum - w * 0.69314718055994530942f / s;
        }
        if (top) pick(l, which, count, top, [&](int rank, unsigned long long key) {
            p.top_ids[r * top + rank] = key_id(key);
            p.top_logprobs[r * top + rank] = key ? (key_value(key) - M) * p.scale - log_sum : -INFINITY;
        });
    };
    // more candidates than the list holds (equal logits, say): one after the other, each the largest behind the last one
    if (top && count > LP_LIST) {
        const int from = first * LP_TILE, to = last * LP_TILE < vocab ? last * LP_TILE : vocab;
        unsigned long long before = ~0ull;
        for (int k = 0; k < top; ++k) {
            unsigned long long best = 0;
            for (int i = from + tid; i < to; i += LP_NT) {
                const unsigned long long key = rank_key(Elem<T>::to_f(row[i]), i);
                if (key < before && key > best) best = key;
            }
#pragma unroll
            for (int d = 1; d < 64; d *= 2) {
                const unsigned long long o = __shfl_xor(best, d, 64);
                best = o > best ? o : best;
            }
            __syncthreads();
            if ((tid & 63) == 0) l.list[1][wave] = best;
            __syncthreads();
#pragma unroll
            for (int i = 0; i < LP_WAVES; ++i) best = l.list[1][i] > best ? l.list[1][i] : best;
            if (tid == 0) l.list[0][k] = best;
            before = best;
        }
        __syncthreads();
        count = top;
    }
    if (a.parts == 1) { finish(M, s, w, 0, count); return; }

    // ---- a part of a row: its result, and whoever comes last joins them ----
    auto put = [&](unsigned long long *q, unsigned long long v) { __hip_atomic_store(q, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); };
    auto get = [&](const unsigned long long *q) { return __hip_atomic_load(q, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); };
    unsigned long long *mine = a.partial + (r * a.parts + t.x) * LP_PART_WORDS;
    if (tid == 0) { put(mine, __builtin_bit_cast(unsigned long long, f32x2{M, s})); put(mine + 1, __builtin_bit_cast(unsigned long long, f32x2{w, 0.f})); }
    if (top) pick(l, 0, count, top, [&](int rank, unsigned long long key) { put(mine + 2 + rank, key); });
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the stores above have reached the memory that all XCDs see
    __syncthreads();
    if (tid == 0) l.came = __hip_atomic_fetch_add(a.arrived + r, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    if (l.came != a.parts - 1) return;
    if (tid == 0) __hip_atomic_store(a.arrived + r, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    const unsigned long long *all = a.partial + r * a.parts * LP_PART_WORDS;
    M = -INFINITY;
    f32x2 ms[LP_PARTS], wz[LP_PARTS];
#pragma unroll
    for (int i = 0; i < LP_PARTS; ++i) {
        ms[i] = __builtin_bit_cast(f32x2, get(all + (i < a.parts ? i : 0) * LP_PART_WORDS));
        wz[i] = __builtin_bit_cast(f32x2, get(all + (i < a.parts ? i : 0) * LP_PART_WORDS + 1));
        M = fmaxf(M, ms[i][0]);
    }
    if (tid == 0) l.count = 0;
    __syncthreads();
    for (int i = tid; i < a.parts * top; i += LP_NT) {
        const unsigned long long key = get(all + i / top * LP_PART_WORDS + 2 + i % top);
        if (key) l.list[0][atomicAdd(&l.count, 1)] = key;
    }
    s = w = 0.f;
#pragma unroll
    for (int i = 0; i < LP_PARTS; ++i)
        if (i < a.parts) {
            if (ms[i][0] > -INFINITY) {
                const float d = (ms[i][0] - M) * c, f = __builtin_amdgcn_exp2f(d);
                w += f == 0.f ? 0.f : f * fmaf(d, ms[i][1], wz[i][0]);
                s = fmaf(f, ms[i][1], s);
            } else s += ms[i][1];
        }
    __syncthreads();
    finish(M, s, w, 0, l.count);
}

template <typename T, int LOOP = LOOP_ANY>
__global__ __launch_bounds__(LP_NT) void token_logprobs_kernel(LogprobsArgs a, BlpArgs blp) {
    __shared__ LogprobsLds l;
    tiles<LOOP>(blp, [&](TileIdx t) { logprobs_tile<T>(a, t, l); });
}

static int plan_token_logprobs(const gp_token_logprobs_params *p, LogprobsArgs *a, size_t *work_bytes) {
    GP_REQUIRE(p && p->logits, "null token_logprobs params");
    GP_REQUIRE(p->dtype == GP_F32 || p->dtype == GP_F16 || p->dtype == GP_BF16, "token_logprobs dtype %d", p->dtype);
    GP_REQUIRE(p->rows > 0 && p->rows < (1L << 31) && p->vocab > 0 && p->vocab < (1 << 30) && p->ld >= p->vocab, "token_logprobs: rows, vocab (below 2^30) and a row stride that holds it");
    GP_REQUIRE(((uintptr_t)p->logits & (p->dtype == GP_F32 ? 3 : 1)) == 0, "token_logprobs: logits are not aligned to their type");
    GP_REQUIRE(p->top >= 0 && p->top <= LP_TOP, "token_logprobs: 0 to %d alternatives", LP_TOP);
    GP_REQUIRE(!p->top || (p->top_ids && p->top_logprobs), "token_logprobs: alternatives need a place to go to");
    GP_REQUIRE(p->logprob || p->entropy || p->top, "token_logprobs: nothing is asked for");
    GP_REQUIRE(!p->logprob || p->tokens, "token_logprobs: log probabilities of which tokens?");
    GP_REQUIRE(p->scale >= 0.f && usable_scale(p->scale), "token_logprobs: the scale must be 0 (for 1) or from 2^-100 to 2^100");
    *a = LogprobsArgs{};
    a->p = *p;
    if (p->scale == 0.f) a->p.scale = 1.f;
    // rows of at least four tiles are cut while there are compute units without one, into parts of two tiles or more
    const long tiles = ((long)p->vocab + LP_TILE - 1) / LP_TILE;
    const long want = std::max(1l, std::min({(long)LP_PARTS, device_cus() / p->rows, tiles / 2}));
    a->tiles_per_part = (int)((tiles + want - 1) / want);
    a->parts = (int)((tiles + a->tiles_per_part - 1) / a->tiles_per_part);
    *work_bytes = 0;
    if (a->parts > 1) {
        const size_t counters = join_counter_bytes();  // (rows: at most half as many as compute units)
        *work_bytes = counters + (size_t)p->rows * a->parts * LP_PART_WORDS * sizeof(unsigned long long);
        a->arrived = (int *)p->work;
        a->partial = (unsigned long long *)((char *)p->work + counters);
    }
    return GP_SUCC;
}

}  // namespace gp

using namespace gp;

extern "C" int gp_token_logprobs_work_bytes(const gp_token_logprobs_params *p, size_t *bytes) {
    LogprobsArgs a;
    size_t n;
    if (int rc = plan_token_logprobs(p, &a, &n)) return rc;
    GP_REQUIRE(bytes, "token_logprobs: no place for the size");
    *bytes = n;
    return GP_SUCC;
}

extern "C" int gp_launch_token_logprobs(const gp_token_logprobs_params *p, const gp_preempt_ctx *ctx, gp_stream s, gp_launch_info *info) {
    LogprobsArgs a;
    size_t n;
    if (int rc = plan_token_logprobs(p, &a, &n)) return rc;
    GP_REQUIRE(n == 0 || (p->work && ((uintptr_t)p->work & 15) == 0 && p->work_bytes >= n), "token_logprobs: needs a workspace of %zu bytes, 16-byte aligned", n);
    const int rows = (int)p->rows;
    switch (p->dtype) {
        case GP_F32: return launch_tiles(GP_KSET(token_logprobs_kernel<float), a.parts, rows, ctx, s, info, a, 0, 1, LP_NT);
        case GP_F16: return launch_tiles(GP_KSET(token_logprobs_kernel<_Float16), a.parts, rows, ctx, s, info, a, 0, 1, LP_NT);
        default: return launch_tiles(GP_KSET(token_logprobs_kernel<__bf16), a.parts, rows, ctx, s, info, a, 0, 1, LP_NT);
    }
}
