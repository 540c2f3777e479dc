// Attention over a paged cache for few query rows: a step of a decoder, where the cache is read once and its arithmetic is little.
//
// Bound by memory: 2 * D values of the cache per key.  So keys and values go from memory to the registers that the matrix instructions
// read, without LDS and without a barrier; the four wavefronts of a workgroup take turns over a stretch of keys, each with a running
// reference (the largest score, or a little below it) and sum of its own, and meet at its end.
//
// A tile is one head of the cache, up to 16 * NT query rows of a sequence that share it (its new tokens times the query heads of the
// head), and one of `shares` equal parts of the keys of all sequences, one sequence behind the other: how long they are only the device knows,
// and a part that ends inside a sequence leaves a result to be joined with its neighbours', by whoever of them comes last.
//
//   S^T = K Q^T    v_mfma_f32_16x16x32, K as A: lane l holds 8 values of key l % 16.  Which of the head's values a lane holds is free as long as the
//                  queries are laid out alike: 16 consecutive bytes of a key per lane and load.
//   O^T = V^T P^T  V^T as A, and P as B in the layout that S^T came out in: lane l has keys 4 * (l / 16) + 0..3 of two neighbouring tiles of
//                  16.  So lane l loads these eight rows of V, D / 16 consecutive values from (D / 16) * (l % 16) on, and a few byte permutations turn
//                  them into eight (four) A operands whose row l % 16 is the head's value (D / 16) * (l % 16) + j.
//
// Measured (32 heads, 8 cached of 128): 64 sequences of 2048 to 8192 keys, e4m3, 108 us for 625 MB, 5.8 TB/s (a kernel that only reads: 7.1; sequences of one
// length: 6.2 to 6.7, since where a sequence ends its successor's loads begin anew); one of 131072 keys, 50 us for 268 MB, of which some 10 are the chain
// length, pages, keys in front and the join of 32 parts behind; 24 sequences with 4 new tokens each, bf16, 57 us for 282 MB.
#pragma once
#include <type_traits>
#include "kv_cache.hpp"
#include "tile_loop.hpp"

namespace gp {

constexpr int FEW_WAVES = 4, FEW_NT = 64 * FEW_WAVES;
template <bool E8> constexpr int few_step_keys() { return E8 ? 64 : 32; }  // of a wavefront: 16 KB of keys and values of 128
template <bool E8> constexpr int few_unit() { return FEW_WAVES * few_step_keys<E8>(); }
constexpr int FEW_SPAN = 64 * 16 * FEW_WAVES;  // keys for which the lanes hold the pages and scales: 64 tiles of 16 for each wavefront

struct FewArgs {
    gp_paged_attention_params p;
    int group;        // query heads to a head of the cache
    int row_blocks;   // of 16 * NT rows
    int shares;       // parts of the keys, per head and row block, at most; 0: every sequence is a part
    int *arrived;     // workspace: a counter for every (head, row block, part), 0 between launches
    float *partial;   // ... and for every tile two results: 16 * NT rows of D values, then their maxima and sums
};

template <int NT, int D> constexpr int few_partial_floats() { return 16 * NT * (D + 2); }
template <int NT, int D> constexpr int few_lds_floats() { return FEW_WAVES * 16 * NT * (D + 4 + 2); }

__device__ __forceinline__ f32x4 mma16(u32x4 a, u32x4 b, f32x4 c, _Float16) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mma16(u32x4 a, u32x4 b, f32x4 c, __bf16) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
// two e4m3 values (bytes 0 and 1, or 2 and 3) in 16 bits: exact in either type
template <bool HI> __device__ __forceinline__ unsigned widen(unsigned raw, _Float16) { return __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(raw, 1.f, HI)); }
template <bool HI> __device__ __forceinline__ unsigned widen(unsigned raw, __bf16) { return __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(raw, 1.f, HI)); }

// the scale of a page's head
__device__ __forceinline__ float page_scale(const float *scales, long at) { return within_scales(scales[at]); }

// Exponents are taken against a reference m that a row's largest one, `top`, exceeds by at most `room`.  What is rounded to 16 bits for the second product is 2^(x - m).  fp16's
// numbers become fixed-point ones below 2^-14, so there m is put below the largest and may be exceeded by what fp16 has room for: beside its half unit, a probability
// is off by at most 2^-36 of the row's largest (against the largest itself by 2^-25: 131072 keys of half that each were lost, 0.2 % of their row, while the sum in the denominator
// had them).  bf16 has fp32's range.  Measured over many rows of 128, fp16: level with m at the largest, raised when it is exceeded 2^8-fold; put 14 below it, it is raised
// oftener: 592 -> 604 us.
template <typename T> struct Reference {
    static constexpr bool FP16 = std::is_same<T, _Float16>::value;
    static constexpr float room(float wanted) { return FP16 ? 15.f : wanted; }
    // (beyond 2^20, where the difference would be rounded to other steps, the largest itself)
    static __device__ __forceinline__ float below(float top) { return FP16 && fabsf(top) < 0x1p20f ? top - 11.f : top; }
};

// stores and loads of what another workgroup reads or has written within the launch
__device__ __forceinline__ void put_shared(float *p, f32x2 v) { __hip_atomic_store((unsigned long long *)p, __builtin_bit_cast(unsigned long long, v), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
__device__ __forceinline__ f32x2 get_shared(const float *p) { return __builtin_bit_cast(f32x2, __hip_atomic_load((const unsigned long long *)p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT)); }

template <typename V> __device__ __forceinline__ V load_cache(const char *p) { return __builtin_nontemporal_load((const V *)p); }

// One sequence as a block of rows sees it
struct FewSequence {
    SeqTokens s;
    int nrows;       // of the block and those behind it
    int bound, kmin, kend;  // keys; those that every row of the block sees, and that some row does
    int units;       // of few_unit keys: what the parts are made of (a sequence that sees nothing counts as one: it gets its zeros)
};
template <int ROWS, int UNIT>
__device__ __forceinline__ FewSequence few_sequence(const FewArgs &a, const SeqTokens &s, int rb) {
    const gp_paged_attention_params &p = a.p;
    FewSequence f;
    f.s = s;
    f.nrows = f.s.rows * a.group - rb * ROWS;
    f.bound = (int)seq_bound(f.s, p.max_len, p.table_width, p.cache.page_size);
    const int last = (rb * ROWS + (f.nrows < ROWS ? f.nrows : ROWS) - 1) / a.group, first = rb * ROWS / a.group;
    f.kend = (int)keys_seen(f.bound, f.s.first + last, p.causal);
    f.kmin = (int)keys_seen(f.bound, f.s.first + first, p.causal);
    f.units = f.nrows <= 0 ? 0 : f.kend <= UNIT ? 1 : (f.kend + UNIT - 1) / UNIT;
    return f;
}

// Keys [c0, kend) of one sequence; then its rows are finished, or its part of them waits in slot `slot` for the others.
// first_share, last_share: the parts that the sequence's keys are spread over.
template <typename T, int D, bool E8, int NT>
__device__ __forceinline__ void attend_stretch(const FewArgs &a, const FewSequence &f, int b, int hr, int c0, int c1, float *slot, int first_share, int last_share, float *lds) {
    // (products and sums are contracted where the code says so and nowhere else, and rounded to fp32 before they are rounded to 16 bits, so that the
    // plain and the preemptible kernels give the same bits)
#pragma clang fp contract(off)
    const gp_paged_attention_params &p = a.p;
    constexpr int KS = few_step_keys<E8>(), TILES = KS / 16, PAIRS = KS / 32;  // keys of a wavefront's step
    constexpr int ROWS = 16 * NT, VD = D / 16, KL = E8 ? D / 64 : D / 32;
    constexpr int ES = E8 ? 1 : 2;  // bytes of a value
    constexpr float ROOM = Reference<T>::room(0.f);
    typedef unsigned int VRow __attribute__((ext_vector_type(VD * ES / 4)));  // a lane's values of one key
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), col = lane & 15, g = lane >> 4;
    const int rb = hr % a.row_blocks, kvh = hr / a.row_blocks, P = p.cache.page_size;
    const SeqTokens &s = f.s;
    const int nrows = f.nrows, bound = f.bound, kmin = f.kmin, kend = c1 < f.kend ? c1 : f.kend;

    // ---- queries: column l % 16 of tile n, in the order of values that the keys are loaded in ----
    u32x4 q[NT][D / 32];
    int seen[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        const int r = rb * ROWS + n * 16 + col, token = r / a.group, hg = r - token * a.group;
        const bool there = n * 16 + col < nrows;
        seen[n] = there ? (int)keys_seen(bound, s.first + token, p.causal) : 0;
        const T *row = (const T *)p.q + (s.row0 + (there ? token : 0)) * p.ld_q + ((long)kvh * a.group + (there ? hg : 0)) * D;
#pragma unroll
        for (int k = 0; k < D / 32; ++k) {
            const int d = E8 ? 64 * (k / 2) + 16 * g + 8 * (k % 2) : 32 * k + 8 * g;
            q[n][k] = *(const u32x4 *)(row + d);
            if (!there) q[n][k] = u32x4{0, 0, 0, 0};  // (zeros, though nobody looks at them: with other rows here the multipliers draw more, 108 us become 115)
        }
    }
    f32x4 o[NT][VD];
    float m[NT], l[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        m[n] = -INFINITY; l[n] = 0.f;
#pragma unroll
        for (int j = 0; j < VD; ++j) o[n][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    const float scale2 = p.scale * 1.44269504088896340736f;  // log2(e): exponentials are powers of two
    const char *K = (const char *)p.cache.k, *V = (const char *)p.cache.v;
    const unsigned koff = (unsigned)(col * D + (E8 ? 16 : 8) * g) * ES, voff = (unsigned)(4 * g * D + VD * col) * ES;

    for (int base = c0; base < kend; base += FEW_SPAN) {
        // lane i: the page and the scales of the i-th tile of 16 keys that this wavefront takes
        const int key_of_lane = base + ((lane / TILES) * FEW_WAVES + wave) * KS + lane % TILES * 16;
        const int page_l = key_of_lane < kend ? page_of(p.page_table, p.table_width, b, key_of_lane / P, p.cache.pages) : -1;
        float ks_l = scale2, vs_l = 1.f, lv_l = 0.f;
        if constexpr (E8) {
            if (page_l >= 0) {
                const long at = (long)page_l * p.cache.kv_heads + kvh;
                ks_l = scale2 * page_scale(p.cache.k_scale, at);
                vs_l = page_scale(p.cache.v_scale, at);
            }
            lv_l = __builtin_amdgcn_logf(vs_l);
            vs_l = 1.f / vs_l;
        }
        const int left = (kend - base < FEW_SPAN ? kend - base : FEW_SPAN) - wave * KS;
        const int steps = left <= 0 ? 0 : (left + FEW_WAVES * KS - 1) / (FEW_WAVES * KS);
        u32x4 kr[TILES][KL];
        VRow vr[PAIRS][8];
        auto tile_at = [&](int step, int i) -> long {  // byte offset of the i-th tile of a step in the pool (one that is not there: page 0)
            const int at = step * TILES + i, page = __builtin_amdgcn_readlane(page_l, at);
            const int key = base + (step * FEW_WAVES + wave) * KS + i * 16;
            return (((long)(page < 0 ? 0 : page) * p.cache.kv_heads + kvh) * P + (key & (P - 1))) * D * ES;
        };
        auto load_k = [&](int step) {
#pragma unroll
            for (int i = 0; i < TILES; ++i) {
                const char *at = K + tile_at(step, i);
#pragma unroll
                for (int k = 0; k < KL; ++k) kr[i][k] = load_cache<u32x4>(at + koff + k * 64);
            }
        };
        auto load_v = [&](int step) {
#pragma unroll
            for (int pr = 0; pr < PAIRS; ++pr)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const char *at = V + tile_at(step, 2 * pr + h);
#pragma unroll
                    for (int e = 0; e < 4; ++e) vr[pr][4 * h + e] = load_cache<VRow>(at + voff + e * D * ES);
                }
        };
        if (steps > 0) { load_k(0); load_v(0); }
#pragma unroll 1
        for (int step = 0; step < steps; ++step) {
            // ---- scores of 16 keys at a time: x[n][i][e] belongs to key 4 g + e of tile i and query l % 16 ----
            f32x4 x[NT][TILES];
#pragma unroll
            for (int i = 0; i < TILES; ++i) {
#pragma unroll
                for (int n = 0; n < NT; ++n) x[n][i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int k = 0; k < KL; ++k) {
                    if constexpr (E8) {
                        const u32x4 r = kr[i][k];
                        const u32x4 k0 = {widen<false>(r[0], T()), widen<true>(r[0], T()), widen<false>(r[1], T()), widen<true>(r[1], T())};
                        const u32x4 k1 = {widen<false>(r[2], T()), widen<true>(r[2], T()), widen<false>(r[3], T()), widen<true>(r[3], T())};
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
                            x[n][i] = mma16(k0, q[n][2 * k], x[n][i], T());
                            x[n][i] = mma16(k1, q[n][2 * k + 1], x[n][i], T());
                        }
                    } else {
#pragma unroll
                        for (int n = 0; n < NT; ++n) x[n][i] = mma16(kr[i][k], q[n][k], x[n][i], T());
                    }
                }
            }
            if (step + 1 < steps) load_k(step + 1);
            // ---- masks: the keys behind a row's last, tiles that are not there, and (once for all rows) what is behind the sequence's end ----
            const int key0 = base + (step * FEW_WAVES + wave) * KS;
            float ks[TILES], lv[TILES], iv[TILES];
            bool whole = key0 + KS <= kmin && key0 + KS <= kend;
#pragma unroll
            for (int i = 0; i < TILES; ++i) {
                const int at = step * TILES + i;
                whole = whole && __builtin_amdgcn_readlane(page_l, at) >= 0;
                ks[i] = E8 ? __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, ks_l), at)) : scale2;
                lv[i] = E8 ? __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, lv_l), at)) : 0.f;
                iv[i] = E8 ? __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, vs_l), at)) : 1.f;
            }
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int i = 0; i < TILES; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e) x[n][i][e] = E8 ? fmaf(x[n][i][e], ks[i], lv[i]) : x[n][i][e] * ks[i];
            if (!whole) {
#pragma unroll
                for (int i = 0; i < TILES; ++i) {
                    const int first = key0 + i * 16;
                    int lim = __builtin_amdgcn_readlane(page_l, step * TILES + i) < 0 ? 0 : kend;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int key = first + 4 * g + e;
#pragma unroll
                        for (int n = 0; n < NT; ++n)
                            if (key >= lim || key >= seen[n]) x[n][i][e] = -INFINITY;
                        if (key >= lim) vr[i / 2][4 * (i % 2) + e] = VRow(0);
                    }
                }
            }
            // ---- running reference and sum.  8 bits: x has the logarithm of the values' scale added, so that what is rounded to 16
            // bits is the probability times that scale, at most 2^ROOM; the sum takes the scale back out ----
            u32x4 pb[NT][PAIRS];
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                float top = x[n][0][0];
#pragma unroll
                for (int i = 0; i < TILES; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e) top = fmaxf(top, x[n][i][e]);
                top = fmaxf(top, __shfl_xor(top, 16, 64));
                top = fmaxf(top, __shfl_xor(top, 32, 64));
                if (__any(top > m[n] + ROOM)) {
                    const float now = fmaxf(m[n], Reference<T>::below(top)), f = now == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m[n] - now);
                    m[n] = now;
                    l[n] *= f;
#pragma unroll
                    for (int j = 0; j < VD; ++j) o[n][j] *= f;
                }
                const float mm = m[n] == -INFINITY ? 0.f : m[n];
#pragma unroll
                for (int i = 0; i < TILES; ++i) {
                    float part = 0.f;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        x[n][i][e] = __builtin_amdgcn_exp2f(x[n][i][e] - mm);
                        part += x[n][i][e];
                    }
                    l[n] = E8 ? fmaf(part, iv[i], l[n]) : l[n] + part;
                }
#pragma unroll
                for (int pr = 0; pr < PAIRS; ++pr) {
                    typedef T tx8 __attribute__((ext_vector_type(8)));
                    tx8 y;
#pragma unroll
                    for (int e = 0; e < 4; ++e) { y[e] = Elem<T>::from_f(x[n][2 * pr][e]); y[4 + e] = Elem<T>::from_f(x[n][2 * pr + 1][e]); }
                    pb[n][pr] = __builtin_bit_cast(u32x4, y);
                }
            }
            // ---- O^T += V^T P^T ----
#pragma unroll
            for (int pr = 0; pr < PAIRS; ++pr)
#pragma unroll
                for (int j = 0; j < VD; j += 2) {
                    u32x4 v0, v1;  // of the lane's values j and j + 1, eight keys each
#pragma unroll
                    for (int kp = 0; kp < 4; ++kp) {
                        if constexpr (E8) {
                            // bytes j of two keys, then bytes j + 1
                            const unsigned two = __builtin_amdgcn_perm(vr[pr][2 * kp + 1][j / 4], vr[pr][2 * kp][j / 4], j % 4 == 0 ? 0x05010400u : 0x07030602u);
                            v0[kp] = widen<false>(two, T());
                            v1[kp] = widen<true>(two, T());
                        } else {
                            v0[kp] = __builtin_amdgcn_perm(vr[pr][2 * kp + 1][j / 2], vr[pr][2 * kp][j / 2], 0x05040100u);
                            v1[kp] = __builtin_amdgcn_perm(vr[pr][2 * kp + 1][j / 2], vr[pr][2 * kp][j / 2], 0x07060302u);
                        }
                    }
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        o[n][j] = mma16(v0, pb[n][pr], o[n][j], T());
                        o[n][j + 1] = mma16(v1, pb[n][pr], o[n][j + 1], T());
                    }
                }
            if (step + 1 < steps) load_v(step + 1);
        }
    }

    // ---- the four wavefronts' results meet: O = sum_w a_w O_w, a_w = 2^(m_w - max m), m_w its reference ----
    constexpr int LD = D + 4;
    float *ml = lds + FEW_WAVES * ROWS * LD;
    __syncthreads();  // (the previous tile's are still being read)
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        l[n] += __shfl_xor(l[n], 16, 64);
        l[n] += __shfl_xor(l[n], 32, 64);
        const int r = n * 16 + col;
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int j = 0; j < VD; j += 4)
                *(f32x4 *)(lds + (wave * ROWS + r) * LD + (4 * g + e) * VD + j) = f32x4{o[n][j][e], o[n][j + 1][e], o[n][j + 2][e], o[n][j + 3][e]};
        if (g == 0) *(f32x2 *)(ml + 2 * (wave * ROWS + r)) = f32x2{m[n], l[n]};
    }
    __syncthreads();
    const int rows = nrows < ROWS ? nrows : ROWS;
    auto finish = [&](int r, int d, f32x4 v, float sum) {
        const int rr = rb * ROWS + r, token = rr / a.group, hg = rr - token * a.group;
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        typedef T tx4 __attribute__((ext_vector_type(4)));
        tx4 y;
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = Elem<T>::from_f(rounded(v[e] * inv));
        *(tx4 *)((T *)p.out + (s.row0 + token) * p.ld_out + ((long)kvh * a.group + hg) * D + d) = y;
    };
    const int parts = last_share - first_share + 1;
    for (int u = tid; u < rows * (D / 4); u += FEW_NT) {
        const int r = u / (D / 4), d = u % (D / 4) * 4;
        float top = -INFINITY, sum = 0.f;
#pragma unroll
        for (int w = 0; w < FEW_WAVES; ++w) top = fmaxf(top, ml[2 * (w * ROWS + r)]);
        const float base = top == -INFINITY ? 0.f : top;
        f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < FEW_WAVES; ++w) {
            const f32x2 x = *(const f32x2 *)(ml + 2 * (w * ROWS + r));
            const float f = __builtin_amdgcn_exp2f(x[0] - base);
            sum = fmaf(f, x[1], sum);
            const f32x4 y = *(const f32x4 *)(lds + (w * ROWS + r) * LD + d);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = fmaf(f, y[e], v[e]);
        }
        if (parts == 1) finish(r, d, v, sum);
        else {
            put_shared(slot + r * D + d, f32x2{v[0], v[1]});
            put_shared(slot + r * D + d + 2, f32x2{v[2], v[3]});
            if (d == 0) put_shared(slot + ROWS * D + 2 * r, f32x2{top, sum});
        }
    }
    if (parts == 1) return;
    // ---- whoever comes last joins the parts, in their order ----
    __shared__ int came;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the stores above have reached the memory that all XCDs see
    __syncthreads();
    int *arrived = a.arrived + (long)hr * a.shares + first_share;  // (of the one sequence that goes on behind that part)
    if (tid == 0) came = __hip_atomic_fetch_add(arrived, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    if (came != parts - 1) return;
    if (tid == 0) __hip_atomic_store(arrived, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    // (up to FEW_JOIN of them at a time: first their factors, which every thread needs, then their values, eight loads of a thread in flight.
    // A part that no row saw anything of has factor 0, and its values are zeros.)
    const float *all = a.partial + ((long)hr * a.shares + first_share) * 2 * few_partial_floats<NT, D>();
    auto part_at = [&](int i) { return all + (2l * i + (i == 0)) * few_partial_floats<NT, D>(); };  // the first part is what its tile did last
    constexpr int FEW_JOIN = few_lds_floats<NT, D>() / (2 * ROWS) < 256 ? few_lds_floats<NT, D>() / (2 * ROWS) : 256;
    constexpr int ITEMS = (ROWS * D / 4 + FEW_NT - 1) / FEW_NT;  // of a thread: four values of one row
    f32x4 v[ITEMS];
    float top[ITEMS], sum[ITEMS];
#pragma unroll
    for (int k = 0; k < ITEMS; ++k) { v[k] = f32x4{0.f, 0.f, 0.f, 0.f}; top[k] = -INFINITY; sum[k] = 0.f; }
    for (int i0 = 0; i0 < parts; i0 += FEW_JOIN) {
        const int n = parts - i0 < FEW_JOIN ? parts - i0 : FEW_JOIN;
        __syncthreads();
        for (int u = tid; u < n * rows; u += FEW_NT) {
            const int i = u / rows, r = u - i * rows;
            *(f32x2 *)(lds + 2 * (i * ROWS + r)) = get_shared(part_at(i0 + i) + ROWS * D + 2 * r);
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < ITEMS; ++k) {
            const int u = tid + k * FEW_NT, r = u / (D / 4), d = u % (D / 4) * 4;
            if (r >= rows) continue;
            float now = top[k];
            for (int i = 0; i < n; ++i) now = fmaxf(now, lds[2 * (i * ROWS + r)]);
            const float base = now == -INFINITY ? 0.f : now, f0 = __builtin_amdgcn_exp2f(top[k] - base);
            top[k] = now;
            sum[k] *= f0;
            v[k] *= f0;
            for (int i = 0; i < n; i += 8) {
                f32x2 y[8][2];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float *from = part_at(i0 + (i + e < n ? i + e : i)) + r * D + d;
                    y[e][0] = get_shared(from);
                    y[e][1] = get_shared(from + 2);
                }
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    if (i + e >= n) break;
                    const f32x2 ms = *(const f32x2 *)(lds + 2 * ((i + e) * ROWS + r));
                    const float f = __builtin_amdgcn_exp2f(ms[0] - base);
                    sum[k] = fmaf(f, ms[1], sum[k]);
#pragma unroll
                    for (int c = 0; c < 4; ++c) v[k][c] = fmaf(f, y[e][c / 2][c % 2], v[k][c]);
                }
            }
        }
    }
#pragma unroll
    for (int k = 0; k < ITEMS; ++k) {
        const int u = tid + k * FEW_NT, r = u / (D / 4), d = u % (D / 4) * 4;
        if (r < rows) finish(r, d, v[k], sum[k]);
    }
}

template <typename T, int D, bool E8, int NT>
__device__ __forceinline__ void attend_few(const FewArgs &a, TileIdx t, float *lds) {
    const gp_paged_attention_params &p = a.p;
    constexpr int ROWS = 16 * NT, UNIT = few_unit<E8>();
    const int lane = threadIdx.x & 63, hr = t.y, rb = hr % a.row_blocks, batch = p.batch;
    if (a.shares == 0) {  // a tile per sequence
        const FewSequence f = few_sequence<ROWS, UNIT>(a, seq_tokens(p.start, p.kv_len, t.x, p.tokens, p.max_new), rb);
        if (f.nrows > 0) attend_stretch<T, D, E8, NT>(a, f, t.x, hr, 0, f.kend, nullptr, 0, 0, lds);
        return;
    }
    // ---- all units; then the sequence in which this part begins.  Every wavefront for itself, 64 sequences at a time, one to a lane ----
    int r0, r1, len;  // of the lane's sequence
    auto look = [&](int b0) {
        const int b = b0 + lane < batch ? b0 + lane : batch - 1;
        r0 = p.start ? p.start[b] : b;
        r1 = p.start ? p.start[b + 1] : b + 1;
        len = p.kv_len[b];
        return b0 + lane < batch ? few_sequence<ROWS, UNIT>(a, seq_tokens_of(r0, r1, len, p.tokens, p.max_new), rb).units : 0;
    };
    int total = 0, n = 0;
    for (int b0 = batch <= 64 ? 0 : (batch - 1) / 64 * 64; b0 >= 0; b0 -= 64) total += n = look(b0);  // (the first 64 last: they are looked at next)
#pragma unroll
    for (int d = 1; d < 64; d *= 2) total += __shfl_xor(total, d, 64);
    total = __builtin_amdgcn_readfirstlane(total);
    // (joining a part costs as much as a few units, more for more rows.  Us in parts of two units / of four at least, 32 query heads over 8 cached ones of 128: one new token, which is 4 rows,
    // over 1000 keys, bf16, 10.8 / 12.8; over 4000 and 16000, e4m3, 12.5 / 15.7 and 17.2 / 19.1; eight new tokens, which are 32 rows, 17.3 / 19.0, 22.7 / 25.2 and 39.3 / 33.2; over
    // 131072 level, 50 and 82)
    constexpr int LEAST = NT == 1 ? 2 : 4;
    const int shares = total / LEAST < 1 ? 1 : total / LEAST < a.shares ? total / LEAST : a.shares;
    if (total == 0 || t.x >= shares) return;  // (no sequence has rows in this block)
    const int lo = part_begin(t.x, total, shares), hi = part_begin(t.x + 1, total, shares);
    float *slots = a.partial + ((long)hr * a.shares + t.x) * 2 * few_partial_floats<NT, D>();
    walk_part(batch, 64, lo, hi, [&](int b0, int unit, int &at, int &i) {
        if (b0) n = look(b0);
        int upto = n;
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
            const int x = __shfl_up(upto, d, 64);
            if (lane >= d) upto += x;
        }
        const unsigned long long behind = __ballot(at + upto > unit);
        if (behind) i = __builtin_ctzll(behind);
        at += behind ? __builtin_amdgcn_readlane(upto - n, i) : __builtin_amdgcn_readlane(upto, 63);
        return behind != 0;
    }, look, [&](int b, int i, int at) {
        const FewSequence f = few_sequence<ROWS, UNIT>(a, seq_tokens_of(__builtin_amdgcn_readlane(r0, i), __builtin_amdgcn_readlane(r1, i), __builtin_amdgcn_readlane(len, i), p.tokens, p.max_new), rb);
        if (f.units == 0) return 0;
        const int u0 = lo > at ? lo - at : 0, u1 = hi - at < f.units ? hi - at : f.units;
        attend_stretch<T, D, E8, NT>(a, f, b, hr, u0 * UNIT, u1 == f.units ? f.kend : u1 * UNIT, slots + (u0 == 0) * few_partial_floats<NT, D>(),
                                     part_of(at, total, shares), part_of(at + f.units - 1l, total, shares), lds);
        return f.units;
    });
}

template <typename T, int D, bool E8, int NT, int LOOP = LOOP_ANY>
__global__ __launch_bounds__(FEW_NT, 2) void paged_few_kernel(FewArgs a, BlpArgs blp) {
    extern __shared__ __attribute__((aligned(16))) unsigned char few_lds[];
    tiles<LOOP>(blp, [&](TileIdx t) { attend_few<T, D, E8, NT>(a, t, (float *)few_lds); });
}

}  // namespace gp
