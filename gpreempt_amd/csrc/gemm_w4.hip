// Products of a few rows of activations with a matrix of 4-bit numbers: C = act(A W^T + bias + residual), W[n, k] = s[n, g] (q[n, k] - z[n, g]), g = k / group.
//
// ---- few rows ----
// Bound by memory: half a byte of W per 2 M flop.  So the numbers go from memory to the registers that the matrix instructions read, without LDS and without a barrier in the loop.  A byte 0000qqqq
// is the e4m3 number 2^-9 q (fixed-point below 8, with an exponent from there on), so an instruction of the 8-bit caches widens two of them to fp16 or bf16, exactly.  Zeros are a second product,
// with -2^-9 z everywhere in its other operand, and scales come in once per group, in fp32:
//   C = 2^9 sum_g s_g (sum_k a 2^-9 q + sum_k a (-2^-9 z_g)).
// Nothing is rounded to 16 bits but the result.
//
// A tile is 16 * NT rows of W and up to 16 * MT rows of A.  Its wavefronts take an equal part of the values of a row each, 128 at a time, and add their sums up in LDS, in their order.
//   v_mfma_f32_16x16x32   A as A: lane l has 8 values of row l % 16; W as B: lane l has 8 values of row l % 16 of W; the result's column l % 16 is a row of W, so a lane has one
//                         scale per group.  A lane fetches 16 bytes of W, 32 neighbours, and the four groups of 16 lanes exchange what they have, so that an instruction takes 32
//                         neighbours of W and of A: within a group, and a row of A's in one piece.
// Measured: 1 x 22528 x 4096, bf16, groups of 128: 15 us for 48 MB; 5 x 131001 x 4096, groups of 32, 85 us for 304 MB, 3.6 TB/s, of 128, 64 us, 4.4 TB/s: beside W, what is fetched of A and the vector
// instructions (50 to 75 for 16 x 128 of W) take a share of the time that deeper prefetching, or A through LDS (a barrier a step: 68 -> 84 us, of 128), did not hide.
#include "kv_cache.hpp"
#include "paged_few.hpp"
#include "launch_tiles.hpp"

namespace gp {

constexpr int W4_CHUNK = 128;  // values of a wavefront's step
constexpr int W4_PANEL = 256;  // groups whose scales are in LDS at a time

struct W4Args {
    gp_gemm_w4_params p;
    int groups;  // of a row
    int panel;   // of them, at a time
    int rows, cols;  // tiles (many rows)
};
inline __host__ __device__ int w4_scale_stride(int panel) { return panel + 1; }
template <int MT, int NT, int WAVES> inline size_t w4_lds_bytes(int panel) {
    return std::max((size_t)16 * NT * w4_scale_stride(panel) * sizeof(unsigned), (size_t)WAVES * 256 * MT * NT * sizeof(float));
}

// What is not finite must not come out as a number: apply_act's ReLU takes NaN to 0, and an infinite scale times a group's negative sum to 0 too, where scale * (q - zero) in front of the sum has both
// signs.  So NaN stays NaN, and an infinite scale is one.
template <typename T> __device__ __forceinline__ T finite_or_nan(T scale) { return Elem<T>::from_f(fmaf(Elem<T>::to_f(scale), 0.f, Elem<T>::to_f(scale))); }
__device__ __forceinline__ float act_of_sum(float v, int act) { return act == GP_ACT_RELU ? (v <= 0.f ? 0.f : v) : apply_act(v, act); }

// rows r0 .. r3 of a 4 x 4 matrix of (registers, groups of 16 lanes) become its columns
__device__ __forceinline__ void transpose_lane_groups(u32x4 &r) {
    auto swap32 = [](unsigned &x, unsigned &y) { const auto s = __builtin_amdgcn_permlane32_swap(x, y, false, false); x = s[0]; y = s[1]; };
    auto swap16 = [](unsigned &x, unsigned &y) { const auto s = __builtin_amdgcn_permlane16_swap(x, y, false, false); x = s[0]; y = s[1]; };
    unsigned a = r[0], b = r[1], c = r[2], d = r[3];
    swap32(a, c);
    swap32(b, d);
    swap16(a, b);
    swap16(c, d);
    r = u32x4{a, b, c, d};
}

// eight 4-bit numbers as 2^-9 times themselves, in their order
template <typename T> __device__ __forceinline__ u32x4 widen_nibbles(unsigned raw) {
    const unsigned even = raw & 0x0F0F0F0Fu, odd = (raw >> 4) & 0x0F0F0F0Fu;
    const unsigned x = __builtin_amdgcn_perm(odd, even, 0x05010400u), y = __builtin_amdgcn_perm(odd, even, 0x07030602u);
    return u32x4{widen<false>(x, T()), widen<true>(x, T()), widen<false>(y, T()), widen<true>(y, T())};
}

template <typename T, int G, int MT, int NT, int WAVES>
__device__ __forceinline__ void w4_tile(const W4Args &a, TileIdx t, char *lds) {
#pragma clang fp contract(off)  // (the plain and the preemptible kernels give the same bits)
    const gp_gemm_w4_params &p = a.p;
    constexpr bool WHOLE = G == W4_CHUNK;  // (K is a multiple of a step)
    constexpr int PER = G / 32;  // instructions to a group
    constexpr int AHEAD_A = MT == 1 && NT == 4 ? 2 : 1, AHEAD = NT == 4 ? 2 : 4;  // steps that A and that W is fetched ahead
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), col = lane & 15, g = lane >> 4;
    const int n0 = t.x * 16 * NT, m0 = t.y * 16 * MT;
    const unsigned char *w[NT];
    const T *x[MT];
#pragma unroll
    for (int i = 0; i < NT; ++i) {
        const int n = n0 + 16 * i + col;
        w[i] = (const unsigned char *)p.W + (long)(n < p.N ? n : p.N - 1) * p.ldw;
    }
#pragma unroll
    for (int i = 0; i < MT; ++i) {
        const int m = m0 + 16 * i + col;
        x[i] = (const T *)p.A + (long)(m < p.M ? m : p.M - 1) * p.lda + 8 * g;
    }
    f32x4 total[MT][NT];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) total[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    typedef T tx2 __attribute__((ext_vector_type(2)));
    unsigned *scales = (unsigned *)lds;  // a group's scale, and -2^-9 times its zero
    const int stride = w4_scale_stride(a.panel);

    for (int g0 = 0; g0 < a.groups; g0 += a.panel) {
        const int gn = a.groups - g0 < a.panel ? a.groups - g0 : a.panel, len = gn * G;
        const long k0 = (long)g0 * G;
        const int chunks = (len + W4_CHUNK - 1) / W4_CHUNK, c0 = wave * chunks / WAVES, c1 = (wave + 1) * chunks / WAVES;
        u32x4 raw[AHEAD][NT], act[AHEAD_A][MT][4];
        auto load_w = [&](int c, u32x4 (&r)[NT]) {
            const int at = 64 * c + 16 * g, last = len / 2 - 16;  // (what is behind the row's end is not multiplied)
#pragma unroll
            for (int i = 0; i < NT; ++i) r[i] = *(const u32x4 *)(w[i] + k0 / 2 + (at < last ? at : last));
        };
        auto load_a = [&](int c, int j, u32x4 (&to)[MT][4]) {
            const int at = c * W4_CHUNK + 32 * j;
            if (!WHOLE && at >= len) return;
#pragma unroll
            for (int i = 0; i < MT; ++i) to[i][j] = *(const u32x4 *)(x[i] + k0 + at);
        };
#pragma unroll
        for (int d = 0; d < AHEAD; ++d)
            if (c0 + d < c1) load_w(c0 + d, raw[d]);
#pragma unroll
        for (int d = 0; d < AHEAD_A; ++d)
            if (c0 + d < c1) {
#pragma unroll
                for (int j = 0; j < 4; ++j) load_a(c0 + d, j, act[d]);
            }
        __syncthreads();  // (what is in LDS is still being read)
        // (eight neighbouring groups of a row to a thread; rows start anywhere)
        typedef T Eight __attribute__((ext_vector_type(8), aligned(sizeof(T))));
        typedef unsigned char Bytes __attribute__((ext_vector_type(8), aligned(1)));
        const int per_row = (gn + 7) / 8;
#pragma unroll 2
        for (int u = tid; u < 16 * NT * per_row; u += 64 * WAVES) {
            const int r = u / per_row, at = (u - r * per_row) * 8, n = n0 + r < p.N ? n0 + r : p.N - 1;
            const T *from = (const T *)p.scales + (long)n * p.ld_scales + g0 + at;
            const uint8_t *zero = p.zeros ? p.zeros + (long)n * p.ld_zeros + g0 + at : nullptr;
            Eight s = {};
            Bytes z = {8, 8, 8, 8, 8, 8, 8, 8};
            if (at + 8 <= gn) {
                s = *(const Eight *)from;
                if (zero) z = *(const Bytes *)zero;
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) {  // (behind the last one that one again, so that all are fetched at once)
                    const int i = at + e < gn ? e : gn - 1 - at;
                    s[e] = from[i];
                    if (zero) z[e] = zero[i];
                }
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const T minus = Elem<T>::from_f((float)z[e] * -0x1p-9f);  // (exact: a whole number of eight bits)
                if (at + e < gn) scales[r * stride + at + e] = __builtin_bit_cast(unsigned, tx2{finite_or_nan((T)s[e]), minus});
            }
        }
        __syncthreads();
        auto chunk = [&](int c, u32x4 (&r)[NT], u32x4 (&a)[MT][4]) {
            f32x4 acc[MT][NT];
            unsigned sz[NT];
#pragma unroll
            for (int i = 0; i < NT; ++i) transpose_lane_groups(r[i]);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (!WHOLE && c * W4_CHUNK + 32 * j >= len) break;
                if (j % PER == 0) {
#pragma unroll
                    for (int k = 0; k < NT; ++k) sz[k] = scales[(16 * k + col) * stride + (c * W4_CHUNK + 32 * j) / G];
                }
#pragma unroll
                for (int k = 0; k < NT; ++k) {
                    const u32x4 b = widen_nibbles<T>(r[k][j]);
                    const unsigned zero = __builtin_amdgcn_perm(sz[k], sz[k], 0x07060706u);
#pragma unroll
                    for (int i = 0; i < MT; ++i) {
                        acc[i][k] = mma16(a[i][j], u32x4{zero, zero, zero, zero}, j % PER == 0 ? f32x4{0.f, 0.f, 0.f, 0.f} : acc[i][k], T());
                        acc[i][k] = mma16(a[i][j], b, acc[i][k], T());
                    }
                }
                if (c + AHEAD_A < c1) load_a(c + AHEAD_A, j, a);
                if (j % PER == PER - 1) {
#pragma unroll
                    for (int k = 0; k < NT; ++k) {
                        const tx2 both = __builtin_bit_cast(tx2, sz[k]);
                        const float scale = Elem<T>::to_f(both[0]);
#pragma unroll
                        for (int i = 0; i < MT; ++i)
#pragma unroll
                            for (int e = 0; e < 4; ++e) total[i][k][e] = fmaf(scale, acc[i][k][e], total[i][k][e]);
                    }
                }
            }
            if (c + AHEAD < c1) load_w(c + AHEAD, r);
        };
        for (int c = c0; c < c1; c += AHEAD)
            static_for<0, AHEAD>([&](auto d) {
                if (c + d < c1) chunk(c + d, raw[d], act[d % AHEAD_A]);
            });
    }

    // ---- the wavefronts' sums, in their order ----
    float *red = (float *)lds;
    constexpr int COLS = 16 * NT, TILE = 16 * MT * COLS;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int k = 0; k < NT; ++k)
#pragma unroll
            for (int e = 0; e < 4; ++e) red[wave * TILE + (16 * i + 4 * g + e) * COLS + 16 * k + col] = total[i][k][e];
    __syncthreads();
    const int rows = p.M - m0 < 16 * MT ? p.M - m0 : 16 * MT;
    for (int u = tid; u < rows * COLS; u += 64 * WAVES) {
        const int m = m0 + u / COLS, n = n0 + u % COLS;
        float v = 0.f;
#pragma unroll
        for (int k = 0; k < WAVES; ++k) v += red[k * TILE + u];
        if (n >= p.N) continue;
        v *= 512.f;
        const long at = m * p.ldc + n;
        if (p.bias) v += Elem<T>::to_f(((const T *)p.bias)[n]);
        if (p.residual) v += Elem<T>::to_f(((const T *)p.residual)[at]);
        ((T *)p.C)[at] = Elem<T>::from_f(rounded(act_of_sum(v, p.act)));
    }
}

template <typename T, int G, int MT, int NT, int WAVES, int LOOP = LOOP_ANY>
__global__ __launch_bounds__(64 * WAVES, MT * NT > 2 ? 2 : 4) void gemm_w4_kernel(W4Args a, BlpArgs blp) {
    extern __shared__ __attribute__((aligned(16))) unsigned char w4_lds[];
    tiles<LOOP>(blp, [&](TileIdx t) { w4_tile<T, G, MT, NT, WAVES>(a, t, (char *)w4_lds); });
}

// ---- many rows ----
// Bound by the vector instructions that make 16-bit numbers of W's (23 for eight numbers in bf16, 13 in fp16, which 128 rows of A share) and scale the groups' sums (16 for 32 x 32 results and a group),
// and by the matrix instructions, which seldom overlap with them.  A tile is 128 rows of A and 128 of W, a quarter of these to a wavefront, which has what it takes of W in registers; A comes through
// LDS, 128 values of a row at a time in two buffers.
//   v_mfma_f32_32x32x16   A as A, W as B: lane l has 8 values of row l % 32.
// The products are of A with q - z, whole numbers of eight bits and exact; a group's sum meets its scale in fp32: nothing is rounded to 16 bits but the result, as for few rows.
// Measured (rounding scale * (q - z) to 16 bits in front of the products in brackets): 4001 x 8192 x 8192, bf16, groups of 128: 640 to 706 us, 760 to 840 TFLOP/s (571 to 577); fp16 633 to 667 (568 to 604); of 64 736 to 743 (614 to 633); of 32 861 to 901 (606 to 622);
// 2048 x 4096 x 4096 82 to 92 (88 to 93), 1024 x 4096 x 4096 62 (72), 128 x 22528 x 4096 58 (68).  Tiles of 256 x 256 in eight wavefronts, one to a compute unit: 645, of 64 642, of 32 797, 2048 x 4096 x 4096 174.  Widening W a step
// ahead between the matrix instructions: 687.
constexpr int W4M_ROWS = 128, W4M_NT = 256, W4M_STEP = 128;
constexpr int W4M_BUFFER = W4M_ROWS * W4M_STEP * 2;  // bytes
constexpr int W4M_BAND = 8;  // rows of tiles that are worked on side by side

// eight 4-bit numbers minus `zero`, in their order: whole numbers of eight bits, exact in either type
__device__ __forceinline__ u32x4 less_zero(unsigned raw, float zero, __bf16) {
    unsigned even = raw & 0x0F0F0F0Fu, odd = (raw >> 4) & 0x0F0F0F0Fu;
    asm("" : "+v"(even), "+v"(odd));  // (a byte to fp32 is one instruction; the compiler goes back to `raw`, and shifts and masks for each of them)
    typedef __bf16 tx2 __attribute__((ext_vector_type(2)));
    u32x4 y;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const f32x2 x = {(float)(even >> (8 * i) & 255u) - zero, (float)(odd >> (8 * i) & 255u) - zero};
        y[i] = __builtin_bit_cast(unsigned, __builtin_convertvector(x, tx2));
    }
    return y;
}
__device__ __forceinline__ u32x4 less_zero(unsigned raw, float zero, _Float16) {
    const unsigned even = raw & 0x0F0F0F0Fu, odd = (raw >> 4) & 0x0F0F0F0Fu;
    const unsigned x = __builtin_amdgcn_perm(odd, even, 0x05010400u), y = __builtin_amdgcn_perm(odd, even, 0x07030602u);
    const _Float16 z = (_Float16)(1024.f + zero);
    const f16x2 zz = {z, z};
    // (the bits 0x6400 + n are 1024 + n)
    auto pair = [&](unsigned bytes, unsigned pick) { return __builtin_bit_cast(unsigned, __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, bytes, pick)) - zz); };
    return u32x4{pair(x, 0x04010400u), pair(x, 0x04030402u), pair(y, 0x04010400u), pair(y, 0x04030402u)};
}

template <typename T, int G>
__device__ __forceinline__ void w4_many_tile(const W4Args &a, int tile_m, int tile_n, char *lds) {
#pragma clang fp contract(off)
    const gp_gemm_w4_params &p = a.p;
    constexpr bool WHOLE = G == W4M_STEP;  // (K is a multiple of a step)
    constexpr int MB = W4M_ROWS / 32, GROUPS = W4M_STEP / G, SLICES = G / 16;  // of a step; instructions of a group
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), l32 = lane & 31, half = lane >> 5;
    const int m0 = tile_m * W4M_ROWS, n = (tile_n * 4 + wave) * 32 + l32, row_of_w = n < p.N ? n : p.N - 1;
    const unsigned char *w = (const unsigned char *)p.W + (long)row_of_w * p.ldw;
    const T *scale = (const T *)p.scales + (long)row_of_w * p.ld_scales;
    const unsigned char *zero = p.zeros ? p.zeros + (long)row_of_w * p.ld_zeros : w;  // (where there are none, something is fetched all the same and left: no branch in the loop)
    f32x16 total[MB];
#pragma unroll
    for (int i = 0; i < MB; ++i)
#pragma unroll
        for (int v = 0; v < 16; ++v) total[i][v] = 0.f;
    const int steps = (p.K + W4M_STEP - 1) / W4M_STEP;
    // ---- A: thread (row tid / 16 + 16 i, 16 bytes tid % 16) ----
    const int chunk = tid % 16, row = tid / 16;
    const int slot = row * 256 + ((chunk ^ row) & 15) * 16;
    const T *x0 = (const T *)p.A + chunk * 8;
    u32x4 ar[8];
    auto load_a = [&](int step) {  // (what is behind the rows' end is not multiplied: the row's first values instead)
        const int k = step * W4M_STEP + chunk * 8;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int m = m0 + row + 16 * i;
            ar[i] = *(const u32x4 *)(x0 + (long)(m < p.M ? m : p.M - 1) * p.lda + (WHOLE || k < p.K ? step * W4M_STEP : -chunk * 8));
        }
    };
    auto store_a = [&](char *buf) {
#pragma unroll
        for (int i = 0; i < 8; ++i) *(u32x4 *)(buf + slot + i * 16 * 256) = ar[i];
    };
    // ---- W: of 64 values the lane's 32; the step's scales and zeros ----
    u32x4 raw[2];
    T sc[GROUPS];
    unsigned char ze[GROUPS];
    auto load_w = [&](int step) {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const int k = step * W4M_STEP + 64 * t + 32 * half;
            raw[t] = *(const u32x4 *)(w + (WHOLE || k < p.K ? k / 2 : 0));
        }
#pragma unroll
        for (int g = 0; g < GROUPS; ++g) {
            const int at = step * GROUPS + g < a.groups ? step * GROUPS + g : 0;
            sc[g] = scale[at];
            ze[g] = zero[at];
        }
    };
    load_a(0);
    load_w(0);
    __syncthreads();  // (the previous tile's buffers are still being read)
    store_a(lds);
    __syncthreads();
    for (int step = 0; step < steps; ++step) {
        const char *buf = lds + step % 2 * W4M_BUFFER;
        const int next = step + 1 < steps ? step + 1 : step;  // (behind the last step: the last one again, which nobody reads)
        load_a(next);
        float s[GROUPS], z[GROUPS];
#pragma unroll
        for (int g = 0; g < GROUPS; ++g) {
            s[g] = Elem<T>::to_f(finite_or_nan(sc[g]));
            z[g] = p.zeros ? (float)ze[g] : 8.f;
        }
        // (the halves of a wavefront exchange what they have, so that an instruction takes 16 neighbours: within a group)
        unsigned mine[2][4];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const auto x = __builtin_amdgcn_permlane32_swap(raw[t][0], raw[t][1], false, false), y = __builtin_amdgcn_permlane32_swap(raw[t][2], raw[t][3], false, false);
            mine[t][0] = x[0]; mine[t][1] = y[0]; mine[t][2] = x[1]; mine[t][3] = y[1];
        }
        load_w(next);
#pragma unroll
        for (int g = 0; g < GROUPS; ++g) {
            if (!WHOLE && step * GROUPS + g >= a.groups) break;
            u32x4 b[SLICES];
#pragma unroll
            for (int j = 0; j < SLICES; ++j) b[j] = less_zero(mine[(g * SLICES + j) / 4][(g * SLICES + j) % 4], z[g], T());
#pragma unroll
            for (int i = 0; i < MB; ++i) {
                f32x16 acc;
#pragma unroll
                for (int v = 0; v < 16; ++v) acc[v] = 0.f;
#pragma unroll
                for (int j = 0; j < SLICES; ++j)
                    Elem<T>::mma(*(const u32x4 *)(buf + (32 * i + l32) * 256 + (((2 * (g * SLICES + j) + half) ^ l32) & 15) * 16), b[j], acc);
#pragma unroll
                for (int v = 0; v < 16; ++v) total[i][v] = fmaf(s[g], acc[v], total[i][v]);
            }
        }
        store_a(lds + (step + 1) % 2 * W4M_BUFFER);
        __syncthreads();
    }
    // ---- total[i][v]: row 32 i + 8 (v / 4) + 4 half + v % 4 of the tile, the lane's row of W ----
    if (n >= p.N) return;
    const float bias = p.bias ? Elem<T>::to_f(((const T *)p.bias)[n]) : 0.f;
#pragma unroll
    for (int i = 0; i < MB; ++i)
#pragma unroll
        for (int v = 0; v < 16; ++v) {
            const int m = m0 + 32 * i + 8 * (v / 4) + 4 * half + v % 4;
            if (m >= p.M) continue;
            const long at = m * p.ldc + n;
            float y = total[i][v];
            if (p.bias) y += bias;
            if (p.residual) y += Elem<T>::to_f(((const T *)p.residual)[at]);
            ((T *)p.C)[at] = Elem<T>::from_f(rounded(act_of_sum(y, p.act)));
        }
}

template <typename T, int G, int LOOP = LOOP_ANY>
__global__ __launch_bounds__(W4M_NT, 2) void gemm_w4_many_kernel(W4Args a, BlpArgs blp) {
    extern __shared__ __attribute__((aligned(16))) unsigned char w4_lds[];
    tiles<LOOP>(blp, [&](TileIdx t) {
        // (bands of tiles: neighbours share rows of A and of W)
        const int band = t.x / (W4M_BAND * a.cols), in = t.x - band * W4M_BAND * a.cols, high = a.rows - band * W4M_BAND < W4M_BAND ? a.rows - band * W4M_BAND : W4M_BAND;
        w4_many_tile<T, G>(a, band * W4M_BAND + in % high, in / high, (char *)w4_lds);
    });
}

template <typename T, int G>
static int launch_w4_many(W4Args a, const gp_preempt_ctx *ctx, gp_stream s, gp_launch_info *info) {
    a.rows = (int)(((long)a.p.M + W4M_ROWS - 1) / W4M_ROWS);
    a.cols = (int)(((long)a.p.N + 127) / 128);
    GP_REQUIRE((long)a.rows * a.cols < (1L << 31) && (long)a.cols * W4M_BAND < (1L << 31), "gemm_w4: too large");
    return launch_tiles(GP_KSET(gemm_w4_many_kernel<T, G), a.rows * a.cols, 1, ctx, s, info, a, 2 * W4M_BUFFER, 1, W4M_NT);
}

template <typename T, int G, int MT, int NT, int WAVES>
static int launch_w4(const W4Args &a, const gp_preempt_ctx *ctx, gp_stream s, gp_launch_info *info) {
    const long nx = ((long)a.p.N + 16 * NT - 1) / (16 * NT), ny = ((long)a.p.M + 16 * MT - 1) / (16 * MT);
    GP_REQUIRE(nx * ny < (1L << 31), "gemm_w4: too large");
    return launch_tiles(GP_KSET(gemm_w4_kernel<T, G, MT, NT, WAVES), (int)nx, (int)ny, ctx, s, info, a, w4_lds_bytes<MT, NT, WAVES>(a.panel), 1, 64 * WAVES);
}

template <typename T, int G>
static int choose_w4(const W4Args &a, const gp_preempt_ctx *ctx, gp_stream s, gp_launch_info *info) {
    // Many rows' tiles of 128 x 128, or few rows at a time, in tiles of up to 64 x 16: the first takes 50 (groups of 128), 60 (64), 90 us (32) for K = 4096 as long as the chip is not full, the second goes by how
    // many there are.  Us, many / few, bf16 (fp16 within 5 %), K = 4096, tiles of 64 x 16 in brackets: groups of 128: 128 x 4096 (512) 51 / 38, 400 x 1400 (616) 52 / 53, 600 x 1000 (630) 57 / 53, 65 x 6700
    // (838) 49 / 71, 256 x 4096 (1024) 51 / 72, 72 x 22528 (2816) 56 / 103; of 64: 616 61 / 54, 838 60 / 74, 1024 61 / 75; of 32: 838 88 / 72, 1024 89 / 72, 128 x 9200 (1150) 92 / 90, 128 x 11000 (1376) 97 / 108.
    const long tiles = ((long)a.p.M + 63) / 64 * (((long)a.p.N + 15) / 16);
    if (a.p.M > 64 && 4 * tiles >= (G == 128 ? 10l : G == 64 ? 12l : 18l) * device_cus()) return launch_w4_many<T, G>(a, ctx, s, info);
    // Rows of W for each wavefront, and wavefronts: what is fetched of A counts as much as W does, so a wavefront takes several rows' sixteens at once where there are enough of them for all compute
    // units.  Us (K = 4096, groups of 128, bf16) in tiles of 16 rows for 8 wavefronts / 32 for 4 / 64 for 4: 1 x 4096 6.0 / 8.2 / 10.6, 1 x 22528 19 / 16.2 / 17.0, 5 x 131001 104 / 87 / 68,
    // 24 x 4096 10.6 / 12 / 15, 24 x 22528 48 / 35 / 27, 24 x 131001 246 / 178 / 107, 64 x 4096 19 / 24, 64 x 22528 106 / 57.
    const long sixteens = ((long)a.p.N + 15) / 16;
    if (sixteens < 4l * device_cus())
        return a.p.M <= 16 ? launch_w4<T, G, 1, 1, 8>(a, ctx, s, info) : a.p.M <= 32 ? launch_w4<T, G, 2, 1, 8>(a, ctx, s, info) : launch_w4<T, G, 4, 1, 8>(a, ctx, s, info);
    if (a.p.M > 32) return launch_w4<T, G, 4, 2, 4>(a, ctx, s, info);
    if (a.p.M > 16) return launch_w4<T, G, 2, 4, 4>(a, ctx, s, info);
    return sixteens < 16l * device_cus() ? launch_w4<T, G, 1, 2, 4>(a, ctx, s, info) : launch_w4<T, G, 1, 4, 4>(a, ctx, s, info);
}

}  // namespace gp

using namespace gp;

extern "C" int gp_launch_gemm_w4(const gp_gemm_w4_params *p, const gp_preempt_ctx *ctx, gp_stream s, gp_launch_info *info) {
    GP_REQUIRE(p && p->A && p->W && p->scales && p->C, "null gemm_w4 params");
    GP_REQUIRE(p->dtype == GP_F16 || p->dtype == GP_BF16, "gemm_w4: fp16 or bf16 only (dtype %d)", p->dtype);
    GP_REQUIRE(p->M > 0 && p->N > 0 && p->K > 0, "gemm_w4: M, N and K must be positive");
    GP_REQUIRE(p->M <= (1 << 30) && p->N <= (1 << 30) && p->K <= (1 << 30), "gemm_w4: M, N and K must be at most 2^30");
    GP_REQUIRE(p->group == 32 || p->group == 64 || p->group == 128, "gemm_w4: group must be 32, 64 or 128");
    GP_REQUIRE(p->K % p->group == 0, "gemm_w4: K must be a multiple of the group");
    GP_REQUIRE(p->lda % 8 == 0 && p->lda >= p->K, "gemm_w4: lda must be a multiple of 8 elements that holds a row");
    GP_REQUIRE(p->ldw % 16 == 0 && p->ldw >= p->K / 2, "gemm_w4: ldw must be a multiple of 16 bytes that holds a row");
    const int groups = p->K / p->group;
    GP_REQUIRE(p->ld_scales >= groups && (!p->zeros || p->ld_zeros >= groups), "gemm_w4: row strides of scales and zeros must hold a row's groups");
    GP_REQUIRE(p->ldc >= p->N, "gemm_w4: ldc must hold a row");
    GP_REQUIRE(aligned16(p->A) && aligned16(p->W), "gemm_w4: A and W must be 16-byte aligned");
    GP_REQUIRE(((uintptr_t)p->C | (uintptr_t)p->scales | (uintptr_t)p->bias | (uintptr_t)p->residual) % 2 == 0, "gemm_w4: C, scales, bias and residual must be aligned to their elements");
    GP_REQUIRE(p->act == GP_ACT_NONE || p->act == GP_ACT_RELU || p->act == GP_ACT_GELU, "gemm_w4: act %d", p->act);
    const W4Args a{*p, groups, std::min(groups, W4_PANEL), 0, 0};
    switch (p->group * 2 + (p->dtype == GP_F16)) {
#define GP_W4(T, F16, G) case G * 2 + F16: return choose_w4<T, G>(a, ctx, s, info);
        GP_W4(_Float16, 1, 32) GP_W4(__bf16, 0, 32) GP_W4(_Float16, 1, 64) GP_W4(__bf16, 0, 64) GP_W4(_Float16, 1, 128) GP_W4(__bf16, 0, 128)
#undef GP_W4
    }
    return GP_OUTOFRANGE;
}
