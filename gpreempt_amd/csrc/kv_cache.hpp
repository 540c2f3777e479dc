// What the operators on a paged cache share: the check of the cache's description, and conversions of 8-bit values.
#pragma once
#include "mma.hpp"
#include "../../include/util/page_map.h"

namespace gp {

inline bool aligned16(const void *p) { return ((uintptr_t)p & 15) == 0; }

inline int check_kv_cache(const gp_kv_cache &c, int dtype, const char *who) {
    GP_REQUIRE(dtype == GP_F16 || dtype == GP_BF16, "%s: fp16 or bf16 only (dtype %d)", who, dtype);
    GP_REQUIRE(c.dtype == dtype || c.dtype == GP_E4M3, "%s: a cache of dtype %d for activations of dtype %d", who, c.dtype, dtype);
    GP_REQUIRE(c.head_dim == 64 || c.head_dim == 128, "%s: head_dim must be 64 or 128", who);
    GP_REQUIRE(c.page_size == 16 || c.page_size == 32 || c.page_size == 64 || c.page_size == 128, "%s: page_size must be 16, 32, 64 or 128", who);
    GP_REQUIRE(c.kv_heads > 0 && c.pages > 0, "%s: cache shape", who);
    GP_REQUIRE(c.k && c.v && aligned16(c.k) && aligned16(c.v), "%s: keys and values of the cache must be there, 16-byte aligned", who);
    GP_REQUIRE(c.dtype != GP_E4M3 || (c.k_scale && c.v_scale), "%s: an 8-bit cache needs its scales", who);
    return GP_SUCC;
}

// keeps the compiler from making one operation, with a single rounding, of the arithmetic in front and a conversion behind
__device__ __forceinline__ float rounded(float x) {
    asm("" : "+v"(x));
    return x;
}

// A page's scale as everybody takes it, between the borders that the header names: their ratio, and its inverse, are in fp32's normal range, so no
// probability times a scale is lost next to another's.  (NaN becomes the lower one)
constexpr float LEAST_SCALE = 0x1p-60f, MOST_SCALE = 0x1p60f;
__device__ __forceinline__ float within_scales(float s) { return fminf(fmaxf(s, LEAST_SCALE), MOST_SCALE); }

typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));

// eight e4m3 values of 8 bytes
__device__ __forceinline__ void unpack_e4m3(u32x2 raw, float (&x)[8]) {
#pragma unroll
    for (int w = 0; w < 2; ++w) {
        const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)raw[w], false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)raw[w], true);
        x[4 * w] = lo[0]; x[4 * w + 1] = lo[1]; x[4 * w + 2] = hi[0]; x[4 * w + 3] = hi[1];
    }
}

// to the nearest e4m3 value, ties to even; beyond the largest (448) the largest, NaN stays NaN
__device__ __forceinline__ u32x2 pack_e4m3(const float (&x)[8]) {
    float y[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = x[i] > 448.f ? 448.f : x[i] < -448.f ? -448.f : x[i];
    u32x2 raw;
#pragma unroll
    for (int w = 0; w < 2; ++w) {
        int v = __builtin_amdgcn_cvt_pk_fp8_f32(y[4 * w], y[4 * w + 1], 0, false);
        raw[w] = (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(y[4 * w + 2], y[4 * w + 3], v, true);
    }
    return raw;
}

}  // namespace gp
