// Log probabilities of given tokens, entropy and largest alternatives of rows of logits.
#include <algorithm>
#include <cmath>
#include "mma.hpp"
#include "launch_tiles.hpp"

namespace gp {

constexpr int LP_NT = 256, LP_TOP = 32;

// Order of the alternatives in one number: the larger logit first, then the lower token.  0: no alternative (NaN, -infinity).
__device__ __forceinline__ unsigned long long rank_key(float x, int id) {
    if (!(x > -INFINITY)) return 0;
    const unsigned bits = __builtin_bit_cast(unsigned, x == 0.f ? 0.f : x);  // (one zero)
    return (unsigned long long)(bits & 0x80000000u ? ~bits : bits | 0x80000000u) << 32 | (0xFFFFFFFFu - (unsigned)id);
}
__device__ __forceinline__ float key_value(unsigned long long key) {
    const unsigned u = (unsigned)(key >> 32);
    return __builtin_bit_cast(float, u & 0x80000000u ? u & 0x7FFFFFFFu : ~u);
}
__device__ __forceinline__ int key_id(unsigned long long key) { return (int)(0xFFFFFFFFu - (unsigned)key); }

__device__ __forceinline__ float block_sum(float x, float *lds) {
    __syncthreads();
    lds[threadIdx.x] = x;
    __syncthreads();
    float s = 0.f;
    for (int i = 0; i < LP_NT; ++i) s += lds[i];
    return s;
}

// One row per tile, read once for the largest value, once for the sums, once more for every alternative.
template <typename T>
__device__ __forceinline__ void logprobs_tile(const gp_token_logprobs_params &p, TileIdx t, float *lds, unsigned long long *keys) {
    const int tid = threadIdx.x;
    const T *x = (const T *)p.logits + (long)t.x * p.ld;
    float m = -INFINITY;
    for (int i = tid; i < p.vocab; i += LP_NT) m = fmaxf(m, Elem<T>::to_f(x[i]));
    __syncthreads();
    lds[tid] = m;
    __syncthreads();
    for (int i = 0; i < LP_NT; ++i) m = fmaxf(m, lds[i]);
    float sum = 0.f, weighted = 0.f;
    for (int i = tid; i < p.vocab; i += LP_NT) {
        const float v = Elem<T>::to_f(x[i]);
        const float y = v == -INFINITY ? -INFINITY : (v - m) * p.scale, e = expf(y);
        sum += e;
        if (e > 0.f) weighted = fmaf(e, y, weighted);
    }
    sum = block_sum(sum, lds);
    weighted = block_sum(weighted, lds);
    const float log_sum = logf(sum);
    const bool empty = sum == 0.f;
    if (tid == 0) {
        if (p.logprob) {
            const long id = p.tokens[t.x];
            float r = 0.f;
            if (id >= 0 && id < p.vocab) {
                const float v = Elem<T>::to_f(x[id]);
                r = empty ? -INFINITY : (v == -INFINITY && sum == sum ? -INFINITY : (v - m) * p.scale - log_sum);
            }
            p.logprob[t.x] = r;
        }
        if (p.entropy) p.entropy[t.x] = empty ? 0.f : log_sum - weighted / sum;
    }
    unsigned long long last = ~0ull;
    for (int k = 0; k < p.top; ++k) {
        unsigned long long best = 0;
        for (int i = tid; i < p.vocab; i += LP_NT) {
            const unsigned long long key = rank_key(Elem<T>::to_f(x[i]), i);
            if (key < last && key > best) best = key;
        }
        __syncthreads();
        keys[tid] = best;
        __syncthreads();
        for (int i = 0; i < LP_NT; ++i) best = best < keys[i] ? keys[i] : best;
        if (tid == 0) {
            p.top_ids[(long)t.x * p.top + k] = best ? key_id(best) : -1;
            p.top_logprobs[(long)t.x * p.top + k] = best ? (key_value(best) - m) * p.scale - log_sum : -INFINITY;
        }
        last = best;
    }
}

template <typename T, int LOOP = LOOP_ANY>
__global__ __launch_bounds__(LP_NT) void token_logprobs_kernel(gp_token_logprobs_params p, BlpArgs blp) {
    __shared__ float lds[LP_NT];
    __shared__ unsigned long long keys[LP_NT];
    tiles<LOOP>(blp, [&](TileIdx t) { logprobs_tile<T>(p, t, lds, keys); });
}

static int check_token_logprobs(const gp_token_logprobs_params *p) {
    GP_REQUIRE(p && p->logits, "null token_logprobs params");
    GP_REQUIRE(p->dtype == GP_F32 || p->dtype == GP_F16 || p->dtype == GP_BF16, "token_logprobs dtype %d", p->dtype);
    GP_REQUIRE(p->rows > 0 && p->rows < (1L << 31) && p->vocab > 0 && p->vocab < (1 << 30) && p->ld >= p->vocab, "token_logprobs: rows, vocab (below 2^30) and a row stride that holds it");
    GP_REQUIRE(((uintptr_t)p->logits & (p->dtype == GP_F32 ? 3 : 1)) == 0, "token_logprobs: logits are not aligned to their type");
    GP_REQUIRE(p->top >= 0 && p->top <= LP_TOP, "token_logprobs: 0 to %d alternatives", LP_TOP);
    GP_REQUIRE(!p->top || (p->top_ids && p->top_logprobs), "token_logprobs: alternatives need a place to go to");
    GP_REQUIRE(p->logprob || p->entropy || p->top, "token_logprobs: nothing is asked for");
    GP_REQUIRE(!p->logprob || p->tokens, "token_logprobs: log probabilities of which tokens?");
    GP_REQUIRE(p->scale >= 0.f && std::isfinite(p->scale), "token_logprobs: the scale must be finite and not negative");
    return GP_SUCC;
}

}  // namespace gp

using namespace gp;

extern "C" int gp_token_logprobs_work_bytes(const gp_token_logprobs_params *p, size_t *bytes) {
    if (int rc = check_token_logprobs(p)) return rc;
    GP_REQUIRE(bytes, "token_logprobs: no place for the size");
    *bytes = 0;
    return GP_SUCC;
}

extern "C" int gp_launch_token_logprobs(const gp_token_logprobs_params *p, const gp_preempt_ctx *ctx, gp_stream s, gp_launch_info *info) {
    if (int rc = check_token_logprobs(p)) return rc;
    gp_token_logprobs_params a = *p;
    if (a.scale == 0.f) a.scale = 1.f;
    switch (p->dtype) {
        case GP_F32: return launch_tiles(GP_KSET(token_logprobs_kernel<float), (int)p->rows, 1, ctx, s, info, a, 0, 1, LP_NT);
        case GP_F16: return launch_tiles(GP_KSET(token_logprobs_kernel<_Float16), (int)p->rows, 1, ctx, s, info, a, 0, 1, LP_NT);
        default: return launch_tiles(GP_KSET(token_logprobs_kernel<__bf16), (int)p->rows, 1, ctx, s, info, a, 0, 1, LP_NT);
    }
}
