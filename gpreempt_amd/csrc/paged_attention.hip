// Attention of a batch of sequences' new tokens over the pages of a cache.
#include <algorithm>
#include "kv_cache.hpp"
#include "launch_tiles.hpp"

namespace gp {

constexpr int PA_NT = 256;

struct PagedArgs {
    gp_paged_attention_params p;
    int group;  // query heads to a head of the cache
};

// the scale of a page's head, within the bounds that the header names
__device__ __forceinline__ float page_scale(const float *scales, long at) { return fminf(fmaxf(scales[at], 0x1p-60f), 0x1p60f); }

// One query of one head per tile: 256 keys at a time, one to a thread; then a thread to every value of the head.
template <typename T, int D, bool E8>
__device__ __forceinline__ void attend_tile(const PagedArgs &a, TileIdx t, float *lds) {
    const gp_paged_attention_params &p = a.p;
    float *q = lds, *w = q + D, *red = w + PA_NT;
    const int head = t.x, i = t.y % p.max_new, b = t.y / p.max_new, tid = threadIdx.x, P = p.cache.page_size, kvh = head / a.group;
    const SeqTokens s = seq_tokens(p.start, p.kv_len, b, p.tokens, p.max_new);
    if (i >= s.rows) return;
    const long bound = seq_bound(s, p.max_len, p.table_width, P), seen = keys_seen(bound, s.first + i, p.causal);
    const T *qrow = (const T *)p.q + (s.row0 + i) * p.ld_q + (long)head * D;
    __syncthreads();
    if (tid < D) q[tid] = Elem<T>::to_f(qrow[tid]);
    __syncthreads();
    float m = -INFINITY, l = 0.f, o = 0.f;
    for (long k0 = 0; k0 < seen; k0 += PA_NT) {
        const long key = k0 + tid;
        const int page = key < seen ? page_of(p.page_table, p.table_width, b, key / P, p.cache.pages) : -1;
        float x = -INFINITY;
        if (page >= 0) {
            const long at = (((long)page * p.cache.kv_heads + kvh) * P + key % P) * D;
            float dot = 0.f;
            for (int d = 0; d < D; d += 8) {
                float y[8];
                if constexpr (E8) unpack_e4m3(*(const u32x2 *)((const unsigned char *)p.cache.k + at + d), y);
                else for (int e = 0; e < 8; ++e) y[e] = Elem<T>::to_f(((const T *)p.cache.k)[at + d + e]);
                for (int e = 0; e < 8; ++e) dot = fmaf(q[d + e], y[e], dot);
            }
            if constexpr (E8) dot *= page_scale(p.cache.k_scale, (long)page * p.cache.kv_heads + kvh);
            x = dot * p.scale;
        }
        red[tid] = x;
        __syncthreads();
        float mm = m;
        for (int e = 0; e < PA_NT; ++e) mm = fmaxf(mm, red[e]);
        const float base = mm == -INFINITY ? 0.f : mm, f = expf(m - base);
        w[tid] = page < 0 ? 0.f : expf(x - base);
        __syncthreads();
        float sum = 0.f;
        for (int e = 0; e < PA_NT; ++e) sum += w[e];
        l = l * f + sum;
        if (tid < D) {
            o *= f;
            for (int e = 0; e < PA_NT && k0 + e < seen; ++e) {
                const int pg = page_of(p.page_table, p.table_width, b, (k0 + e) / P, p.cache.pages);
                if (pg < 0) continue;
                const long hd = (long)pg * p.cache.kv_heads + kvh, at = (hd * P + (k0 + e) % P) * D + tid;
                float v;
                if constexpr (E8) v = __builtin_amdgcn_cvt_pk_f32_fp8(((const unsigned char *)p.cache.v)[at], false)[0] * page_scale(p.cache.v_scale, hd);
                else v = Elem<T>::to_f(((const T *)p.cache.v)[at]);
                o = fmaf(w[e], v, o);
            }
        }
        m = mm;
        __syncthreads();
    }
    if (tid < D) ((T *)p.out)[(s.row0 + i) * p.ld_out + (long)head * D + tid] = Elem<T>::from_f(l == 0.f ? 0.f : o / l);
}

template <typename T, int D, bool E8, int LOOP = LOOP_ANY>
__global__ __launch_bounds__(PA_NT) void paged_attention_kernel(PagedArgs a, BlpArgs blp) {
    __shared__ float lds[D + 2 * PA_NT];
    tiles<LOOP>(blp, [&](TileIdx t) { attend_tile<T, D, E8>(a, t, lds); });
}

static int check_paged_attention(const gp_paged_attention_params *p, PagedArgs *a) {
    GP_REQUIRE(p && p->kv_len && p->page_table && p->q && p->out, "null paged_attention params");
    if (int rc = check_kv_cache(p->cache, p->dtype, "paged_attention")) return rc;
    GP_REQUIRE(p->batch > 0 && p->tokens > 0 && p->max_new > 0 && p->max_len > 0 && p->table_width > 0, "paged_attention: batch, tokens, max_new, max_len and table_width must be positive");
    GP_REQUIRE(p->start || p->tokens >= p->batch, "paged_attention: one new token per sequence needs a row for each");
    GP_REQUIRE(p->heads > 0 && p->heads % p->cache.kv_heads == 0, "paged_attention: heads must be a multiple of the cache's");
    const long cols = (long)p->heads * p->cache.head_dim;
    GP_REQUIRE(p->ld_q % 8 == 0 && p->ld_out % 8 == 0 && p->ld_q >= cols && p->ld_out >= cols, "paged_attention: row strides must be multiples of 8 elements that hold the heads");
    GP_REQUIRE(aligned16(p->q) && aligned16(p->out), "paged_attention: 16-byte alignment");
    *a = PagedArgs{*p, p->heads / p->cache.kv_heads};
    if (!p->start) a->p.max_new = 1;
    if (a->p.scale == 0.f) a->p.scale = 1.f;
    GP_REQUIRE((long)p->batch * a->p.max_new < (1L << 31) && (long)p->batch * a->p.max_new * p->heads < (1L << 31), "paged_attention: too large");
    return GP_SUCC;
}

}  // namespace gp

using namespace gp;

extern "C" int gp_paged_attention_work_bytes(const gp_paged_attention_params *p, size_t *bytes) {
    PagedArgs a;
    if (int rc = check_paged_attention(p, &a)) return rc;
    GP_REQUIRE(bytes, "paged_attention: no place for the size");
    *bytes = 0;
    return GP_SUCC;
}

extern "C" int gp_launch_paged_attention(const gp_paged_attention_params *p, const gp_preempt_ctx *ctx, gp_stream s, gp_launch_info *info) {
    PagedArgs a;
    if (int rc = check_paged_attention(p, &a)) return rc;
    const bool e8 = p->cache.dtype == GP_E4M3, f16 = p->dtype == GP_F16;
#define GP_PAGED(T, D, E8) return launch_tiles(GP_KSET(paged_attention_kernel<T, D, E8), p->heads, p->batch * a.p.max_new, ctx, s, info, a, 0, 1, PA_NT)
    if (p->cache.head_dim == 128) {
        if (f16) { if (e8) GP_PAGED(_Float16, 128, true); GP_PAGED(_Float16, 128, false); }
        if (e8) GP_PAGED(__bf16, 128, true);
        GP_PAGED(__bf16, 128, false);
    }
    if (f16) { if (e8) GP_PAGED(_Float16, 64, true); GP_PAGED(_Float16, 64, false); }
    if (e8) GP_PAGED(__bf16, 64, true);
    GP_PAGED(__bf16, 64, false);
#undef GP_PAGED
}
