// Attention over whole prompts, of different lengths and packed one behind the other, without a cache.
//
// A tile is one head of keys and values and 128 query rows of a sequence that share it (its tokens times the query heads of the head): many_keys in paged_many.hpp,
// its keys and values from rows of the packed tensors.  Bound as that is, by matrix and vector instructions that seldom overlap.
//
// Measured: four sequences of 1024 to 8192 tokens, causal, 32 heads over 8 of 128, bf16: 1409 to 1529 us on different days, 910 to 987 TFLOP/s (a large matrix product: 1150).  37 sequences of 48 to 384, 12 heads of 64, fp16, not
// causal: 28 us for 55 MB: 1332 workgroups of six steps at most, whose beginnings count as much as their steps.  Heads of 64: three workgroups to a compute unit (32 registers less than the compiler takes by
// itself): 973 -> 920 us for four sequences up to 8192, with four 1270.
#include "paged_many.hpp"
#include "launch_tiles.hpp"

namespace gp {

struct PackedArgs {
    gp_packed_attention_params p;
    int group;       // query heads to a head of keys and values
    int row_blocks;  // of MANY_ROWS rows
};

template <typename T, int D>
__device__ __forceinline__ void attend_packed(const PackedArgs &a, TileIdx t, char *lds) {
#pragma clang fp contract(off)  // (as in attend_stretch)
    const gp_packed_attention_params &p = a.p;
    constexpr int DB = D / 32;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), l32 = lane & 31, half = lane >> 5;
    const int rb = a.row_blocks - 1 - t.x, b = t.y % p.batch, kvh = t.y / p.batch;  // (the last rows see most keys: they come first)
    const int r0 = p.start[b], r1 = p.start[b + 1];
    const SeqTokens s = seq_tokens_of(r0, r1, 0, p.tokens, p.max_len);
    const int nrows = s.rows * a.group - rb * MANY_ROWS;
    if (nrows <= 0) return;
    const int last_token = (rb * MANY_ROWS + (nrows < MANY_ROWS ? nrows : MANY_ROWS) - 1) / a.group;
    const int kend = (int)keys_seen(s.rows, last_token, p.causal);
    const int r = wave * 32 + l32, token = (rb * MANY_ROWS + r) / a.group, hg = rb * MANY_ROWS + r - token * a.group;
    const bool there = r < nrows;
    const int seen = there ? (int)keys_seen(s.rows, token, p.causal) : 0;
    const T *q = (const T *)p.q + (s.row0 + (there ? token : 0)) * p.ld_q + ((long)kvh * a.group + (there ? hg : 0)) * D;
    const long first = (s.row0 * p.ld_kv + (long)kvh * D) * sizeof(T);
    f32x16 o[DB];
    float m, l;
    many_keys<T, D, false>(PackedKeys{(const char *)p.k + first, (const char *)p.v + first, p.ld_kv * (long)sizeof(T), s.rows - 1}, ManyRow{there, seen, q}, p.scale, kend, s.rows, 0,
                           (kend + MANY_KEYS - 1) / MANY_KEYS, lds, o, m, l);
    l += __shfl_xor(l, 32, 64);
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

template <typename T, int D, int LOOP = LOOP_ANY>
__global__ __launch_bounds__(MANY_NT, D == 64 ? 3 : 2) void packed_attention_kernel(PackedArgs a, BlpArgs blp) {
    extern __shared__ __attribute__((aligned(16))) unsigned char packed_lds[];
    // (claims through counters are dealt out, or one of an XCD's would have the longest prompt: four prompts up to 8192, preemptible, 2099 -> 1584 us)
    tiles<LOOP>(blp, [&](TileIdx t) { attend_packed<T, D>(a, dealt_tile<LOOP>(blp, t), (char *)packed_lds); });
}

}  // namespace gp

using namespace gp;

extern "C" int gp_launch_packed_attention(const gp_packed_attention_params *p, const gp_preempt_ctx *ctx, gp_stream s, gp_launch_info *info) {
    GP_REQUIRE(p && p->start && p->q && p->k && p->v && p->out, "null packed_attention params");
    GP_REQUIRE(p->dtype == GP_F16 || p->dtype == GP_BF16, "packed_attention: fp16 or bf16 only (dtype %d)", p->dtype);
    GP_REQUIRE(p->head_dim == 64 || p->head_dim == 128, "packed_attention: head_dim must be 64 or 128");
    GP_REQUIRE(p->batch > 0 && p->tokens > 0 && p->max_len > 0, "packed_attention: batch, tokens and max_len must be positive");
    GP_REQUIRE(p->kv_heads > 0 && p->heads > 0 && p->heads % p->kv_heads == 0, "packed_attention: heads must be a multiple of those of the keys and values");
    const long q_cols = (long)p->heads * p->head_dim, kv_cols = (long)p->kv_heads * p->head_dim;
    GP_REQUIRE(p->ld_q % 8 == 0 && p->ld_kv % 8 == 0 && p->ld_out % 8 == 0 && p->ld_q >= q_cols && p->ld_kv >= kv_cols && p->ld_out >= q_cols,
               "packed_attention: row strides must be multiples of 8 elements that hold the heads");
    GP_REQUIRE(p->ld_kv <= (1L << 25), "packed_attention: ld_kv must be at most 2^25");  // (64 rows within 32 bits of bytes: many_keys)
    GP_REQUIRE(aligned16(p->q) && aligned16(p->k) && aligned16(p->v) && aligned16(p->out), "packed_attention: 16-byte alignment");
    GP_REQUIRE(usable_scale(p->scale), "packed_attention: the scale must be 0 (for 1) or of a magnitude from 2^-100 to 2^100");
    PackedArgs a{*p, p->heads / p->kv_heads, 0};
    if (a.p.scale == 0.f) a.p.scale = 1.f;
    if (a.p.max_len > p->tokens) a.p.max_len = (int)p->tokens;  // (no sequence has more rows than there are)
    const long rows = (long)a.p.max_len * a.group, heads = (long)p->batch * p->kv_heads;
    GP_REQUIRE(rows < (1L << 30) && heads < (1L << 30), "packed_attention: too large");
    a.row_blocks = (int)((rows + MANY_ROWS - 1) / MANY_ROWS);
    GP_REQUIRE(heads * a.row_blocks < (1L << 31), "packed_attention: too large");
    switch (p->head_dim * 2 + (p->dtype == GP_F16)) {
#define GP_PACKED(T, F16, D) case D * 2 + F16: return launch_tiles(GP_KSET(packed_attention_kernel<T, D), a.row_blocks, (int)heads, ctx, s, info, a, many_lds_bytes<D>(), 1, MANY_NT);
        GP_PACKED(_Float16, 1, 64) GP_PACKED(__bf16, 0, 64) GP_PACKED(_Float16, 1, 128) GP_PACKED(__bf16, 0, 128)
#undef GP_PACKED
    }
    return GP_OUTOFRANGE;
}
