// Attention of a batch of sequences' new tokens over the pages of a cache.
#include <algorithm>
#include "paged_few.hpp"
#include "paged_many.hpp"
#include "launch_tiles.hpp"

namespace gp {

struct PagedPlan {
    FewArgs few;
    ManyArgs many;
    int nt;             // query rows of a tile, in sixteens; 0: many
    int tiles_x; long tiles_y;
    size_t work_bytes;
};

// in_front: bytes in front of the parts of results in the workspace, the counters among them
static int plan_paged_attention(const gp_paged_attention_params *p, size_t in_front, PagedPlan *pl) {
    GP_REQUIRE(p && p->kv_len && p->page_table && p->q && p->out, "null paged_attention params");
    if (int rc = check_kv_cache(p->cache, p->dtype, "paged_attention")) return rc;
    GP_REQUIRE(p->batch > 0 && p->tokens > 0 && p->max_new > 0 && p->max_len > 0 && p->table_width > 0, "paged_attention: batch, tokens, max_new, max_len and table_width must be positive");
    GP_REQUIRE(p->max_len <= (1 << 30), "paged_attention: max_len must be at most 2^30");
    GP_REQUIRE(p->start || p->tokens >= p->batch, "paged_attention: one new token per sequence needs a row for each");
    GP_REQUIRE(p->heads > 0 && p->heads % p->cache.kv_heads == 0, "paged_attention: heads must be a multiple of the cache's");
    const long cols = (long)p->heads * p->cache.head_dim;
    GP_REQUIRE(p->ld_q % 8 == 0 && p->ld_out % 8 == 0 && p->ld_q >= cols && p->ld_out >= cols, "paged_attention: row strides must be multiples of 8 elements that hold the heads");
    GP_REQUIRE(aligned16(p->q) && aligned16(p->out), "paged_attention: 16-byte alignment");
    GP_REQUIRE(usable_scale(p->scale), "paged_attention: the scale must be 0 (for 1) or of a magnitude from 2^-100 to 2^100");
    *pl = PagedPlan{};
    FewArgs &a = pl->few;
    a.p = *p;
    a.group = p->heads / p->cache.kv_heads;
    if (!p->start) a.p.max_new = 1;
    if (a.p.scale == 0.f) a.p.scale = 1.f;
    const long rows = (long)a.p.max_new * a.group;
    GP_REQUIRE(rows < (1L << 30) && (long)p->batch * a.p.max_new < (1L << 31), "paged_attention: too large");
    // Many rows: blocks of 128 of them over keys that come through LDS, if there are such blocks for a quarter of the compute units.  Us in such blocks / in blocks of 32 rows with
    // the keys in parts, for rows of each of 8 cached heads of 128 over 4000 keys, e4m3: 128 rows of 1, 2, 4, 8 sequences 35 / 26, 36 / 27, 37 / 34, 38 / 43; 256 rows of 1, 2, 4, 8
    // 36 / 27, 36 / 34, 38 / 43, 54 / 79; 96 rows of 4 (chosen: the second) 36 / 39, of 32 over 2000 keys 51 / 91.  Up to 64 rows are two blocks of 32 at most: 64 rows of 1, 8, and of 32
    // sequences over 2000 keys 35 / 25, 37 / 38, 50 / 58.
    const long many_blocks = (rows + MANY_ROWS - 1) / MANY_ROWS, many_units = many_blocks * p->cache.kv_heads * p->batch;
    if (rows > 64 && 4 * many_units >= device_cus()) {
        const long blocks = many_blocks, tiles_y = (long)p->cache.kv_heads * p->batch, units = many_units;
        const long want = many_shares((p->max_len + MANY_KEYS - 1) / MANY_KEYS, std::min(64l, 2l * device_cus() / units));
        GP_REQUIRE(units * want < (1L << 31), "paged_attention: too large");
        pl->many = ManyArgs{a.p, a.group, (int)blocks, (int)want, nullptr, nullptr};
        if (want > 1) {
            const size_t counters = in_front;  // (units: at most as many as compute units)
            pl->work_bytes = counters + (size_t)(units * want) * (p->cache.head_dim == 64 ? many_partial_floats<64>() : many_partial_floats<128>()) * sizeof(float);
            pl->many.arrived = (int *)p->work;
            pl->many.partial = (float *)((char *)p->work + counters);
        }
        pl->tiles_x = (int)(blocks * want);
        pl->tiles_y = tiles_y;
        return GP_SUCC;
    }
    pl->nt = rows <= 16 ? 1 : 2;
    const long blocks = (rows + 16 * pl->nt - 1) / (16 * pl->nt), heads = blocks * p->cache.kv_heads, units = heads * p->batch;
    GP_REQUIRE(units < (1L << 30), "paged_attention: too large");
    a.row_blocks = (int)blocks;
    // Short sequences get a tile each.  The keys of longer ones are dealt out in equal parts, one per compute unit: 64 sequences of 2048 to 8192 keys (8 heads
    // of 128, e4m3) 108 us, with tiles of 2816 keys of one sequence 119; one sequence of 131072 keys 50 us, with two or four parts per compute unit 56 and
    // 68 (whoever comes last has more to join).
    const int unit = p->cache.dtype == GP_E4M3 ? few_unit<true>() : few_unit<false>();
    const long most = (p->max_len + unit - 1l) / unit;
    GP_REQUIRE(most * p->batch < (1L << 31), "paged_attention: too large");
    pl->tiles_x = p->batch;
    pl->tiles_y = heads;
    if (most > 4) pl->tiles_x = a.shares = (int)std::min(std::max(1l, device_cus() / heads), most * p->batch);
    if (a.shares > 1) {
        const size_t counters = in_front;  // (heads * shares: at most as many as compute units)
        pl->work_bytes = counters + (size_t)heads * a.shares * 2 * 16 * pl->nt * (p->cache.head_dim + 2) * sizeof(float);
        a.arrived = (int *)p->work;
        a.partial = (float *)((char *)p->work + counters);
    }
    GP_REQUIRE(heads * pl->tiles_x < (1L << 31), "paged_attention: too large");
    return GP_SUCC;
}

int paged_work_bytes(const gp_paged_attention_params *p, size_t in_front, size_t *bytes) {
    PagedPlan pl;
    if (int rc = plan_paged_attention(p, in_front, &pl)) return rc;
    *bytes = pl.work_bytes;
    return GP_SUCC;
}

int launch_paged(const gp_paged_attention_params *p, size_t in_front, const gp_preempt_ctx *ctx, gp_stream s, gp_launch_info *info) {
    PagedPlan pl;
    if (int rc = plan_paged_attention(p, in_front, &pl)) return rc;
    GP_REQUIRE(pl.work_bytes == 0 || (p->work && aligned16(p->work) && p->work_bytes >= pl.work_bytes), "paged_attention: needs a workspace of %zu bytes, 16-byte aligned", pl.work_bytes);
    const bool e8 = p->cache.dtype == GP_E4M3, f16 = p->dtype == GP_F16;
    if (pl.nt == 0) {
        switch (p->cache.head_dim * 4 + e8 * 2 + f16) {
#define GP_MANY(T, F16, D, E8) case D * 4 + E8 * 2 + F16: return launch_tiles(GP_KSET(paged_many_kernel<T, D, E8), pl.tiles_x, (int)pl.tiles_y, ctx, s, info, pl.many, many_lds_bytes<D>(), 1, MANY_NT);
            GP_MANY(_Float16, 1, 64, 0) GP_MANY(__bf16, 0, 64, 0) GP_MANY(_Float16, 1, 64, 1) GP_MANY(__bf16, 0, 64, 1)
            GP_MANY(_Float16, 1, 128, 0) GP_MANY(__bf16, 0, 128, 0) GP_MANY(_Float16, 1, 128, 1) GP_MANY(__bf16, 0, 128, 1)
#undef GP_MANY
        }
        return GP_OUTOFRANGE;
    }
    const int key = p->cache.head_dim * 8 + e8 * 4 + f16 * 2 + (pl.nt == 2);
    switch (key) {
#define GP_FEW(T, F16, D, E8, NT) case D * 8 + E8 * 4 + F16 * 2 + (NT == 2): return launch_tiles(GP_KSET(paged_few_kernel<T, D, E8, NT), pl.tiles_x, (int)pl.tiles_y, ctx, s, info, pl.few, few_lds_floats<NT, D>() * sizeof(float), 1, FEW_NT);
#define GP_FEW_BOTH(D, E8, NT) GP_FEW(_Float16, 1, D, E8, NT) GP_FEW(__bf16, 0, D, E8, NT)
        GP_FEW_BOTH(64, 0, 1) GP_FEW_BOTH(64, 0, 2) GP_FEW_BOTH(64, 1, 1) GP_FEW_BOTH(64, 1, 2)
        GP_FEW_BOTH(128, 0, 1) GP_FEW_BOTH(128, 0, 2) GP_FEW_BOTH(128, 1, 1) GP_FEW_BOTH(128, 1, 2)
#undef GP_FEW_BOTH
#undef GP_FEW
    }
    return GP_OUTOFRANGE;
}

}  // namespace gp

using namespace gp;

extern "C" int gp_paged_attention_work_bytes(const gp_paged_attention_params *p, size_t *bytes) {
    size_t n;
    if (int rc = paged_work_bytes(p, join_counter_bytes(), &n)) return rc;
    GP_REQUIRE(bytes, "paged_attention: no place for the size");
    *bytes = n;
    return GP_SUCC;
}

extern "C" int gp_launch_paged_attention(const gp_paged_attention_params *p, const gp_preempt_ctx *ctx, gp_stream s, gp_launch_info *info) { return launch_paged(p, join_counter_bytes(), ctx, s, info); }
