// Attention of a batch of sequences that begin with the same tokens, in the same pages of the cache.
#include "kv_cache.hpp"

using namespace gp;

static int check_prefix(const gp_prefix_attention_params *p, size_t *bytes) {
    GP_REQUIRE(p, "null prefix_attention params");
    if (int rc = gp_paged_attention_work_bytes(&p->attention, bytes)) return rc;
    GP_REQUIRE(p->shared_len >= 0 && p->shared_len % p->attention.cache.page_size == 0, "prefix_attention: shared_len must be whole pages");
    GP_REQUIRE(p->shared_len == 0 || p->shared_table, "prefix_attention: where are the shared pages?");
    return GP_SUCC;
}

extern "C" int gp_prefix_attention_work_bytes(const gp_prefix_attention_params *p, size_t *bytes) { return check_prefix(p, bytes); }

extern "C" int gp_launch_prefix_attention(const gp_prefix_attention_params *p, const gp_preempt_ctx *ctx, gp_stream s, gp_launch_info *info) {
    size_t bytes;
    if (int rc = check_prefix(p, &bytes)) return rc;
    return gp_launch_paged_attention(&p->attention, ctx, s, info);
}
