// sfg_api_paged.hip -- the C ABI of the operators that choose what a paged cache
// keeps and reads: tree attention, attention with accumulated weights, sparse
// attention over selected pages, page bounds, token selection and compaction.
// Arguments are checked on the host, as in sfg_api.hip.
#include <math.h>

#include <algorithm>

#include "sfg_api_util.hpp"
#include "sfg_kernels.hpp"

namespace {

using sfg::check_launch;
using sfg::fail;

constexpr int64_t kMaxInt = 0x7FFFFFFF;
constexpr int64_t kMostUnits = (1 << 21) - 1;    // (sequence, kv head)s: up to 2048 threads each
constexpr int64_t kMostColumns = (1 << 22) - 1;  // 1024 threads each

hipStream_t as_stream(void* s) { return static_cast<hipStream_t>(s); }

bool float_dtype(int dt) { return dt == SFG_F32 || dt == SFG_BF16; }

// Sizes of the pools and tables.  Positions, page ids and query columns are 32-bit
// on the device; a launch holds fewer than 2^32 threads.
int check_pool(const char* what, const void* table, int pool_dtype, int64_t batch, int64_t kv_heads, int64_t head_dim,
               int64_t page_tokens, int64_t pages_per_seq, int64_t num_pages) {
    if (!table || batch <= 0 || kv_heads <= 0 || head_dim <= 0 || page_tokens <= 0 || pages_per_seq <= 0 || num_pages <= 0)
        return fail(SFG_ERR_INVALID_CONFIG, "%s: invalid configuration", what);
    if (!float_dtype(pool_dtype)) return fail(SFG_ERR_UNSUPPORTED, "%s: pool dtype %d", what, pool_dtype);
    if (head_dim > 256) return fail(SFG_ERR_UNSUPPORTED, "%s: head_dim %lld > 256", what, (long long)head_dim);
    if (page_tokens > kMaxInt / 2 || pages_per_seq > kMaxInt / 2 / page_tokens || num_pages > kMaxInt || batch > (1 << 20) ||
        kv_heads > (1 << 20) || batch * kv_heads > kMostUnits)
        return fail(SFG_ERR_UNSUPPORTED, "%s: sizes beyond 32-bit positions", what);
    return SFG_OK;
}

// Whether the query columns can be counted (batch and kv_heads are positive).
bool countable(const sfg_paged_attn_args& a) {
    return a.batch <= kMostColumns && a.q_heads <= kMostColumns && a.rows <= kMostColumns &&
           a.batch * a.q_heads <= kMostColumns && a.batch * a.q_heads * a.rows <= kMostColumns;
}

int check_args(const char* what, const sfg_paged_attn_args* a) {
    if (!a) return fail(SFG_ERR_SHAPE, "%s: null arguments", what);
    const int rc = check_pool(what, a->page_table, a->kv_dtype, a->batch, a->kv_heads, a->head_dim, a->page_tokens,
                              a->pages_per_seq, a->num_pages);
    if (rc != SFG_OK) return rc;
    if (!a->q || !a->k_pool || !a->v_pool || !a->out || a->q_heads <= 0 || a->q_heads % a->kv_heads || a->rows <= 0 ||
        a->max_context < 0)
        return fail(SFG_ERR_INVALID_CONFIG, "%s: invalid configuration", what);
    if (!float_dtype(a->q_dtype)) return fail(SFG_ERR_UNSUPPORTED, "%s: query dtype %d", what, a->q_dtype);
    if (!float_dtype(a->out_dtype)) return fail(SFG_ERR_UNSUPPORTED, "%s: output dtype %d", what, a->out_dtype);
    if (!countable(*a))
        return fail(SFG_ERR_UNSUPPORTED, "%s: 2^22 query columns or more", what);
    return SFG_OK;
}

int check_context(const char* what, int64_t keys, int64_t capacity) {
    if (keys <= capacity) return SFG_OK;
    return fail(SFG_ERR_GUARD, "%s: paged KV length violates compiled guard (%lld > %lld)", what, (long long)keys,
                (long long)capacity);
}

int check_workspace(const char* what, size_t need, const void* ws, size_t bytes) {
    if (need > 0 && (reinterpret_cast<uintptr_t>(ws) & 15))
        return fail(SFG_ERR_WORKSPACE, "%s: workspace off a 16-byte boundary", what);
    if (need == 0 || (ws && bytes >= need)) return SFG_OK;
    return fail(SFG_ERR_WORKSPACE, "%s: workspace %zu < %zu", what, ws ? bytes : 0, need);
}

sfg::ChosenLaunch launch_of(int mode, const sfg_paged_attn_args& a) {
    sfg::ChosenLaunch c{};
    c.mode = mode;
    c.q = a.q; c.q_dtype = a.q_dtype;
    c.k_pool = a.k_pool; c.v_pool = a.v_pool; c.kv_dtype = a.kv_dtype;
    c.page_table = a.page_table; c.seq_lens = a.seq_lens;
    c.out = a.out; c.out_dtype = a.out_dtype;
    c.batch = a.batch; c.q_heads = a.q_heads; c.kv_heads = a.kv_heads; c.rows = a.rows; c.head_dim = a.head_dim;
    c.page_tokens = a.page_tokens; c.pages_per_seq = a.pages_per_seq; c.num_pages = a.num_pages;
    c.max_context = a.max_context;
    c.kv_splits = a.kv_splits;
    c.scale = a.scale > 0.0f ? a.scale : 1.0f / sqrtf(static_cast<float>(a.head_dim));
    return c;
}

// The tokens a unit of query columns walks at most.
int64_t walked(int mode, const sfg_paged_attn_args& a, int64_t top) {
    if (mode == sfg::kChosenTree) return a.max_context + a.rows;
    if (mode == sfg::kChosenWeights) return a.max_context;
    return std::min((a.max_context + a.page_tokens - 1) / a.page_tokens, top) * a.page_tokens;
}

sfg::ChosenPlan plan_of(int mode, const sfg_paged_attn_args& a, int64_t top, bool ragged) {
    const bool bf16 = a.q_dtype == SFG_BF16 && a.kv_dtype == SFG_BF16 && a.out_dtype == SFG_BF16;
    return sfg::plan_chosen(mode, bf16, ragged, a.batch, a.q_heads, a.kv_heads, a.rows, a.head_dim, a.page_tokens,
                            walked(mode, a, top), a.kv_splits);
}

size_t page_keys_bytes(const sfg_paged_attn_args& a) {
    return sfg::page_select_workspace_bytes(a.batch, a.kv_heads, a.rows, (a.max_context + a.page_tokens - 1) / a.page_tokens);
}

// What a workspace query goes by (its pointers may be null: it covers a call with lengths
// and one without).
bool sized(const sfg_paged_attn_args* a) {
    return a && a->batch > 0 && a->q_heads > 0 && a->kv_heads > 0 && a->q_heads % a->kv_heads == 0 && a->rows > 0 &&
           a->head_dim > 0 && a->head_dim <= 256 && a->page_tokens > 0 && a->page_tokens <= kMaxInt / 2 &&
           a->max_context >= 0 && a->max_context <= kMaxInt / 2 && countable(*a);
}

}  // namespace

extern "C" {

size_t sfg_hip_attn_tree_workspace_v1(const sfg_paged_attn_args* a) {
    return sized(a) ? plan_of(sfg::kChosenTree, *a, 0, true).bytes() : 0;
}

int sfg_hip_attn_tree_v1(const sfg_paged_attn_args* a, const uint32_t* tree_mask, int64_t mask_stride, void* workspace,
                         size_t workspace_bytes, void* stream) {
    int rc = check_args("attn_tree", a);
    if (rc != SFG_OK) return rc;
    if (!tree_mask || (mask_stride != 0 && mask_stride < a->rows * ((a->rows + 31) / 32)))
        return fail(SFG_ERR_SHAPE, "attn_tree: no mask, or sequences' masks overlap");
    const int64_t capacity = a->pages_per_seq * a->page_tokens;  // (the sum below is taken only of lengths within it)
    if ((rc = check_context("attn_tree", a->max_context, capacity)) != SFG_OK) return rc;
    if ((rc = check_context("attn_tree", a->max_context + a->rows, capacity)) != SFG_OK) return rc;
    const sfg::ChosenPlan plan = plan_of(sfg::kChosenTree, *a, 0, a->seq_lens != nullptr);
    if ((rc = check_workspace("attn_tree", plan.bytes(), workspace, workspace_bytes)) != SFG_OK) return rc;
    sfg::ChosenLaunch c = launch_of(sfg::kChosenTree, *a);
    c.mask = tree_mask;
    c.mask_stride = mask_stride;
    sfg::launch_chosen(c, plan, workspace, as_stream(stream));
    return check_launch("attn_tree");
}

size_t sfg_hip_attn_weights_workspace_v1(const sfg_paged_attn_args* a) {
    return sized(a) ? plan_of(sfg::kChosenWeights, *a, 0, true).bytes() : 0;
}

int sfg_hip_attn_weights_v1(const sfg_paged_attn_args* a, float* weights, int64_t weights_ld, void* workspace,
                            size_t workspace_bytes, void* stream) {
    int rc = check_args("attn_weights", a);
    if (rc != SFG_OK) return rc;
    if (a->max_context <= 0 || a->rows > a->max_context)
        return fail(SFG_ERR_INVALID_CONFIG, "attn_weights: %lld rows over %lld tokens", (long long)a->rows,
                    (long long)a->max_context);
    if ((rc = check_context("attn_weights", a->max_context, a->pages_per_seq * a->page_tokens)) != SFG_OK) return rc;
    if (a->max_context > (1 << 23))
        return fail(SFG_ERR_UNSUPPORTED, "attn_weights: more than 2^23 tokens");
    if (!weights || weights_ld < a->max_context)
        return fail(SFG_ERR_SHAPE, "attn_weights: weights of %lld tokens for sequences up to %lld", (long long)weights_ld,
                    (long long)a->max_context);
    const sfg::ChosenPlan plan = plan_of(sfg::kChosenWeights, *a, 0, a->seq_lens != nullptr);
    if ((rc = check_workspace("attn_weights", plan.bytes(), workspace, workspace_bytes)) != SFG_OK) return rc;
    sfg::ChosenLaunch c = launch_of(sfg::kChosenWeights, *a);
    c.weights = weights;
    c.weights_ld = weights_ld;
    sfg::launch_chosen(c, plan, workspace, as_stream(stream));
    return check_launch("attn_weights");
}

size_t sfg_hip_attn_sparse_workspace_v1(const sfg_paged_attn_args* a, int64_t top_pages) {
    return sized(a) && top_pages > 0 ? page_keys_bytes(*a) + plan_of(sfg::kChosenSparse, *a, top_pages, true).bytes() : 0;
}

int sfg_hip_attn_sparse_v1(const sfg_paged_attn_args* a, const void* bounds, int64_t top_pages, int64_t sink_pages,
                           int64_t recent_pages, int32_t* selected, void* workspace, size_t workspace_bytes, void* stream) {
    int rc = check_args("attn_sparse", a);
    if (rc != SFG_OK) return rc;
    if (a->max_context <= 0 || a->rows > a->max_context)
        return fail(SFG_ERR_INVALID_CONFIG, "attn_sparse: %lld rows over %lld tokens", (long long)a->rows,
                    (long long)a->max_context);
    if (!bounds || !selected || top_pages <= 0 || sink_pages < 0 || recent_pages < 0 || top_pages > kMaxInt ||
        sink_pages > top_pages || recent_pages > top_pages - sink_pages)
        return fail(SFG_ERR_SHAPE, "attn_sparse: %lld pages with %lld first and %lld newest ones", (long long)top_pages,
                    (long long)sink_pages, (long long)recent_pages);
    if ((rc = check_context("attn_sparse", a->max_context, a->pages_per_seq * a->page_tokens)) != SFG_OK) return rc;
    const sfg::ChosenPlan plan = plan_of(sfg::kChosenSparse, *a, top_pages, a->seq_lens != nullptr);
    const size_t keys = page_keys_bytes(*a);
    if ((rc = check_workspace("attn_sparse", keys + plan.bytes(), workspace, workspace_bytes)) != SFG_OK) return rc;
    sfg::ChosenLaunch c = launch_of(sfg::kChosenSparse, *a);
    c.selected = selected;
    c.top = top_pages;
    sfg::launch_page_select(c, bounds, sink_pages, recent_pages, selected, workspace, as_stream(stream));
    sfg::launch_chosen(c, plan, static_cast<char*>(workspace) + keys, as_stream(stream));
    return check_launch("attn_sparse");
}

int sfg_hip_kv_page_bounds_v1(const void* k_pool, int pool_dtype, const int32_t* page_table, const int32_t* seq_lens,
                              int64_t max_context, int64_t fresh, void* bounds, int64_t batch, int64_t kv_heads,
                              int64_t head_dim, int64_t page_tokens, int64_t pages_per_seq, int64_t num_pages,
                              void* stream) {
    int rc = check_pool("kv_page_bounds", page_table, pool_dtype, batch, kv_heads, head_dim, page_tokens, pages_per_seq,
                        num_pages);
    if (rc != SFG_OK) return rc;
    if (!k_pool || !bounds || max_context <= 0 || fresh <= 0)
        return fail(SFG_ERR_SHAPE, "kv_page_bounds: invalid arguments");
    if ((rc = check_context("kv_page_bounds", max_context, pages_per_seq * page_tokens)) != SFG_OK) return rc;
    sfg::launch_page_bounds(k_pool, pool_dtype, page_table, seq_lens, max_context, fresh, bounds, batch, kv_heads, head_dim,
                            page_tokens, pages_per_seq, num_pages, as_stream(stream));
    return check_launch("kv_page_bounds");
}

int sfg_hip_kv_select_v1(const float* weights, int64_t weights_ld, const int32_t* seq_lens, int64_t max_context,
                         int64_t budget, int64_t recent, int32_t* keep, int32_t* kept_lens, float* kept_weights,
                         int64_t batch, int64_t kv_heads, void* stream) {
    if (!weights || !keep || !kept_lens || batch <= 0 || kv_heads <= 0 || max_context <= 0 || weights_ld < max_context)
        return fail(SFG_ERR_SHAPE, "kv_select: invalid arguments");
    if (kept_lens == seq_lens) return fail(SFG_ERR_SHAPE, "kv_select: kept_lens is seq_lens");
    if (budget <= 0 || recent < 0 || recent > budget)
        return fail(SFG_ERR_INVALID_CONFIG, "kv_select: a budget of %lld tokens with the newest %lld", (long long)budget,
                    (long long)recent);
    if (max_context > kMaxInt / 2 || budget > kMaxInt / 2 || batch > (1 << 20) || kv_heads > (1 << 20) ||
        batch * kv_heads > kMostUnits)
        return fail(SFG_ERR_UNSUPPORTED, "kv_select: sizes beyond 32-bit positions");
    sfg::launch_kv_select(weights, weights_ld, seq_lens, max_context, budget, recent, keep, kept_lens, kept_weights, batch,
                          kv_heads, as_stream(stream));
    return check_launch("kv_select");
}

int sfg_hip_kv_compact_v1(void* k_pool, void* v_pool, int pool_dtype, const int32_t* page_table, const int32_t* base,
                          const int32_t* keep, int64_t keep_heads, int64_t keep_ld, const int32_t* counts,
                          int32_t* new_lens, int64_t max_keep, int64_t batch, int64_t kv_heads, int64_t head_dim,
                          int64_t page_tokens, int64_t pages_per_seq, int64_t num_pages, void* stream) {
    int rc = check_pool("kv_compact", page_table, pool_dtype, batch, kv_heads, head_dim, page_tokens, pages_per_seq,
                        num_pages);
    if (rc != SFG_OK) return rc;
    if (!k_pool || !v_pool || !keep || !counts || !new_lens || max_keep <= 0 || keep_ld < max_keep ||
        (keep_heads != 1 && keep_heads != kv_heads))
        return fail(SFG_ERR_SHAPE, "kv_compact: invalid arguments");
    if ((rc = check_context("kv_compact", max_keep, pages_per_seq * page_tokens)) != SFG_OK) return rc;
    sfg::launch_kv_compact(k_pool, v_pool, pool_dtype, page_table, base, keep, keep_heads, keep_ld, counts, new_lens,
                           max_keep, batch, kv_heads, head_dim, page_tokens, pages_per_seq, num_pages, as_stream(stream));
    return check_launch("kv_compact");
}

}  // extern "C"
