// sfg_api_kv8.hip -- the C ABI of a step over a paged cache held in 8 bits: pages and
// slots, rotary positions, appends, attention.  Arguments are checked on the host, as in
// sfg_api.hip.
#include <math.h>

#include "sfg_api_util.hpp"
#include "sfg_kernels.hpp"
#include "sfg_kv8.hpp"

namespace {

using sfg::check_launch;
using sfg::fail;

constexpr int64_t kMaxInt = 0x7FFFFFFF;
constexpr int64_t kMostRows = (1 << 22) - 1;  // rows of a step, and query columns: 1024 threads each
constexpr int64_t kMostHeads = 65535;         // a launch's second dimension

hipStream_t as_stream(void* s) { return static_cast<hipStream_t>(s); }

bool float_dtype(int dt) { return dt == SFG_F32 || dt == SFG_BF16; }
bool code_dtype(int dt) { return dt == SFG_I8 || dt == SFG_FP8; }

struct Span {
    const void* p;
    int64_t bytes;
    bool meets(const Span& o) const {
        const uintptr_t a = reinterpret_cast<uintptr_t>(p), b = reinterpret_cast<uintptr_t>(o.p);
        return p && o.p && a < b + static_cast<uint64_t>(o.bytes) && b < a + static_cast<uint64_t>(bytes);
    }
};

// `count` rows of `bytes`, `stride` bytes from one to the next (at least `bytes`).
struct Rows {
    const void* p;
    int64_t stride, bytes, count;
    int64_t at() const { return static_cast<int64_t>(reinterpret_cast<uintptr_t>(p)); }
    int64_t end() const { return at() + (count - 1) * stride + bytes; }
    static Rows all(const void* p, int64_t bytes) { return {p, bytes, bytes, 1}; }
    // n rows from `from` on: does one of them meet [b, b + size)?  The first that ends behind b does, or none.
    static bool one(int64_t from, int64_t stride, int64_t bytes, int64_t n, int64_t b, int64_t size) {
        const int64_t ahead = b - bytes - from, i = ahead < 0 ? 0 : ahead / stride + 1;
        return i < n && from + i * stride < b + size;
    }
    bool meets(const Rows& o) const {
        if (!p || !o.p || at() >= o.end() || o.at() >= end()) return false;
        if (o.count == 1) return one(at(), stride, bytes, count, o.at(), o.bytes);
        if (count == 1) return o.meets(*this);
        // of one stride: row i and row j lie as row i - j and row 0 do
        if (stride == o.stride) return one(at() - (o.count - 1) * stride, stride, bytes, count + o.count - 1, o.at(), o.bytes);
        for (int64_t i = 0; i < count; ++i)
            if (one(o.at(), o.stride, o.bytes, o.count, at() + i * stride, bytes)) return true;
        return false;
    }
};
// (sizes that no memory has are cut)
int64_t times(int64_t a, int64_t b) { return a > (int64_t{1} << 56) / b ? int64_t{1} << 56 : a * b; }

// What the attention's checks and its workspace query share; pointers apart.
bool sized(const sfg_kv8_attn_args& a) {
    return a.batch > 0 && a.q_heads > 0 && a.kv_heads > 0 && a.q_heads % a.kv_heads == 0 && a.head_dim > 0 &&
           a.head_dim <= 256 && a.page_tokens > 0 && a.page_tokens <= kMaxInt / 2 && a.max_context >= 0 &&
           a.max_context <= kMaxInt / 2 && a.tokens > 0 && a.tokens <= kMostRows && a.q_heads <= kMostHeads &&
           a.tokens * a.q_heads <= kMostRows && a.batch <= kMostRows && a.max_rows > 0 && a.max_rows <= a.tokens;
}

}  // namespace

extern "C" {

int sfg_hip_kv_plan_v1(const sfg_kv_plan_args* a, void* stream) {
    if (!a) return fail(SFG_ERR_SHAPE, "kv_plan: null arguments");
    if (!a->counts || !a->seq_lens || !a->page_table || !a->free_pages || !a->free_count || !a->starts || !a->positions ||
        !a->slots || a->batch <= 0 || a->pages_per_seq <= 0 || a->num_pages <= 0 || a->page_tokens <= 0 || a->max_tokens <= 0)
        return fail(SFG_ERR_INVALID_CONFIG, "kv_plan: invalid configuration");
    if (a->page_tokens > kMaxInt / 2 || a->pages_per_seq > kMaxInt / 2 / a->page_tokens || a->num_pages > kMaxInt / 2 ||
        a->batch > (1 << 20) || a->batch * a->pages_per_seq > kMaxInt)
        return fail(SFG_ERR_UNSUPPORTED, "kv_plan: sizes beyond 32-bit positions");
    if (a->max_tokens > kMostRows) return fail(SFG_ERR_UNSUPPORTED, "kv_plan: 2^22 rows or more");
    const int64_t lens = 4 * a->batch;
    const Span written[] = {{a->seq_lens, lens}, {a->page_table, 4 * a->batch * a->pages_per_seq}, {a->free_pages, 4 * a->num_pages},
                            {a->free_count, 4}, {a->starts, lens + 4}, {a->positions, 4 * a->max_tokens}, {a->slots, 8 * a->max_tokens}};
    constexpr int kWritten = sizeof written / sizeof *written;
    for (int i = 0; i < kWritten; ++i) {
        for (int j = i + 1; j < kWritten; ++j)
            if (written[i].meets(written[j])) return fail(SFG_ERR_SHAPE, "kv_plan: lists or tables overlap");
        // (keep and counts are read before the lengths of the same sequence are written)
        for (const int32_t* in : {a->keep, a->counts})
            if (written[i].meets({in, lens}) && in != a->seq_lens) return fail(SFG_ERR_SHAPE, "kv_plan: lists or tables overlap");
    }
    sfg::launch_kv_plan(*a, as_stream(stream));
    return check_launch("kv_plan");
}

int sfg_hip_rope_inv_freq_host_v1(double* inv_freq, float* magnitude, int64_t rotary_dim, const sfg_rope_scaling* s) {
    if (!inv_freq || !magnitude || !s || rotary_dim <= 0 || rotary_dim % 2)
        return fail(SFG_ERR_SHAPE, "rope_inv_freq: invalid arguments");
    const int kind = s->kind;
    if (kind < SFG_ROPE_PLAIN || kind > SFG_ROPE_RAMP) return fail(SFG_ERR_UNSUPPORTED, "rope_inv_freq: scaling %d", kind);
    if (!(s->theta > 1.0) || !isfinite(s->theta)) return fail(SFG_ERR_INVALID_CONFIG, "rope_inv_freq: theta %g", s->theta);
    if (kind != SFG_ROPE_PLAIN && (!(s->factor >= 1.0) || !isfinite(s->factor)))
        return fail(SFG_ERR_INVALID_CONFIG, "rope_inv_freq: factor %g", s->factor);
    if ((kind == SFG_ROPE_BANDS || kind == SFG_ROPE_RAMP) &&
        (!(s->context > 0.0) || !isfinite(s->context) || !(s->low > 0.0) || !(s->high > s->low) || !isfinite(s->high)))
        return fail(SFG_ERR_INVALID_CONFIG, "rope_inv_freq: context %g, turns %g .. %g", s->context, s->low, s->high);
    const double r = static_cast<double>(rotary_dim), f = s->factor;
    const double theta = kind == SFG_ROPE_BASE && rotary_dim > 2 ? s->theta * pow(f, r / (r - 2.0)) : s->theta;
    auto pair_of = [&](double turns) { return r * log(s->context / (2.0 * M_PI * turns)) / (2.0 * log(theta)); };
    const double from = kind == SFG_ROPE_RAMP ? fmax(floor(pair_of(s->high)), 0.0) : 0.0;
    const double to = kind == SFG_ROPE_RAMP ? fmin(ceil(pair_of(s->low)), r - 1.0) : 0.0;
    for (int64_t i = 0; i < rotary_dim / 2; ++i) {
        double w = pow(theta, -2.0 * static_cast<double>(i) / r);
        if (kind == SFG_ROPE_LINEAR) w /= f;
        if (kind == SFG_ROPE_BANDS) {
            const double t = fmin(fmax((s->context * w / (2.0 * M_PI) - s->low) / (s->high - s->low), 0.0), 1.0);
            w *= t + (1.0 - t) / f;
        }
        if (kind == SFG_ROPE_RAMP) {
            const double t = fmin(fmax((static_cast<double>(i) - from) / fmax(to - from, 0.001), 0.0), 1.0);
            w *= 1.0 - t + t / f;
        }
        inv_freq[i] = w;
    }
    *magnitude = kind == SFG_ROPE_RAMP ? static_cast<float>(0.1 * log(f) + 1.0) : 1.0f;
    return SFG_OK;
}

int sfg_hip_rope_turns_host_v1(uint64_t* turns, const double* inv_freq, int64_t pairs) {
    if (!turns || !inv_freq || pairs <= 0) return fail(SFG_ERR_SHAPE, "rope_turns: invalid arguments");
    for (int64_t i = 0; i < pairs; ++i)
        if (!isfinite(inv_freq[i])) return fail(SFG_ERR_INVALID_CONFIG, "rope_turns: angle %g", inv_freq[i]);
    for (int64_t i = 0; i < pairs; ++i) {
        // (long double holds 64 bits of the fraction)
        const long double t = static_cast<long double>(inv_freq[i]) / 6.283185307179586476925286766559L;
        const long double x = floorl((t - floorl(t)) * 18446744073709551616.0L + 0.5L);
        turns[i] = x >= 18446744073709551616.0L ? 0 : static_cast<uint64_t>(x);
    }
    return SFG_OK;
}

int sfg_hip_rope_v1(const sfg_rope_args* a, void* stream) {
    if (!a) return fail(SFG_ERR_SHAPE, "rope: null arguments");
    if (!a->positions || !a->turns || a->tokens <= 0 || a->q_heads < 0 || a->kv_heads < 0 || a->q_heads + a->kv_heads <= 0 ||
        a->head_dim <= 0 || a->rotary_dim <= 0 || a->rotary_dim % 2 || a->rotary_dim > a->head_dim || !isfinite(a->magnitude))
        return fail(SFG_ERR_INVALID_CONFIG, "rope: invalid configuration");
    if (!float_dtype(a->dtype)) return fail(SFG_ERR_UNSUPPORTED, "rope: dtype %d", a->dtype);
    if (a->layout != SFG_ROPE_HALF && a->layout != SFG_ROPE_INTERLEAVED) return fail(SFG_ERR_UNSUPPORTED, "rope: layout %d", a->layout);
    if (a->tokens > kMostRows || a->q_heads > kMostHeads || a->kv_heads > kMostHeads || a->head_dim > 1024)
        return fail(SFG_ERR_UNSUPPORTED, "rope: 2^22 rows, 2^16 heads or more, or head_dim over 1024");
    const struct { const void* in; const void* out; int64_t heads, in_stride, out_stride; } part[] = {
        {a->q, a->q_out, a->q_heads, a->q_stride, a->q_out_stride}, {a->k, a->k_out, a->kv_heads, a->k_stride, a->k_out_stride}};
    for (const auto& p : part) {
        if (p.heads == 0 && !p.in && !p.out) continue;
        if (p.heads == 0 || !p.in || !p.out || p.in_stride < p.heads * a->head_dim || p.out_stride < p.heads * a->head_dim ||
            p.in_stride > kMaxInt || p.out_stride > kMaxInt)
            return fail(SFG_ERR_SHAPE, "rope: heads without rows, or rows closer than their heads");
        if (p.in == p.out && p.in_stride != p.out_stride) return fail(SFG_ERR_SHAPE, "rope: in place with two strides");
    }
    const int64_t size = a->dtype == SFG_F32 ? 4 : 2;
    auto rows = [&](const void* p, int64_t stride, int64_t heads) { return Rows{p, stride * size, heads * a->head_dim * size, a->tokens}; };
    for (const auto& w : part) {
        const Rows out = rows(w.out, w.out_stride, w.heads);
        for (const auto& r : part)
            if ((!(&r == &w && r.in == w.out) && out.meets(rows(r.in, r.in_stride, r.heads))) ||
                (&r > &w && out.meets(rows(r.out, r.out_stride, r.heads))))
                return fail(SFG_ERR_SHAPE, "rope: an output overlaps other rows");
        if (out.meets(Rows::all(a->positions, 4 * a->tokens)) || out.meets(Rows::all(a->turns, 8 * (a->rotary_dim / 2))))
            return fail(SFG_ERR_SHAPE, "rope: an output overlaps positions or turns");
    }
    sfg::launch_rope(*a, as_stream(stream));
    return check_launch("rope");
}

int sfg_hip_kv8_append_v1(const sfg_kv8_append_args* a, void* stream) {
    if (!a) return fail(SFG_ERR_SHAPE, "kv8_append: null arguments");
    if (!a->keys || !a->values || !a->k_pool || !a->v_pool || !a->scales || !a->slots || a->tokens <= 0 || a->kv_heads <= 0 ||
        a->head_dim <= 0 || a->page_tokens <= 0 || a->num_pages <= 0)
        return fail(SFG_ERR_INVALID_CONFIG, "kv8_append: invalid configuration");
    if (!float_dtype(a->dtype)) return fail(SFG_ERR_UNSUPPORTED, "kv8_append: dtype %d", a->dtype);
    if (!code_dtype(a->pool_dtype)) return fail(SFG_ERR_UNSUPPORTED, "kv8_append: pool dtype %d", a->pool_dtype);
    if (a->head_dim > 256) return fail(SFG_ERR_UNSUPPORTED, "kv8_append: head_dim %lld > 256", (long long)a->head_dim);
    if (a->tokens > kMostRows || a->kv_heads > kMostHeads || a->page_tokens > kMaxInt / 512 || a->num_pages > kMaxInt)
        return fail(SFG_ERR_UNSUPPORTED, "kv8_append: sizes beyond 32-bit positions");
    if (a->key_stride < a->kv_heads * a->head_dim || a->value_stride < a->kv_heads * a->head_dim || a->key_stride > kMaxInt ||
        a->value_stride > kMaxInt)
        return fail(SFG_ERR_SHAPE, "kv8_append: rows closer than their heads");
    sfg::launch_kv8_append(*a, as_stream(stream));
    return check_launch("kv8_append");
}

size_t sfg_hip_attn_kv8_workspace_v1(const sfg_kv8_attn_args* a) { return a && sized(*a) ? sfg::workspace_attn_kv8(*a) : 0; }

int sfg_hip_attn_kv8_v1(const sfg_kv8_attn_args* a, void* workspace, size_t workspace_bytes, void* stream) {
    if (!a) return fail(SFG_ERR_SHAPE, "attn_kv8: null arguments");
    if (!a->q || !a->out || !a->k_pool || !a->v_pool || !a->scales || !a->page_table || a->batch <= 0 || a->tokens <= 0 ||
        a->max_rows <= 0 || a->q_heads <= 0 || a->kv_heads <= 0 || a->q_heads % a->kv_heads || a->head_dim <= 0 ||
        a->page_tokens <= 0 || a->pages_per_seq <= 0 || a->num_pages <= 0 || a->max_context < 0)
        return fail(SFG_ERR_INVALID_CONFIG, "attn_kv8: invalid configuration");
    if (!float_dtype(a->q_dtype)) return fail(SFG_ERR_UNSUPPORTED, "attn_kv8: query dtype %d", a->q_dtype);
    if (!float_dtype(a->out_dtype)) return fail(SFG_ERR_UNSUPPORTED, "attn_kv8: output dtype %d", a->out_dtype);
    if (!code_dtype(a->pool_dtype)) return fail(SFG_ERR_UNSUPPORTED, "attn_kv8: pool dtype %d", a->pool_dtype);
    if (a->head_dim > 256) return fail(SFG_ERR_UNSUPPORTED, "attn_kv8: head_dim %lld > 256", (long long)a->head_dim);
    if (a->page_tokens > kMaxInt / 512 || a->pages_per_seq > kMaxInt / 2 / a->page_tokens || a->num_pages > kMaxInt || a->batch > (1 << 20))
        return fail(SFG_ERR_UNSUPPORTED, "attn_kv8: sizes beyond 32-bit positions");
    if (a->tokens > kMostRows || a->q_heads > kMostHeads || a->tokens * a->q_heads > kMostRows)
        return fail(SFG_ERR_UNSUPPORTED, "attn_kv8: 2^22 query columns or more");
    if (a->starts ? a->max_rows > a->tokens : a->max_rows > a->tokens || a->tokens != a->batch * a->max_rows)
        return fail(SFG_ERR_SHAPE, "attn_kv8: %lld rows of %lld sequences of up to %lld", (long long)a->tokens, (long long)a->batch,
                    (long long)a->max_rows);
    const int64_t row = a->q_heads * a->head_dim;
    if (a->q_stride < row || a->out_stride < row || a->q_stride > kMaxInt || a->out_stride > kMaxInt)
        return fail(SFG_ERR_SHAPE, "attn_kv8: rows closer than their heads");
    if (a->out == a->q) return fail(SFG_ERR_SHAPE, "attn_kv8: the output is the query");
    if (a->max_context > a->pages_per_seq * a->page_tokens)
        return fail(SFG_ERR_GUARD, "attn_kv8: paged KV length violates compiled guard (%lld > %lld)", (long long)a->max_context,
                    (long long)(a->pages_per_seq * a->page_tokens));
    const sfg::Kv8Plan plan = sfg::plan_attn_kv8(*a);
    if (plan.bytes > 0 && (reinterpret_cast<uintptr_t>(workspace) & 15))
        return fail(SFG_ERR_WORKSPACE, "attn_kv8: workspace off a 16-byte boundary");
    if (plan.bytes > 0 && (!workspace || workspace_bytes < plan.bytes))
        return fail(SFG_ERR_WORKSPACE, "attn_kv8: workspace %zu < %zu", workspace ? workspace_bytes : 0, plan.bytes);
    const int64_t units = times(a->num_pages, a->kv_heads), pool = times(units, a->page_tokens * a->head_dim);
    const int64_t q_size = a->q_dtype == SFG_F32 ? 4 : 2, out_size = a->out_dtype == SFG_F32 ? 4 : 2;
    const Rows q{a->q, a->q_stride * q_size, row * q_size, a->tokens}, out{a->out, a->out_stride * out_size, row * out_size, a->tokens};
    const Rows scratch = Rows::all(plan.bytes > 0 ? workspace : nullptr, static_cast<int64_t>(plan.bytes));
    const Rows read[] = {q, Rows::all(a->k_pool, pool), Rows::all(a->v_pool, pool), Rows::all(a->scales, times(units, 8)),
                         Rows::all(a->page_table, 4 * a->batch * a->pages_per_seq), Rows::all(a->seq_lens, 4 * a->batch),
                         Rows::all(a->starts, 4 * a->batch + 4)};
    if (out.meets(scratch)) return fail(SFG_ERR_SHAPE, "attn_kv8: the output and the workspace overlap");
    for (const Rows& r : read)
        if (out.meets(r) || scratch.meets(r)) return fail(SFG_ERR_SHAPE, "attn_kv8: the output or the workspace overlaps what is read");
    sfg::launch_attn_kv8(*a, plan, workspace, as_stream(stream));
    return check_launch("attn_kv8");
}

}  // extern "C"
