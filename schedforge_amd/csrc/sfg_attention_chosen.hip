// sfg_attention_chosen.hip -- attention over chosen tokens of a paged cache:
//
//  * a tree of drafted tokens (mask bits behind the committed tokens),
//  * decode rows that add each token's attention weight to its accumulator,
//  * decode rows over the pages a selection names.
//
// All three are softmax(c q K^T) V over a set of visible tokens, one pass over
// K and V with the running maximum and sum of the softmax:
//   m' = max(m, max_j s_j),  l' = l e^(m - m') + sum_j e^(s_j - m'),
//   acc' = acc e^(m - m') + sum_j e^(s_j - m') v_j,   out = acc / l.
// The work splits into units: the query columns that read the same tokens.  A
// unit is a (sequence, kv head) with rows x group columns, or for the selected
// pages a (sequence, row, kv head) with group columns.  Splits of a unit's tokens
// leave (m, l, acc) partials, merged in split order.
#include <algorithm>

#include "sfg_kernels.hpp"
#include "sfg_paged.hpp"

namespace sfg {

namespace {

struct ChosenArgs {
    const void* q; int q_f32;               // [B][Hq][rows][D]
    const void* k_pool; const void* v_pool;
    const int32_t* page_table; const int32_t* seq_lens; int max_len;   // lengths are clamped to max_len
    void* out; int out_f32;                 // [B][Hq][rows][D]
    float* part_ml; float* part_acc;        // [unit column][split] of (m, l) and [D]
    int q_heads, kv_heads, rows, head_dim, page_tokens, pages_per_seq, num_pages, splits;
    float scale_log2;                       // scale * log2(e): scores are exponents of 2
    const uint32_t* mask; int64_t mask_stride; int mask_words;   // tree
    float* scores; int64_t scores_ld;       // weights: scaled scores [unit column][ld]
    const int32_t* selected; int top;       // sparse: logical pages [unit][top], ascending, -1 behind
};

// A unit's columns, the tokens it walks and who sees them.
template <int MODE>
struct Unit {
    int b, kvh, row;    // row: the selected pages' query row
    int64_t id;         // (b, kvh) or (b, row, kvh) in order
    int cols;           // query columns
    int walk;           // tokens walked: logical tokens, or the selected pages' in list order
    int total;          // logical tokens that exist
    int all_see;        // tokens below this every column sees
    const int32_t* list;
};

template <int MODE>
__device__ __forceinline__ Unit<MODE> unit_of(const ChosenArgs& p, int b, int y) {
    Unit<MODE> u;
    const int G = p.q_heads / p.kv_heads;
    const int len = p.seq_lens ? min(max(p.seq_lens[b], 0), p.max_len) : p.max_len;
    u.b = b;
    u.list = nullptr;
    if constexpr (MODE == kChosenSparse) {
        u.row = y / p.kv_heads;
        u.kvh = y % p.kv_heads;
        u.id = (static_cast<int64_t>(b) * p.rows + u.row) * p.kv_heads + u.kvh;
        u.cols = G;
        u.total = max(len - p.rows + u.row + 1, 0);
        u.all_see = u.total;
        u.list = p.selected + u.id * p.top;
        // entries in use: the list is packed
        const int pages = (u.total + p.page_tokens - 1) / p.page_tokens;
        u.walk = min(p.top, pages) * p.page_tokens;
    } else {
        u.row = 0;
        u.kvh = y;
        u.id = static_cast<int64_t>(b) * p.kv_heads + y;
        u.cols = p.rows * G;
        if constexpr (MODE == kChosenTree) {
            u.total = len + p.rows;
            u.all_see = len;
        } else {
            u.total = len;
            u.all_see = len - p.rows + 1;
        }
        u.walk = u.total;
    }
    return u;
}

// Query row and head of a unit's column.
template <int MODE>
__device__ __forceinline__ void column_of(const ChosenArgs& p, const Unit<MODE>& u, int col, int& row, int& head) {
    const int G = p.q_heads / p.kv_heads;
    row = MODE == kChosenSparse ? u.row : col / G;
    head = u.kvh * G + (MODE == kChosenSparse ? col : col % G);
}

// Whether query row `row` sees logical token `tok` (< total).
template <int MODE>
__device__ __forceinline__ bool sees(const ChosenArgs& p, const Unit<MODE>& u, int row, int tok) {
    if constexpr (MODE == kChosenTree) {
        const int t = tok - u.all_see;  // all_see: the committed tokens
        if (t < 0) return true;
        return (p.mask[u.b * p.mask_stride + static_cast<int64_t>(row) * p.mask_words + (t >> 5)] >> (t & 31)) & 1u;
    } else if constexpr (MODE == kChosenWeights) {
        return tok < u.total - p.rows + row + 1;
    } else {
        return tok < u.total;
    }
}

// The unit and column of a (unit column) slot, counted through all units.
template <int MODE>
__device__ __forceinline__ Unit<MODE> unit_of_slot(const ChosenArgs& p, int64_t slot, int& col) {
    const int G = p.q_heads / p.kv_heads;
    const int per_unit = MODE == kChosenSparse ? G : p.rows * G;
    const int per_b = MODE == kChosenSparse ? p.rows * p.kv_heads : p.kv_heads;
    const int64_t uid = slot / per_unit;
    col = static_cast<int>(slot % per_unit);
    return unit_of<MODE>(p, static_cast<int>(uid / per_b), static_cast<int>(uid % per_b));
}

// Element offset of column (row, head) of q and out.
__device__ __forceinline__ int64_t column_offset(const ChosenArgs& p, int b, int row, int head) {
    return ((static_cast<int64_t>(b) * p.q_heads + head) * p.rows + row) * p.head_dim;
}

// ===========================================================================
// Any head_dim up to kRowMaxD, any page size, any alignment: one wave per
// (unit column, split).  Lane j scores token j of each 64-token chunk with one
// fp32 FMA chain over the head dimension, then the wave accumulates p V, lane d
// owning dims d, d + 64, ...
// ===========================================================================
template <typename KvT, int MODE>
__global__ __launch_bounds__(64) void chosen_any_kernel(ChosenArgs p) {
    const int lane = threadIdx.x;
    const int64_t slot = blockIdx.x;
    const int split = blockIdx.y;
    int col, row, head;
    const Unit<MODE> u = unit_of_slot<MODE>(p, slot, col);
    column_of<MODE>(p, u, col, row, head);
    const int D = p.head_dim, pt = p.page_tokens;
    const int k0 = static_cast<int>(static_cast<int64_t>(u.walk) * split / p.splits);
    const int k1 = static_cast<int>(static_cast<int64_t>(u.walk) * (split + 1) / p.splits);

    __shared__ float sq[kRowMaxD];
    const int64_t qo = column_offset(p, u.b, row, head);
    for (int d = lane; d < D; d += 64)
        sq[d] = p.q_f32 ? static_cast<const float*>(p.q)[qo + d] : bf16_to_f32(static_cast<const uint16_t*>(p.q)[qo + d]);
    __syncthreads();
    const KvT* kpool = static_cast<const KvT*>(p.k_pool);
    const KvT* vpool = static_cast<const KvT*>(p.v_pool);
    const int32_t* table = p.page_table + static_cast<int64_t>(u.b) * p.pages_per_seq;
    float m = -INFINITY, l = 0.f;
    float acc[4] = {0.f, 0.f, 0.f, 0.f};
    for (int base = k0; base < k1; base += 64) {
        const int j = base + lane;
        float s = -INFINITY;
        int page = -1, at = 0;
        if (j < k1) {
            int lp = j / pt;
            at = j % pt;
            if constexpr (MODE == kChosenSparse) lp = u.list[lp];
            const int tok = lp * pt + at;
            if (lp >= 0 && lp < p.pages_per_seq && tok < u.total) {
                const int id = table[lp];
                if (id >= 0 && id < p.num_pages && sees<MODE>(p, u, row, tok)) {
                    page = id;
                    const KvT* kr = kpool + ((static_cast<int64_t>(id) * p.kv_heads + u.kvh) * pt + at) * D;
                    float dot = 0.f;
                    for (int d = 0; d < D; ++d) dot = fmaf(sq[d], kv_f32(kr, d), dot);
                    s = dot * p.scale_log2;
                }
            }
            if constexpr (MODE == kChosenWeights) p.scores[slot * p.scores_ld + j] = s;
        }
        const float m_new = fmaxf(m, wave_max(s));
        const float pr = page < 0 ? 0.f : m_new == -INFINITY ? (s == -INFINITY ? 0.f : s) : fast_exp2(s - m_new);
        const float alpha = m == -INFINITY ? 0.f : fast_exp2(m - m_new);
        l = l * alpha + wave_sum(pr);
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[r] *= alpha;
        const int count = min(64, k1 - base);
        for (int t = 0; t < count; ++t) {
            const float pt_t = lane_bcast(pr, t);
            const int pg = lane_bcast(page, t);
            if (pg < 0) continue;  // wave-uniform
            const KvT* vb = vpool + (static_cast<int64_t>(pg) * p.kv_heads + u.kvh) * D * pt + lane_bcast(at, t);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int d = lane + 64 * r;
                if (d < D) acc[r] = fmaf(pt_t, kv_f32(vb, static_cast<int64_t>(d) * pt), acc[r]);
            }
        }
        m = m_new;
    }
    if (MODE != kChosenWeights && p.splits == 1) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int d = lane + 64 * r;
            if (d >= D) continue;
            const float o = acc[r] / l;  // nothing visible: 0 / 0
            if (p.out_f32) static_cast<float*>(p.out)[qo + d] = o;
            else static_cast<uint16_t*>(p.out)[qo + d] = f32_to_bf16(o);
        }
        return;
    }
    const int64_t part = slot * p.splits + split;
    if (lane == 0) {
        p.part_ml[2 * part] = m;
        p.part_ml[2 * part + 1] = l;
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const int d = lane + 64 * r;
        if (d < D) p.part_acc[part * D + d] = acc[r];
    }
}

// ===========================================================================
// The splits of a column merged: weights 2^(m_s - M), output sum / L.
// ===========================================================================
// A split's weight; one without a maximum enters as it is (0, or NaN where a score was NaN).
__device__ __forceinline__ float split_weight(float m, float M) { return m == -INFINITY ? 1.f : fast_exp2(m - M); }

__device__ __forceinline__ float split_max(const float* ml, int splits) {
    float M = -INFINITY;
    for (int s = 0; s < splits; ++s) M = fmaxf(M, ml[2 * s]);
    return M;
}

template <int MODE>
__device__ __forceinline__ void merge_column(const ChosenArgs& p, const Unit<MODE>& u, int col, int lane, int lanes) {
    const int64_t slot = u.id * u.cols + col;
    const float* ml = p.part_ml + 2 * slot * p.splits;
    const float* pa = p.part_acc + slot * p.splits * p.head_dim;
    const float M = split_max(ml, p.splits);
    int row, head;
    column_of<MODE>(p, u, col, row, head);
    const int64_t o0 = column_offset(p, u.b, row, head);
    for (int d = lane; d < p.head_dim; d += lanes) {
        float L = 0.f, o = 0.f;
        for (int s = 0; s < p.splits; ++s) {
            const float w = split_weight(ml[2 * s], M);
            L = fmaf(ml[2 * s + 1], w, L);
            o = fmaf(w, pa[static_cast<int64_t>(s) * p.head_dim + d], o);
        }
        const float v = o / L;  // nothing visible: 0 / 0
        if (p.out_f32) static_cast<float*>(p.out)[o0 + d] = v;
        else static_cast<uint16_t*>(p.out)[o0 + d] = f32_to_bf16(v);
    }
}

template <int MODE>
__global__ __launch_bounds__(64) void chosen_combine_kernel(ChosenArgs p) {
    int col;
    const Unit<MODE> u = unit_of_slot<MODE>(p, blockIdx.x, col);
    merge_column<MODE>(p, u, col, threadIdx.x, 64);
}

// The weights' end: every workgroup merges the columns' (m, l) of its (sequence,
// kv head), adds sum_columns 2^(s - M) / L to its 256 tokens' accumulators, and
// takes its share of the output columns.  A column that sees nothing adds nothing.
__global__ __launch_bounds__(256) void chosen_weights_kernel(ChosenArgs p, float* weights, int64_t ld) {
    constexpr int kCols = 64;
    __shared__ float sM[kCols], sR[kCols];
    const Unit<kChosenWeights> u = unit_of<kChosenWeights>(p, blockIdx.x / p.kv_heads, blockIdx.x % p.kv_heads);
    const int tok = blockIdx.y * 256 + threadIdx.x;
    float sum = 0.f;
    for (int c0 = 0; c0 < u.cols; c0 += kCols) {
        const int n = min(kCols, u.cols - c0);
        __syncthreads();
        for (int c = threadIdx.x; c < n; c += 256) {
            const float* ml = p.part_ml + 2 * (u.id * u.cols + c0 + c) * p.splits;
            const float M = split_max(ml, p.splits);
            float L = 0.f;
            for (int s = 0; s < p.splits; ++s) L = fmaf(ml[2 * s + 1], split_weight(ml[2 * s], M), L);
            sM[c] = M;
            sR[c] = L == 0.f ? 0.f : 1.f / L;
        }
        __syncthreads();
        if (tok < u.total)
            for (int c = 0; c < n; ++c) {
                const float s = p.scores[(u.id * u.cols + c0 + c) * p.scores_ld + tok];
                if (s != -INFINITY) sum = fmaf(fast_exp2(s - sM[c]), sR[c], sum);
            }
    }
    if (tok < u.total) weights[u.id * ld + tok] += sum;
    for (int c = blockIdx.y; c < u.cols; c += gridDim.y) merge_column<kChosenWeights>(p, u, c, threadIdx.x, 256);
}

size_t up256(size_t v) { return (v + 255) / 256 * 256; }

template <int MODE>
void launch_mode(const ChosenLaunch& a, const ChosenArgs& p, const ChosenPlan& plan, hipStream_t stream) {
    const unsigned columns = static_cast<unsigned>(a.batch * a.rows * a.q_heads);
    const dim3 grid(columns, static_cast<unsigned>(plan.splits));
    if (a.kv_dtype == SFG_F32) chosen_any_kernel<float, MODE><<<grid, 64, 0, stream>>>(p);
    else chosen_any_kernel<uint16_t, MODE><<<grid, 64, 0, stream>>>(p);
    if constexpr (MODE == kChosenWeights)
        chosen_weights_kernel<<<dim3(static_cast<unsigned>(a.batch * a.kv_heads), static_cast<unsigned>((a.max_context + 255) / 256)),
                                256, 0, stream>>>(p, a.weights, a.weights_ld);
    else if (plan.splits > 1) chosen_combine_kernel<MODE><<<columns, 64, 0, stream>>>(p);
}

}  // namespace

ChosenPlan plan_chosen(int mode, int64_t batch, int64_t q_heads, int64_t kv_heads, int64_t rows, int64_t head_dim,
                       int64_t page_tokens, int64_t keys, int32_t requested) {
    ChosenPlan plan{};
    const int64_t columns = batch * rows * q_heads;
    // >= 1024 waves while every split keeps >= 256 tokens
    int64_t s = 1;
    if (requested > 0) s = std::min<int64_t>(requested, std::max<int64_t>(keys, 1));
    else
        while (columns * s < 1024 && keys / (s * 2) >= 256) s *= 2;
    plan.splits = static_cast<int>(std::min<int64_t>(s, 65535));
    if (mode == kChosenWeights || plan.splits > 1) {
        const size_t parts = static_cast<size_t>(columns) * plan.splits;
        plan.ml_bytes = up256(parts * 2 * sizeof(float));
        plan.acc_bytes = up256(parts * head_dim * sizeof(float));
    }
    if (mode == kChosenWeights) {
        plan.scores_ld = (keys + 15) / 16 * 16;
        plan.scores_bytes = up256(static_cast<size_t>(columns) * plan.scores_ld * sizeof(float));
    }
    return plan;
}

void launch_chosen(const ChosenLaunch& a, const ChosenPlan& plan, void* workspace, hipStream_t stream) {
    ChosenArgs p{};
    p.q = a.q; p.q_f32 = a.q_dtype == SFG_F32;
    p.k_pool = a.k_pool; p.v_pool = a.v_pool;
    p.page_table = a.page_table; p.seq_lens = a.seq_lens; p.max_len = static_cast<int>(a.max_context);
    p.out = a.out; p.out_f32 = a.out_dtype == SFG_F32;
    char* ws = static_cast<char*>(workspace);
    p.part_ml = reinterpret_cast<float*>(ws);
    p.part_acc = reinterpret_cast<float*>(ws + plan.ml_bytes);
    p.scores = reinterpret_cast<float*>(ws + plan.ml_bytes + plan.acc_bytes);
    p.scores_ld = plan.scores_ld;
    p.q_heads = static_cast<int>(a.q_heads); p.kv_heads = static_cast<int>(a.kv_heads);
    p.rows = static_cast<int>(a.rows); p.head_dim = static_cast<int>(a.head_dim);
    p.page_tokens = static_cast<int>(a.page_tokens); p.pages_per_seq = static_cast<int>(a.pages_per_seq);
    p.num_pages = static_cast<int>(a.num_pages); p.splits = plan.splits;
    p.scale_log2 = a.scale * kLog2e;
    p.mask = a.mask; p.mask_stride = a.mask_stride; p.mask_words = static_cast<int>((a.rows + 31) / 32);
    p.selected = a.selected; p.top = static_cast<int>(a.top);
    if (a.mode == kChosenTree) launch_mode<kChosenTree>(a, p, plan, stream);
    else if (a.mode == kChosenWeights) launch_mode<kChosenWeights>(a, p, plan, stream);
    else launch_mode<kChosenSparse>(a, p, plan, stream);
}

}  // namespace sfg
