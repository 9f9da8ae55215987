// sfg_chosen.hpp -- attention over chosen tokens of a paged cache: the arguments, and
// which tokens a unit of query columns walks and sees (sfg_attention_chosen.hip,
// sfg_attention_tree.hip).
#pragma once

#include "sfg_kernels.hpp"
#include "sfg_paged.hpp"

namespace sfg {

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

// A split's weight; one without a maximum enters as it is (0, or NaN where a score was NaN).
__device__ __forceinline__ float split_weight(float m, float M) { return m == -INFINITY ? 1.f : fast_exp2(m - M); }

// The tree's tile kernel (sfg_attention_tree.hip): bf16 queries, pools and output,
// head_dim 64 / 128, 16-token pages.  groups == 0: the kernels here take the call.
struct TreeTiles {
    int waves, col_waves, cols;  // waves of a workgroup, those that split its columns, and the columns
    int64_t chunks;        // column chunks of a unit
    int64_t groups;        // workgroups that the tiles are dealt to, at most
    int least;             // and the least that one takes
    size_t before_bytes, ml_bytes, acc_bytes;
    size_t bytes() const { return before_bytes + ml_bytes + acc_bytes; }
};
struct TreeRuns {
    int32_t* before;       // [batch + 1] tiles before each sequence
    int32_t* unit_flags;   // [unit][chunk] and [group][2]: non-finite values among those that
    int32_t* part_flags;   // not every column sees, left out of a whole unit or of a part
    int batch, chunks, cols, groups, least;
};
TreeTiles plan_tree_tiles(int64_t batch, int64_t kv_heads, int64_t cols, int64_t head_dim, int64_t keys, int32_t requested);
void launch_tree_tiles(ChosenArgs p, const TreeTiles& t, int64_t batch, void* workspace, hipStream_t stream);

}  // namespace sfg
