// sfg_kv_keep.hip -- which tokens and pages of a paged cache are kept and read:
//
//  * page bounds: the smallest and largest key value of each page, head and dim;
//  * page selection: the pages of the largest score per (sequence, row, kv head),
//    score = sum over the group's heads and dims of max(q lo, q hi), an upper bound
//    of the group's summed scores on the page;
//  * token selection: the newest tokens and those of the largest accumulated weight;
//  * compaction: the kept tokens moved to the front, in place.
//
// Selections are exact: ties go to the lower index, and the page scores are summed
// in 64 bits, so that which page is taken does not hang on an order of summation.
#include <algorithm>

#include "sfg_kernels.hpp"
#include "sfg_paged.hpp"

namespace sfg {

namespace {

// Order-preserving integers: a larger key is a larger value; NaN is the smallest,
// both zeros are one value.
__device__ __forceinline__ uint32_t order_key(float v) {
    if (v != v) return 0;
    const uint32_t u = __float_as_uint(v == 0.f ? 0.f : v);
    return (u >> 31) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ uint64_t order_key(double v) {
    if (v != v) return 0;
    const uint64_t u = static_cast<uint64_t>(__double_as_longlong(v == 0.0 ? 0.0 : v));
    return (u >> 63) ? ~u : (u | 0x8000000000000000ull);
}

// ---------------------------------------------------------------- page bounds
struct BoundsArgs {
    const void* k_pool; const int32_t* page_table; const int32_t* seq_lens; int max_len;
    int64_t fresh; void* bounds;
    int kv_heads, head_dim, page_tokens, pages_per_seq, num_pages;
};

// One wave per (sequence, kv head) and page, from the newest page back, lane d owning
// dims d, d + 64, ...; a page is read whole, up to the sequence's end.
template <typename KvT>
__global__ __launch_bounds__(64) void page_bounds_kernel(BoundsArgs a) {
    const int b = blockIdx.x / a.kv_heads, h = blockIdx.x % a.kv_heads;
    const int pt = a.page_tokens, D = a.head_dim;
    const int len = a.seq_lens ? min(max(a.seq_lens[b], 0), a.max_len) : a.max_len;
    for (int page = (len + pt - 1) / pt - 1 - static_cast<int>(blockIdx.y);
         page >= 0 && static_cast<int64_t>(page + 1) * pt > len - a.fresh; page -= static_cast<int>(gridDim.y)) {
        const int id = a.page_table[static_cast<int64_t>(b) * a.pages_per_seq + page];
        if (id < 0 || id >= a.num_pages) continue;
        const int count = min(pt, len - page * pt);
        const int64_t blk = static_cast<int64_t>(id) * a.kv_heads + h;
        const KvT* k = static_cast<const KvT*>(a.k_pool) + blk * pt * D;
        KvT* out = static_cast<KvT*>(a.bounds) + blk * 2 * D;
        for (int d = threadIdx.x; d < D; d += 64) {
            float lo = INFINITY, hi = -INFINITY;
            for (int t = 0; t < count; ++t) {
                const float v = kv_f32(k, static_cast<int64_t>(t) * D + d);
                lo = fminf(lo, v);
                hi = fmaxf(hi, v);
            }
            if constexpr (sizeof(KvT) == 4) {
                out[d] = lo;
                out[D + d] = hi;
            } else {  // values of the pool: exact
                out[d] = f32_to_bf16(lo);
                out[D + d] = f32_to_bf16(hi);
            }
        }
    }
}

// ---------------------------------------------------------------- selection
constexpr int kSelThreads = 1024;
constexpr int kSelBins = 2048;

struct SelShared {
    int hist[kSelBins];
    int wave[kSelThreads / 64];
    int bin, above;
};

// Exclusive sum over the workgroup's threads; total in `all`.
__device__ __forceinline__ int block_exclusive(int v, SelShared& sh, int& all) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int x = v;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int y = __shfl_up(x, o, 64);
        if (lane >= o) x += y;
    }
    __syncthreads();
    if (lane == 63) sh.wave[wave] = x;
    __syncthreads();
    int before = 0;
    all = 0;
    for (int w = 0; w < kSelThreads / 64; ++w) {
        if (w < wave) before += sh.wave[w];
        all += sh.wave[w];
    }
    return before + x - v;
}

// The need-th largest of n keys (1 <= need <= n): every key above `key` is taken, and
// `ties` of those equal to it.  Radix selection from the top, 11 bits a pass: the
// workgroup counts a digit of the keys that match the digits found so far, and the
// bin in which the count from above passes `need` is the next digit.
template <typename Key, typename Load>
__device__ void select_threshold(Load load, int n, int need, SelShared& sh, Key& key, int& ties) {
    constexpr int kBits = sizeof(Key) * 8;
    Key prefix = 0;
    int done = 0;
    while (done < kBits) {
        const int width = min(11, kBits - done);
        const int shift = kBits - done - width;
        __syncthreads();
        for (int i = threadIdx.x; i < kSelBins; i += kSelThreads) sh.hist[i] = 0;
        __syncthreads();
        for (int i = threadIdx.x; i < n; i += kSelThreads) {
            const Key k = load(i);
            if (done == 0 || (k >> (shift + width)) == prefix)
                atomicAdd(&sh.hist[static_cast<int>(k >> shift) & ((1 << width) - 1)], 1);
        }
        __syncthreads();
        // two bins a thread, counted from the top one
        const int top = kSelBins - 1 - 2 * static_cast<int>(threadIdx.x);
        const int c1 = sh.hist[top], c0 = sh.hist[top - 1];
        int all;
        const int above = block_exclusive(c1 + c0, sh, all);
        if (above < need && need <= above + c1) {
            sh.bin = top;
            sh.above = above;
        } else if (above + c1 < need && need <= above + c1 + c0) {
            sh.bin = top - 1;
            sh.above = above + c1;
        }
        __syncthreads();
        prefix = (prefix << width) | static_cast<Key>(sh.bin);
        need -= sh.above;
        done += width;
    }
    key = prefix;
    ties = need;
}

struct TokenSelectArgs {
    const float* weights; int64_t ld; const int32_t* seq_lens; int max_len;
    int budget, recent;
    int32_t* keep; int32_t* kept_lens; float* kept;
    int kv_heads;
};

// One workgroup per (sequence, kv head).
__global__ __launch_bounds__(kSelThreads) void kv_select_kernel(TokenSelectArgs a) {
    __shared__ SelShared sh;
    const int b = blockIdx.x / a.kv_heads, h = blockIdx.x % a.kv_heads;
    const int len = a.seq_lens ? min(max(a.seq_lens[b], 0), a.max_len) : a.max_len;
    const int n = min(len, a.budget);
    const float* w = a.weights + static_cast<int64_t>(blockIdx.x) * a.ld;
    float* kept = a.kept ? a.kept + static_cast<int64_t>(blockIdx.x) * a.ld : nullptr;
    int32_t* keep = a.keep + static_cast<int64_t>(blockIdx.x) * a.budget;
    if (h == 0 && threadIdx.x == 0) a.kept_lens[b] = n;
    // tokens from `old` on are kept; of those before, `need` of the largest weight
    const int old = max(len - a.recent, 0), need = len > n ? a.budget - a.recent : old;
    uint32_t key = 0;
    int ties = 0;
    if (need > 0 && need < old) select_threshold<uint32_t>([&](int i) { return order_key(w[i]); }, old, need, sh, key, ties);
    const bool all_old = need >= old;
    int written = 0, tied = 0;
    for (int base = 0; base < len; base += kSelThreads) {
        const int i = base + threadIdx.x;
        const float v = i < len ? w[i] : 0.f;
        bool equal = false, take = false;
        if (i < len) {
            if (i >= old || all_old) take = true;
            else if (need > 0) {
                const uint32_t k = order_key(v);
                take = k > key;
                equal = k == key;
            }
        }
        int all;
        const int rank = block_exclusive(equal ? 1 : 0, sh, all);
        if (equal && tied + rank < ties) take = true;
        tied += all;
        const int at = written + block_exclusive(take ? 1 : 0, sh, all);
        written += all;
        // (every load of this chunk is behind the sums' barriers, and later chunks
        // read beyond what is written here: kept may be the weights themselves)
        if (take) {
            keep[at] = i;
            if (kept) kept[at] = v;
        }
    }
    for (int i = n + threadIdx.x; i < a.budget; i += kSelThreads) keep[i] = -1;
    if (kept) {
        __syncthreads();
        for (int64_t i = n + threadIdx.x; i < a.ld; i += kSelThreads) kept[i] = 0.f;
    }
}

// ---------------------------------------------------------------- page scores and selection
struct PageScoreArgs {
    const void* q; int q_f32;
    const void* bounds; const int32_t* page_table; const int32_t* seq_lens; int max_len;
    uint64_t* keys; int64_t max_pages;
    int32_t* selected;
    int q_heads, kv_heads, rows, head_dim, page_tokens, pages_per_seq, num_pages, top, sink, recent;
};

__device__ __forceinline__ int row_pages(const PageScoreArgs& a, int b, int row) {
    const int len = a.seq_lens ? min(max(a.seq_lens[b], 0), a.max_len) : a.max_len;
    return (max(len - a.rows + row + 1, 0) + a.page_tokens - 1) / a.page_tokens;
}

// Workgroups of a (sequence, row, kv head) walk its pages, one wave a page.
template <typename KvT>
__global__ __launch_bounds__(256) void page_score_kernel(PageScoreArgs a) {
    __shared__ double up[kRowMaxD], down[kRowMaxD];
    const int64_t unit = blockIdx.x;
    const int h = static_cast<int>(unit % a.kv_heads);
    const int row = static_cast<int>(unit / a.kv_heads % a.rows), b = static_cast<int>(unit / a.kv_heads / a.rows);
    const int pages = row_pages(a, b, row), D = a.head_dim, G = a.q_heads / a.kv_heads;
    for (int d = threadIdx.x; d < D; d += 256) {
        double hi = 0.0, lo = 0.0;
        for (int g = 0; g < G; ++g) {
            const int64_t at = ((static_cast<int64_t>(b) * a.q_heads + h * G + g) * a.rows + row) * D + d;
            const float v = a.q_f32 ? static_cast<const float*>(a.q)[at] : bf16_to_f32(static_cast<const uint16_t*>(a.q)[at]);
            hi += v > 0.f ? v : 0.f;
            lo += v < 0.f ? v : 0.f;
        }
        up[d] = hi;
        down[d] = lo;
    }
    __syncthreads();
    const int lane = threadIdx.x & 63;
    for (int page = blockIdx.y * 4 + (threadIdx.x >> 6); page < pages; page += gridDim.y * 4) {
        const int id = a.page_table[static_cast<int64_t>(b) * a.pages_per_seq + page];
        double s = 0.0;
        if (id >= 0 && id < a.num_pages) {
            const KvT* lo = static_cast<const KvT*>(a.bounds) + (static_cast<int64_t>(id) * a.kv_heads + h) * 2 * D;
            for (int d = lane; d < D; d += 64) {
                s = fma(up[d], static_cast<double>(kv_f32(lo, D + d)), s);
                s = fma(down[d], static_cast<double>(kv_f32(lo, d)), s);
            }
            s = wave_sum(s);
        } else {
            s = -INFINITY;
        }
        if (lane == 0)
            a.keys[unit * a.max_pages + page] = page < a.sink || page >= pages - a.recent ? ~0ull : order_key(s);
    }
}

__global__ __launch_bounds__(kSelThreads) void page_select_kernel(PageScoreArgs a) {
    __shared__ SelShared sh;
    const int64_t unit = blockIdx.x;
    const int row = static_cast<int>(unit / a.kv_heads % a.rows), b = static_cast<int>(unit / a.kv_heads / a.rows);
    const int pages = row_pages(a, b, row), n = min(pages, a.top);
    const uint64_t* keys = a.keys + unit * a.max_pages;
    int32_t* out = a.selected + unit * a.top;
    uint64_t key = 0;
    int ties = 0;
    if (n < pages) select_threshold<uint64_t>([&](int i) { return keys[i]; }, pages, n, sh, key, ties);
    int written = 0, tied = 0;
    for (int base = 0; base < pages; base += kSelThreads) {
        const int i = base + threadIdx.x;
        const uint64_t k = i < pages ? keys[i] : 0;
        const bool equal = i < pages && n < pages && k == key;
        bool take = i < pages && (n == pages || k > key);
        int all;
        const int rank = block_exclusive(equal ? 1 : 0, sh, all);
        if (equal && tied + rank < ties) take = true;
        tied += all;
        const int at = written + block_exclusive(take ? 1 : 0, sh, all);
        written += all;
        if (take) out[at] = i;
    }
    for (int i = n + threadIdx.x; i < a.top; i += kSelThreads) out[i] = -1;
}

// ---------------------------------------------------------------- compaction
struct CompactArgs {
    void* k_pool; void* v_pool; const int32_t* page_table;
    const int32_t* base; const int32_t* keep; int keep_heads; int64_t keep_ld;
    const int32_t* counts; int32_t* new_lens; int max_keep;
    int kv_heads, head_dim, page_tokens, pages_per_seq, num_pages;
};

__device__ __forceinline__ int kept_length(int base, int n, int capacity) {
    return min(base, capacity) + min(n, max(capacity - base, 0));
}
// The new lengths where they replace the old ones or the counts (which every workgroup
// of the move reads).
__global__ __launch_bounds__(256) void kv_kept_lens_kernel(CompactArgs a, int batch) {
    const int b = blockIdx.x * 256 + threadIdx.x;
    if (b >= batch) return;
    const int base = a.base ? max(a.base[b], 0) : 0, n = min(max(a.counts[b], 0), a.max_keep);
    a.new_lens[b] = kept_length(base, n, a.pages_per_seq * a.page_tokens);
}

// Token base + keep[i] -> base + i, keep[i] >= i.  A later token's source lies behind
// every earlier destination, so a workgroup may read ahead; a chunk is written once
// the whole chunk is read (an earlier token's source may be a later destination of
// the same chunk).
//
// Any head_dim up to 256 and page size: one workgroup per (sequence, kv head), thread
// d moving dim d.
template <typename KvT>
__global__ __launch_bounds__(256) void kv_compact_any_kernel(CompactArgs a) {
    constexpr int kChunk = 8;  // tokens a step
    const int b = blockIdx.x / a.kv_heads, h = blockIdx.x % a.kv_heads;
    const int D = a.head_dim, pt = a.page_tokens;
    const int capacity = a.pages_per_seq * pt;
    const int base = a.base ? max(a.base[b], 0) : 0;
    const int n = min(max(a.counts[b], 0), a.max_keep);
    if (a.new_lens != a.base && a.new_lens != a.counts && h == 0 && threadIdx.x == 0)
        a.new_lens[b] = kept_length(base, n, capacity);
    const int32_t* keep = a.keep + (static_cast<int64_t>(b) * a.keep_heads + (a.keep_heads == 1 ? 0 : h)) * a.keep_ld;
    const int32_t* table = a.page_table + static_cast<int64_t>(b) * a.pages_per_seq;
    KvT* kp = static_cast<KvT*>(a.k_pool);
    KvT* vp = static_cast<KvT*>(a.v_pool);
    const int d = threadIdx.x;  // head_dim <= 256
    for (int i0 = 0; i0 < n; i0 += kChunk) {
        KvT kv[kChunk], vv[kChunk];
        int64_t to[kChunk];
        int slot[kChunk];
#pragma unroll
        for (int e = 0; e < kChunk; ++e) {
            const int i = i0 + e;
            to[e] = -1;
            slot[e] = 0;
            kv[e] = vv[e] = KvT(0);
            if (i >= n) continue;
            const int k = keep[i];
            if (k <= i || k >= capacity - base) continue;  // in its place already, or no such token
            const int src = base + k, dst = base + i;
            const int sp = table[src / pt], dp = table[dst / pt];
            if (sp < 0 || sp >= a.num_pages || dp < 0 || dp >= a.num_pages) continue;
            const int64_t sb = static_cast<int64_t>(sp) * a.kv_heads + h;
            to[e] = static_cast<int64_t>(dp) * a.kv_heads + h;
            slot[e] = dst % pt;
            if (d < D) {
                kv[e] = kp[(sb * pt + src % pt) * D + d];
                vv[e] = vp[(sb * D + d) * pt + src % pt];
            }
        }
        __syncthreads();
#pragma unroll
        for (int e = 0; e < kChunk; ++e)
            if (to[e] >= 0 && d < D) {
                kp[(to[e] * pt + slot[e]) * D + d] = kv[e];
                vp[(to[e] * D + d) * pt + slot[e]] = vv[e];
            }
    }
}

// 16-token pages, K rows of whole 16-byte vectors: the order above binds only what a
// destination shares with a source, so each (sequence, kv head) splits into slices of
// its own -- K by vectors of a row, V by dims -- and a workgroup walks its slice's
// destinations in order.  The sources of 2048 tokens at a time are looked up first
// (list, then table) and kept in LDS, so that a chunk's loads wait on nothing else.
//   K: a thread moves one vector of each of 8 tokens a chunk.
//   V: a thread builds one dim's run of a destination page (16 tokens, 32 or 64 bytes)
//      from its tokens' pages; tokens that stay are read from their own place.
constexpr int kCompactSeg = 2048;
constexpr uint32_t kStays = 0xFFFFFFFFu;

template <typename KvT>
__global__ __launch_bounds__(256) void kv_compact_pages_kernel(CompactArgs a, int k_shift, int d_shift, int k_slices, int slices) {
    constexpr int kVecs = 16 / sizeof(KvT);  // elements of a vector
    __shared__ uint32_t src[kCompactSeg];    // page id * 16 + slot, or kStays
    __shared__ int dpage[kCompactSeg / 16];  // destination pages' ids, -1 where nothing may be written
    const int unit = blockIdx.x / slices, slice = blockIdx.x % slices;
    const int b = unit / a.kv_heads, h = unit % a.kv_heads;
    const int D = a.head_dim;
    const int capacity = a.pages_per_seq * kPageTok;
    const int base = a.base ? min(max(a.base[b], 0), capacity) : 0;
    const int n = min(max(a.counts[b], 0), a.max_keep);
    if (a.new_lens != a.base && a.new_lens != a.counts && h == 0 && slice == 0 && threadIdx.x == 0)
        a.new_lens[b] = kept_length(base, n, capacity);
    const int32_t* keep = a.keep + (static_cast<int64_t>(b) * a.keep_heads + (a.keep_heads == 1 ? 0 : h)) * a.keep_ld;
    const int32_t* table = a.page_table + static_cast<int64_t>(b) * a.pages_per_seq;
    KvT* kp = static_cast<KvT*>(a.k_pool);
    KvT* vp = static_cast<KvT*>(a.v_pool);
    const int end = min(base + n, capacity);  // base + n <= 2^30 + 2^30
    for (int s0 = base & ~15; s0 < end; s0 += kCompactSeg) {
        const int count = min(kCompactSeg, (end - s0 + 15) & ~15);
        __syncthreads();
        for (int q = threadIdx.x; q < count; q += 256) {
            const int pos = s0 + q, i = pos - base;
            uint32_t code = kStays;
            if (pos >= base && pos < end) {
                const int k = keep[i];
                if (k > i && k < capacity - base) {
                    const int id = table[(base + k) / kPageTok];
                    if (id >= 0 && id < a.num_pages) code = static_cast<uint32_t>(id) * kPageTok + ((base + k) & 15);
                }
            }
            src[q] = code;
            if ((q & 15) == 0) {
                const int id = table[pos / kPageTok];
                dpage[q / 16] = id >= 0 && id < a.num_pages ? id : -1;
            }
        }
        __syncthreads();
        if (slice < k_slices) {
            const int vecs = D / kVecs;
            const int vec = (slice << k_shift) + (threadIdx.x & ((1 << k_shift) - 1));
            const int per = 256 >> k_shift;  // tokens a step of the workgroup
            uint4* kv4 = reinterpret_cast<uint4*>(kp);
            for (int c0 = 0; c0 < count; c0 += 8 * per) {
                uint4 r[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const int q = c0 + j * per + (threadIdx.x >> k_shift);
                    const uint32_t code = q < count ? src[q] : kStays;
                    r[j] = make_uint4(0, 0, 0, 0);
                    if (code != kStays && vec < vecs)
                        r[j] = kv4[((static_cast<int64_t>(code >> 4) * a.kv_heads + h) * kPageTok + (code & 15)) * vecs + vec];
                }
                __syncthreads();
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const int q = c0 + j * per + (threadIdx.x >> k_shift);
                    if (q < count && src[q] != kStays && dpage[q / 16] >= 0 && vec < vecs)
                        kv4[((static_cast<int64_t>(dpage[q / 16]) * a.kv_heads + h) * kPageTok + (q & 15)) * vecs + vec] = r[j];
                }
            }
        } else {
            const int d = ((slice - k_slices) << d_shift) + (threadIdx.x & ((1 << d_shift) - 1));
            const int per = 256 >> d_shift;  // pages a step
            for (int g0 = 0; g0 < count / 16; g0 += per) {
                const int g = g0 + (threadIdx.x >> d_shift);
                KvT r[kPageTok];
                bool moves = false;
                int64_t own = 0;
                if (g < count / 16 && d < D && dpage[g] >= 0) {
                    own = ((static_cast<int64_t>(dpage[g]) * a.kv_heads + h) * D + d) * kPageTok;
#pragma unroll
                    for (int e = 0; e < kPageTok; ++e) moves |= src[16 * g + e] != kStays;
                    if (moves)
#pragma unroll
                        for (int e = 0; e < kPageTok; ++e) {
                            const uint32_t code = src[16 * g + e];
                            const int64_t at = ((static_cast<int64_t>(code >> 4) * a.kv_heads + h) * D + d) * kPageTok + (code & 15);
                            r[e] = vp[code == kStays ? own + e : at];
                        }
                }
                __syncthreads();
                if (moves) {
                    constexpr int kRun = kPageTok * sizeof(KvT) / 16;
                    uint4 w[kRun];
                    __builtin_memcpy(w, r, sizeof w);
#pragma unroll
                    for (int e = 0; e < kRun; ++e) reinterpret_cast<uint4*>(vp + own)[e] = w[e];
                }
            }
        }
    }
}

}  // namespace

void launch_page_bounds(const void* k_pool, int pool_dtype, const int32_t* page_table, const int32_t* seq_lens,
                        int64_t max_context, int64_t fresh, void* bounds, int64_t batch, int64_t kv_heads,
                        int64_t head_dim, int64_t page_tokens, int64_t pages_per_seq, int64_t num_pages,
                        hipStream_t stream) {
    BoundsArgs a{};
    a.k_pool = k_pool; a.page_table = page_table; a.seq_lens = seq_lens; a.max_len = static_cast<int>(max_context);
    a.fresh = fresh; a.bounds = bounds;
    a.kv_heads = static_cast<int>(kv_heads); a.head_dim = static_cast<int>(head_dim);
    a.page_tokens = static_cast<int>(page_tokens); a.pages_per_seq = static_cast<int>(pages_per_seq);
    a.num_pages = static_cast<int>(num_pages);
    // the newest `fresh` tokens touch at most this many pages
    const int64_t newest = std::min(fresh, max_context);
    const int64_t pages = std::min((max_context + page_tokens - 1) / page_tokens, (newest + page_tokens - 2) / page_tokens + 1);
    const dim3 grid(static_cast<unsigned>(batch * kv_heads), static_cast<unsigned>(std::min<int64_t>(pages, 65535)));
    if (pool_dtype == SFG_F32) page_bounds_kernel<float><<<grid, 64, 0, stream>>>(a);
    else page_bounds_kernel<uint16_t><<<grid, 64, 0, stream>>>(a);
}

size_t page_select_workspace_bytes(int64_t batch, int64_t kv_heads, int64_t rows, int64_t max_pages) {
    return (static_cast<size_t>(batch) * kv_heads * rows * max_pages * sizeof(uint64_t) + 255) / 256 * 256;
}

void launch_page_select(const ChosenLaunch& c, const void* bounds, int64_t sink, int64_t recent, int32_t* selected,
                        void* workspace, hipStream_t stream) {
    PageScoreArgs a{};
    a.q = c.q; a.q_f32 = c.q_dtype == SFG_F32;
    a.bounds = bounds; a.page_table = c.page_table; a.seq_lens = c.seq_lens; a.max_len = static_cast<int>(c.max_context);
    a.keys = static_cast<uint64_t*>(workspace); a.max_pages = (c.max_context + c.page_tokens - 1) / c.page_tokens;
    a.selected = selected;
    a.q_heads = static_cast<int>(c.q_heads); a.kv_heads = static_cast<int>(c.kv_heads);
    a.rows = static_cast<int>(c.rows); a.head_dim = static_cast<int>(c.head_dim);
    a.page_tokens = static_cast<int>(c.page_tokens); a.pages_per_seq = static_cast<int>(c.pages_per_seq);
    a.num_pages = static_cast<int>(c.num_pages); a.top = static_cast<int>(c.top);
    a.sink = static_cast<int>(sink); a.recent = static_cast<int>(recent);
    const unsigned units = static_cast<unsigned>(c.batch * c.rows * c.kv_heads);
    const dim3 grid(units, static_cast<unsigned>(std::min<int64_t>((a.max_pages + 15) / 16, 1024)));
    if (c.kv_dtype == SFG_F32) page_score_kernel<float><<<grid, 256, 0, stream>>>(a);
    else page_score_kernel<uint16_t><<<grid, 256, 0, stream>>>(a);
    page_select_kernel<<<units, kSelThreads, 0, stream>>>(a);
}

void launch_kv_select(const float* weights, int64_t ld, const int32_t* seq_lens, int64_t max_context, int64_t budget,
                      int64_t recent, int32_t* keep, int32_t* kept_lens, float* kept_weights, int64_t batch,
                      int64_t kv_heads, hipStream_t stream) {
    TokenSelectArgs a{};
    a.weights = weights; a.ld = ld; a.seq_lens = seq_lens; a.max_len = static_cast<int>(max_context);
    a.budget = static_cast<int>(budget); a.recent = static_cast<int>(recent);
    a.keep = keep; a.kept_lens = kept_lens; a.kept = kept_weights; a.kv_heads = static_cast<int>(kv_heads);
    kv_select_kernel<<<static_cast<unsigned>(batch * kv_heads), kSelThreads, 0, stream>>>(a);
}

void launch_kv_compact(void* k_pool, void* v_pool, int pool_dtype, const int32_t* page_table, const int32_t* base,
                       const int32_t* keep, int64_t keep_heads, int64_t keep_ld, const int32_t* counts,
                       int32_t* new_lens, int64_t max_keep, int64_t batch, int64_t kv_heads, int64_t head_dim,
                       int64_t page_tokens, int64_t pages_per_seq, int64_t num_pages, hipStream_t stream) {
    CompactArgs a{};
    a.k_pool = k_pool; a.v_pool = v_pool; a.page_table = page_table;
    a.base = base; a.keep = keep; a.keep_heads = static_cast<int>(keep_heads); a.keep_ld = keep_ld;
    a.counts = counts; a.new_lens = new_lens; a.max_keep = static_cast<int>(max_keep);
    a.kv_heads = static_cast<int>(kv_heads); a.head_dim = static_cast<int>(head_dim);
    a.page_tokens = static_cast<int>(page_tokens); a.pages_per_seq = static_cast<int>(pages_per_seq);
    a.num_pages = static_cast<int>(num_pages);
    const int64_t units = batch * kv_heads, esz = pool_dtype == SFG_F32 ? 4 : 2;
    const bool pages = page_tokens == kPageTok && head_dim * esz % 16 == 0 && num_pages <= (1 << 27) &&
                       ((reinterpret_cast<uintptr_t>(k_pool) | reinterpret_cast<uintptr_t>(v_pool)) & 15) == 0;
    if (pages) {
        // slices of 16 vectors and 64 dims, halved while fewer than 512 workgroups result
        int k_shift = 4, d_shift = 6;
        const int64_t vecs = head_dim * esz / 16;
        auto ks = [&] { return (vecs + (1 << k_shift) - 1) >> k_shift; };
        auto ds = [&] { return (head_dim + (1 << d_shift) - 1) >> d_shift; };
        while (k_shift > 1 && units * (ks() + ds()) < 512) {
            --k_shift;
            --d_shift;
        }
        const int slices = static_cast<int>(ks() + ds());
        const unsigned grid = static_cast<unsigned>(units * slices);
        if (pool_dtype == SFG_F32) kv_compact_pages_kernel<float><<<grid, 256, 0, stream>>>(a, k_shift, d_shift, static_cast<int>(ks()), slices);
        else kv_compact_pages_kernel<uint16_t><<<grid, 256, 0, stream>>>(a, k_shift, d_shift, static_cast<int>(ks()), slices);
    } else if (pool_dtype == SFG_F32) {
        kv_compact_any_kernel<float><<<static_cast<unsigned>(units), 256, 0, stream>>>(a);
    } else {
        kv_compact_any_kernel<uint16_t><<<static_cast<unsigned>(units), 256, 0, stream>>>(a);
    }
    if (new_lens == base || new_lens == counts)
        kv_kept_lens_kernel<<<static_cast<unsigned>((batch + 255) / 256), 256, 0, stream>>>(a, static_cast<int>(batch));
}

}  // namespace sfg
