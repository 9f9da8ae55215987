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
#include <type_traits>

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

// Any head_dim and page size: one wave per (sequence, kv head) and page, from the newest page back, lane d owning
// dims d, d + 64, ...; a page is read whole, up to the sequence's end.
template <typename KvT>
__global__ __launch_bounds__(64) void page_bounds_any_kernel(BoundsArgs a) {
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
            if (!(lo <= hi)) lo = hi = NAN;  // no key but NaN
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

// head_dim 64 / 128, 16-token pages: a row is read as 16-byte vectors, 64 of them a load of
// the wave, all of the page's loads before the first comparison (slots past the end
// re-read the last token); lanes of the same vector and other tokens meet by shuffles.
// 3.7 us for the newest page of 16 x 8 heads (12.0 with the loads one by one), 4.5 for all
// of 2 x 4 heads x 6000 tokens.
template <typename KvT, int kD>
__global__ __launch_bounds__(64) void page_bounds_kernel(BoundsArgs a) {
    constexpr int kEl = 16 / sizeof(KvT), kVecs = kD / kEl, kTok = 64 / kVecs, kLoads = kPageTok / kTok;
    const int b = blockIdx.x / a.kv_heads, h = blockIdx.x % a.kv_heads;
    const int len = a.seq_lens ? min(max(a.seq_lens[b], 0), a.max_len) : a.max_len;
    const int lane = threadIdx.x, vec = lane % kVecs, tok = lane / kVecs;
    for (int page = (len + kPageTok - 1) / kPageTok - 1 - static_cast<int>(blockIdx.y);
         page >= 0 && static_cast<int64_t>(page + 1) * kPageTok > len - a.fresh; page -= static_cast<int>(gridDim.y)) {
        const int id = a.page_table[static_cast<int64_t>(b) * a.pages_per_seq + page];
        if (id < 0 || id >= a.num_pages) continue;
        const int last = min(kPageTok, len - page * kPageTok) - 1;
        const int64_t blk = static_cast<int64_t>(id) * a.kv_heads + h;
        const uint4* k = reinterpret_cast<const uint4*>(static_cast<const KvT*>(a.k_pool) + blk * kPageTok * kD);
        uint4 w[kLoads];
#pragma unroll
        for (int i = 0; i < kLoads; ++i) w[i] = k[min(kTok * i + tok, last) * kVecs + vec];
        float lo[kEl], hi[kEl];
#pragma unroll
        for (int e = 0; e < kEl; ++e) {
            lo[e] = INFINITY;
            hi[e] = -INFINITY;
        }
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            KvT v[kEl];
            __builtin_memcpy(v, &w[i], sizeof v);
#pragma unroll
            for (int e = 0; e < kEl; ++e) {
                lo[e] = fminf(lo[e], kv_f32(v, e));
                hi[e] = fmaxf(hi[e], kv_f32(v, e));
            }
        }
#pragma unroll
        for (int o = kVecs; o < 64; o <<= 1)
#pragma unroll
            for (int e = 0; e < kEl; ++e) {
                lo[e] = fminf(lo[e], __shfl_xor(lo[e], o, 64));
                hi[e] = fmaxf(hi[e], __shfl_xor(hi[e], o, 64));
            }
        if (tok == 0) {
            KvT v[2][kEl];
#pragma unroll
            for (int e = 0; e < kEl; ++e) {
                if (!(lo[e] <= hi[e])) lo[e] = hi[e] = NAN;  // no key but NaN
                if constexpr (sizeof(KvT) == 4) {
                    v[0][e] = lo[e];
                    v[1][e] = hi[e];
                } else {  // values of the pool: exact
                    v[0][e] = f32_to_bf16(lo[e]);
                    v[1][e] = f32_to_bf16(hi[e]);
                }
            }
            uint4* out = reinterpret_cast<uint4*>(static_cast<KvT*>(a.bounds) + blk * 2 * kD);
            uint4 x[2];
            __builtin_memcpy(x, v, sizeof x);
            out[vec] = x[0];
            out[kVecs + vec] = x[1];
        }
    }
}

// ---------------------------------------------------------------- selection
// One workgroup of NT threads selects among n values in tiles of NT * K: wave w holds
// 64 K consecutive ones, lane l those at l, l + 64, ... (loads coalesce, and a ballot
// gives the order inside a wave).  Values of one tile stay in registers; those of more
// are read again for each pass.
constexpr int kSelBits = 11, kSelBins = 1 << kSelBits;
constexpr int kSelFew = 64;

template <typename Key, int NT>
struct SelShared {
    int hist[kSelBins];
    int sum[NT / 64], equal[NT / 64];
    Key ones[NT / 64], all[NT / 64];
    Key few[kSelFew];
    int bin, above, count, fill;
    Key found; int ties;
};

// OR over the wave, in every lane (an AND is the complement of the complements' OR).
__device__ __forceinline__ uint32_t wave_or(uint32_t v) {
    int x = static_cast<int>(v);
    x |= __builtin_amdgcn_update_dpp(0, x, 0x111, 0xF, 0xF, false);
    x |= __builtin_amdgcn_update_dpp(0, x, 0x112, 0xF, 0xF, false);
    x |= __builtin_amdgcn_update_dpp(0, x, 0x114, 0xF, 0xF, false);
    x |= __builtin_amdgcn_update_dpp(0, x, 0x118, 0xF, 0xF, false);
    x |= __builtin_amdgcn_update_dpp(0, x, 0x142, 0xA, 0xF, false);
    x |= __builtin_amdgcn_update_dpp(0, x, 0x143, 0xC, 0xF, false);
    return static_cast<uint32_t>(__builtin_amdgcn_readlane(x, 63));
}
__device__ __forceinline__ uint64_t wave_or(uint64_t v) {
    return static_cast<uint64_t>(wave_or(static_cast<uint32_t>(v))) |
           (static_cast<uint64_t>(wave_or(static_cast<uint32_t>(v >> 32))) << 32);
}
__device__ __forceinline__ int bit_length(uint32_t v) { return v ? 32 - __clz(static_cast<int>(v)) : 0; }
__device__ __forceinline__ int bit_length(uint64_t v) { return v ? 64 - __clzll(static_cast<long long>(v)) : 0; }

// The need-th largest of the candidates (1 <= need <= their number): every key above
// `key` is taken and `ties` of those equal to it.  Radix selection below the bits that
// all keys share, 11 bits a pass: the workgroup counts a digit of the keys that match
// the digits found so far; the bin in which the count from above passes `need` is the
// next digit.  Once that bin holds at most 64 keys, one wave ranks them.  Barriers and
// dependent LDS steps bound it: 2048 page scores 7.2 us, 4096 token weights 9.2 us, both
// with their loads and the list, for 128 workgroups or one.
// each(f): calls f(key) for every candidate key of this thread.
template <typename Key, int NT, typename Each>
__device__ __forceinline__ void select_threshold(Each each, int need, SelShared<Key, NT>& sh, Key& key, int& ties) {
    constexpr int kBits = sizeof(Key) * 8, kWaves = NT / 64, kOwn = kSelBins / NT;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    Key ones = 0, zeros = 0;  // bits that are set, or clear, in some key
    each([&](Key k) __attribute__((always_inline)) {
        ones |= k;
        zeros |= ~k;
    });
    ones = wave_or(ones);
    zeros = wave_or(zeros);
    if (lane == 0) {
        sh.ones[wave] = ones;
        sh.all[wave] = zeros;
    }
#pragma unroll
    for (int i = 0; i < kOwn; ++i) sh.hist[threadIdx.x + i * NT] = 0;
    __syncthreads();
    ones = zeros = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
        ones |= sh.ones[w];
        zeros |= sh.all[w];
    }
    // bits from `open` down are not known yet; keys that match agree with `key` above them
    int open = bit_length(static_cast<Key>(ones & zeros));
    key = open == kBits ? Key(0) : ones >> open;
    while (open > 0) {
        const int width = min(kSelBits, open), shift = open - width;
        each([&](Key k) __attribute__((always_inline)) {
            if (open == kBits || (k >> open) == key) atomicAdd(&sh.hist[static_cast<int>(k >> shift) & ((1 << width) - 1)], 1);
        });
        __syncthreads();
        // kOwn bins a thread, counted from the top one
        const int top = kSelBins - 1 - kOwn * static_cast<int>(threadIdx.x);
        int c[kOwn], mine = 0;
#pragma unroll
        for (int i = 0; i < kOwn; ++i) {
            c[i] = sh.hist[top - i];
            mine += c[i];
        }
        const int upto = wave_inclusive(mine);
        if (lane == 63) sh.sum[wave] = upto;
        if (threadIdx.x == 0) sh.fill = 0;
        __syncthreads();
        int above = upto - mine;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) above += w < wave ? sh.sum[w] : 0;
#pragma unroll
        for (int i = 0; i < kOwn; ++i) {
            if (above < need && need <= above + c[i]) {
                sh.bin = top - i;
                sh.above = above;
                sh.count = c[i];
            }
            above += c[i];
            sh.hist[top - i] = 0;  // for the next pass
        }
        __syncthreads();
        key = (key << width) | static_cast<Key>(sh.bin);
        need -= sh.above;
        open = shift;
        const int count = sh.count;
        if (open > 0 && count <= kSelFew) {
            each([&](Key k) __attribute__((always_inline)) {
                if ((k >> open) == key) sh.few[atomicAdd(&sh.fill, 1)] = k;
            });
            __syncthreads();
            // the key with fewer than `need` above it and at least `need` not below it
            if (wave == 0) {
                const Key me = lane < count ? sh.few[lane] : Key(0);
                int over = 0, same = 0;
                for (int i = 0; i < count; ++i) {
                    const Key k = sh.few[i];
                    over += k > me;
                    same += k == me;
                }
                if (lane < count && over < need && need <= over + same) {
                    sh.found = me;
                    sh.ties = need - over;
                }
            }
            __syncthreads();
            key = sh.found;
            need = sh.ties;
            open = 0;
        }
    }
    ties = need;
}

__device__ __forceinline__ int lanes_below(uint64_t mask) {
    return __builtin_amdgcn_mbcnt_hi(static_cast<uint32_t>(mask >> 32), __builtin_amdgcn_mbcnt_lo(static_cast<uint32_t>(mask), 0));
}

// Emits, ascending, the indexes taken among [0, n): those with must(i), and of the
// candidates (the others) the `need` largest keys, ties to the lower index.
// load(i): value i; to_key(value); emit(at, i, value).  A tile's values are all read
// before anything of it is emitted.
template <typename Key, int NT, int K, typename Load, typename ToKey, typename Must, typename Emit>
__device__ __forceinline__ void select_and_emit(int n, int need, bool everything, Load load, ToKey to_key, Must must, Emit emit,
                                                SelShared<Key, NT>& sh) {
    constexpr int kTile = NT * K, kWaves = NT / 64;
    const bool single = n <= kTile;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int first = wave * 64 * K + lane;
    decltype(load(0)) v[K];
    auto read = [&](int tile) __attribute__((always_inline)) {
#pragma unroll
        for (int r = 0; r < K; ++r) {
            const int i = tile + first + 64 * r;
            v[r] = load(min(i, n - 1));
        }
    };
    if (n > 0 && single) read(0);
    Key key = 0;
    int ties = 0;
    const bool ranked = !everything && need > 0;
    if (ranked)
        select_threshold<Key, NT>([&](auto f) __attribute__((always_inline)) {
            for (int tile = 0; tile < n; tile += kTile) {
                if (!single) read(tile);
#pragma unroll
                for (int r = 0; r < K; ++r) {
                    const int i = tile + first + 64 * r;
                    if (i < n && !must(i)) f(to_key(v[r]));
                }
            }
        }, need, sh, key, ties);
    int written = 0, tied = 0;
    for (int tile = 0; tile < n; tile += kTile) {
        if (!single) read(tile);
        uint64_t sure[K], equal[K];
        int n_sure = 0, n_equal = 0;
#pragma unroll
        for (int r = 0; r < K; ++r) {
            const int i = tile + first + 64 * r;
            const bool in = i < n, fixed = everything || must(i);
            const Key k = to_key(v[r]);
            sure[r] = __ballot(in && (fixed || (ranked && k > key)));
            equal[r] = __ballot(in && !fixed && ranked && k == key);
            n_sure += __popcll(sure[r]);
            n_equal += __popcll(equal[r]);
        }
        __syncthreads();
        if (lane == 0) {
            sh.sum[wave] = n_sure;
            sh.equal[wave] = n_equal;
        }
        __syncthreads();
        int sure_before = 0, sure_all = 0, equal_before = 0, equal_all = 0;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            const int s = sh.sum[w], e = sh.equal[w];
            sure_before += w < wave ? s : 0;
            equal_before += w < wave ? e : 0;
            sure_all += s;
            equal_all += e;
        }
        int rank = tied + equal_before;
        int at = written + sure_before + min(rank, ties) - min(tied, ties);
#pragma unroll
        for (int r = 0; r < K; ++r) {
            const bool tie = (equal[r] >> lane) & 1u;
            const bool take = ((sure[r] >> lane) & 1u) || (tie && rank + lanes_below(equal[r]) < ties);
            const uint64_t taken = __ballot(take);
            if (take) emit(at + lanes_below(taken), tile + first + 64 * r, v[r]);
            at += __popcll(taken);
            rank += __popcll(equal[r]);
        }
        written += sure_all + min(tied + equal_all, ties) - min(tied, ties);
        tied += equal_all;
    }
}

struct TokenSelectArgs {
    const float* weights; int64_t ld; const int32_t* seq_lens; int max_len;
    int budget, recent;
    int32_t* keep; int32_t* kept_lens; float* kept;
    int kv_heads;
};

// One workgroup per (sequence, kv head).
template <int NT, int K>
__global__ __launch_bounds__(NT) void kv_select_kernel(TokenSelectArgs a) {
    __shared__ SelShared<uint32_t, NT> sh;
    const int b = blockIdx.x / a.kv_heads, h = blockIdx.x % a.kv_heads;
    const int len = a.seq_lens ? min(max(a.seq_lens[b], 0), a.max_len) : a.max_len;
    const int n = min(len, a.budget);
    const float* w = a.weights + static_cast<int64_t>(blockIdx.x) * a.ld;
    float* kept = a.kept ? a.kept + static_cast<int64_t>(blockIdx.x) * a.ld : nullptr;
    int32_t* keep = a.keep + static_cast<int64_t>(blockIdx.x) * a.budget;
    if (h == 0 && threadIdx.x == 0) a.kept_lens[b] = n;
    // tokens from `old` on are kept; of those before, budget - recent of the largest weight
    const int old = max(len - a.recent, 0);
    // (kept may be the weights themselves: a token's place in the list is at or before its
    // position, so what a tile writes no later tile reads)
    select_and_emit<uint32_t, NT, K>(
        len, a.budget - a.recent, len <= a.budget, [&](int i) { return w[i]; }, [](float v) { return order_key(v); },
        [&](int i) { return i >= old; },
        [&](int at, int i, float v) {
            keep[at] = i;
            if (kept) kept[at] = v;
        }, sh);
    for (int i = n + threadIdx.x; i < a.budget; i += NT) keep[i] = -1;
    if (kept) {
        __syncthreads();
        for (int64_t i = n + threadIdx.x; i < a.ld; i += NT) kept[i] = 0.f;
    }
}

// ---------------------------------------------------------------- page scores and selection
struct PageScoreArgs {
    const void* q; int q_f32;
    const void* bounds; const int32_t* page_table; const int32_t* seq_lens; int max_len;
    uint64_t* keys; int64_t max_pages;
    int32_t* selected;
    int q_heads, kv_heads, rows, head_dim, page_tokens, pages_per_seq, num_pages, top, sink, recent;
    int pages_per_wave;
};

__device__ __forceinline__ int row_pages(const PageScoreArgs& a, int b, int row) {
    const int len = a.seq_lens ? min(max(a.seq_lens[b], 0), a.max_len) : a.max_len;
    return (max(len - a.rows + row + 1, 0) + a.page_tokens - 1) / a.page_tokens;
}

__device__ __forceinline__ double query_at(const PageScoreArgs& a, int b, int head, int row, int d) {
    const int64_t at = ((static_cast<int64_t>(b) * a.q_heads + head) * a.rows + row) * a.head_dim + d;
    return a.q_f32 ? static_cast<const float*>(a.q)[at] : bf16_to_f32(static_cast<const uint16_t*>(a.q)[at]);
}

// The score is the sum over the group's heads and the dims of max(q lo, q hi).  Of numbers that
// is sum_d P_d hi_d + N_d lo_d, P and N the group's sums of max(q, 0) and min(q, 0), which
// makes the work per page independent of the group's size: P and N to LDS.  An infinite or
// NaN bound or query leaves that sum infinite or NaN (P or N times it is, 0 * inf included),
// and the page is then summed term by term.
__device__ __forceinline__ void group_query(const PageScoreArgs& a, int b, int h, int row, double* up, double* down) {
    const int D = a.head_dim, G = a.q_heads / a.kv_heads;
    for (int d = threadIdx.x; d < D; d += 256) {
        double hi = 0.0, lo = 0.0;
        for (int g = 0; g < G; ++g) {
            const double v = query_at(a, b, h * G + g, row, d);
            hi += v < 0.0 ? 0.0 : v;  // (NaN too)
            lo += v < 0.0 ? v : 0.0;
        }
        up[d] = hi;
        down[d] = lo;
    }
    __syncthreads();
}

// The terms of one dim: the larger of q lo and q hi of each head, NaN if either is.
__device__ __forceinline__ double dim_score(const PageScoreArgs& a, int b, int h, int row, int d, double lo, double hi) {
    const int G = a.q_heads / a.kv_heads;
    double s = 0.0;
    for (int g = 0; g < G; ++g) {
        const double v = query_at(a, b, h * G + g, row, d), x = v * lo, y = v * hi;
        s += x != x || x > y ? x : y;
    }
    return s;
}
__device__ __forceinline__ bool is_number(double s) { return fabs(s) < INFINITY; }

// Any head_dim: workgroups of a (sequence, row, kv head) walk its pages, one wave a page.
template <typename KvT>
__global__ __launch_bounds__(256) void page_score_any_kernel(PageScoreArgs a) {
    __shared__ double up[kRowMaxD], down[kRowMaxD];
    const int64_t unit = blockIdx.x;
    const int h = static_cast<int>(unit % a.kv_heads);
    const int row = static_cast<int>(unit / a.kv_heads % a.rows), b = static_cast<int>(unit / a.kv_heads / a.rows);
    const int pages = row_pages(a, b, row), D = a.head_dim;
    if (static_cast<int>(blockIdx.y) * 4 >= pages) return;
    group_query(a, b, h, row, up, down);
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
            if (!is_number(s)) {
                s = 0.0;
                for (int d = lane; d < D; d += 64) s += dim_score(a, b, h, row, d, kv_f32(lo, d), kv_f32(lo, D + d));
                s = wave_sum(s);
            }
        } else {
            s = -INFINITY;
        }
        if (lane == 0) a.keys[unit * a.max_pages + page] = order_key(s);
    }
}

// The value of lane l ^ X in 16-lane rows, both halves of a double.
template <int X>
__device__ __forceinline__ double lane_xor_f64(double v) {
    const uint64_t u = static_cast<uint64_t>(__double_as_longlong(v));
    float lo = __uint_as_float(static_cast<uint32_t>(u)), hi = __uint_as_float(static_cast<uint32_t>(u >> 32));
    if constexpr (X == 1) { lo = lane_xor1(lo); hi = lane_xor1(hi); }
    else if constexpr (X == 2) { lo = lane_xor2(lo); hi = lane_xor2(hi); }
    else if constexpr (X == 4) { lo = lane_xor4(lo); hi = lane_xor4(hi); }
    else { lo = lane_xor8(lo); hi = lane_xor8(hi); }
    return __longlong_as_double(static_cast<long long>((static_cast<uint64_t>(__float_as_uint(hi)) << 32) | __float_as_uint(lo)));
}

// head_dim 64 / 128: 8 or 16 lanes a page, eight dims each, their P and N in registers;
// a wave takes 8 or 4 pages at a time, four such groups' bounds in flight.  Bound by
// reading the bounds (4 D bytes a bf16 page and head): 74 MB, 16 x 8 heads x up to 2048
// pages (lengths of their own), in 18 us from a warm cache, 4.0 TB/s; the 2 D
// double-precision FMAs a page stay under it.
template <typename KvT, int kD>
__global__ __launch_bounds__(256) void page_score_kernel(PageScoreArgs a) {
    constexpr int kLanes = kD / 8, kPer = 64 / kLanes, kGroups = 4;
    __shared__ double up[kD], down[kD];
    const int64_t unit = blockIdx.x;
    const int h = static_cast<int>(unit % a.kv_heads);
    const int row = static_cast<int>(unit / a.kv_heads % a.rows), b = static_cast<int>(unit / a.kv_heads / a.rows);
    const int pages = row_pages(a, b, row);
    if (static_cast<int>(blockIdx.y) * 4 * a.pages_per_wave >= pages) return;
    group_query(a, b, h, row, up, down);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int sub = lane / kLanes, d0 = (lane % kLanes) * 8;
    double P[8], N[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        P[e] = up[d0 + e];
        N[e] = down[d0 + e];
    }
    const int begin = (static_cast<int>(blockIdx.y) * 4 + wave) * a.pages_per_wave;
    const int end = min(begin + a.pages_per_wave, pages);
    // pages_per_wave is at most 64: the wave's page ids, one a lane
    const int mine = begin + lane < end ? a.page_table[static_cast<int64_t>(b) * a.pages_per_seq + begin + lane] : -1;
    uint64_t* keys = a.keys + unit * a.max_pages;
    auto page_sum = [](double s) __attribute__((always_inline)) {  // over the lanes of a page
        s += lane_xor_f64<1>(s);
        s += lane_xor_f64<2>(s);
        s += lane_xor_f64<4>(s);
        if constexpr (kLanes == 16) s += lane_xor_f64<8>(s);
        return s;
    };
    for (int p0 = begin; p0 < end; p0 += kPer * kGroups) {
        constexpr int kV = 8 * sizeof(KvT) / 16;  // vectors of eight dims
        uint4 lo[kGroups][kV], hi[kGroups][kV];
        bool ok[kGroups];
        int odd = 0;  // bit g: the lane's page of group g has no number as its score
#pragma unroll
        for (int g = 0; g < kGroups; ++g) {
            const int page = p0 + g * kPer + sub;
            const int id = __shfl(mine, (page - begin) & 63, 64);
            ok[g] = page < end && id >= 0 && id < a.num_pages;
            const KvT* at = static_cast<const KvT*>(a.bounds) + (static_cast<int64_t>(ok[g] ? id : 0) * a.kv_heads + h) * 2 * kD + d0;
#pragma unroll
            for (int v = 0; v < kV; ++v) {
                lo[g][v] = reinterpret_cast<const uint4*>(at)[v];
                hi[g][v] = reinterpret_cast<const uint4*>(at + kD)[v];
            }
        }
#pragma unroll
        for (int g = 0; g < kGroups; ++g) {
            KvT l[8], u[8];
            __builtin_memcpy(l, lo[g], sizeof l);
            __builtin_memcpy(u, hi[g], sizeof u);
            double s = 0.0;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                s = fma(P[e], static_cast<double>(kv_f32(u, e)), s);
                s = fma(N[e], static_cast<double>(kv_f32(l, e)), s);
            }
            s = page_sum(s);
            odd |= ok[g] && !is_number(s) ? 1 << g : 0;
            const int page = p0 + g * kPer + sub;
            if (lane % kLanes == 0 && page < end) keys[page] = order_key(ok[g] ? s : -INFINITY);
        }
        if (!__any(odd)) continue;
#pragma unroll 1
        for (int g = 0; g < kGroups; ++g) {  // (only those: a sum in another order would part equal pages)
            const int page = p0 + g * kPer + sub;
            const int id = __shfl(mine, (page - begin) & 63, 64);
            double s = 0.0;
            if ((odd >> g) & 1) {
                const KvT* at = static_cast<const KvT*>(a.bounds) + (static_cast<int64_t>(id) * a.kv_heads + h) * 2 * kD + d0;
#pragma unroll 1
                for (int e = 0; e < 8; ++e) s += dim_score(a, b, h, row, d0 + e, kv_f32(at, e), kv_f32(at, kD + e));
            }
            s = page_sum(s);
            if (((odd >> g) & 1) && lane % kLanes == 0) keys[page] = order_key(s);
        }
    }
}

template <int NT, int K>
__global__ __launch_bounds__(NT) void page_select_kernel(PageScoreArgs a) {
    __shared__ SelShared<uint64_t, NT> sh;
    const int64_t unit = blockIdx.x;
    const int row = static_cast<int>(unit / a.kv_heads % a.rows), b = static_cast<int>(unit / a.kv_heads / a.rows);
    const int pages = row_pages(a, b, row), n = min(pages, a.top);
    const uint64_t* keys = a.keys + unit * a.max_pages;
    int32_t* out = a.selected + unit * a.top;
    // (top >= sink + recent: with more pages than top, the first and the newest do not meet)
    select_and_emit<uint64_t, NT, K>(
        pages, a.top - a.sink - a.recent, pages <= a.top, [&](int i) { return keys[i]; }, [](uint64_t k) { return k; },
        [&](int i) { return i < a.sink || i >= pages - a.recent; }, [&](int at, int i, uint64_t) { out[at] = i; }, sh);
    for (int i = n + threadIdx.x; i < a.top; i += NT) out[i] = -1;
}

// Threads and values a thread for up to n values: four waves while they hold them all
// (fewer waves pass their barriers sooner), else sixteen.
template <typename Go>
void by_size(int64_t n, Go go) {
    if (n <= 512) go(std::integral_constant<int, 256>{}, std::integral_constant<int, 2>{});
    else if (n <= 2048) go(std::integral_constant<int, 256>{}, std::integral_constant<int, 8>{});
    else if (n <= 4096) go(std::integral_constant<int, 1024>{}, std::integral_constant<int, 4>{});
    else go(std::integral_constant<int, 1024>{}, std::integral_constant<int, 16>{});
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
// 16 x 8 heads, up to 4096 tokens to 2048: 80 us for 178 MB read (the kept K rows, V's
// lines that hold kept tokens) and 134 written, 104 together with the selection where
// nothing is cached.  Not
// faster: finer slices (129 us at 1024 workgroups), the next chunk's loads before this
// one's stores (110), V as 16-byte vectors shared by a page's tokens (110).
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
    const bool fast = (head_dim == 64 || head_dim == 128) && page_tokens == kPageTok &&
                      ((reinterpret_cast<uintptr_t>(k_pool) | reinterpret_cast<uintptr_t>(bounds)) & 15) == 0;
    if (fast && pool_dtype == SFG_F32) {
        if (head_dim == 128) page_bounds_kernel<float, 128><<<grid, 64, 0, stream>>>(a);
        else page_bounds_kernel<float, 64><<<grid, 64, 0, stream>>>(a);
    } else if (fast) {
        if (head_dim == 128) page_bounds_kernel<uint16_t, 128><<<grid, 64, 0, stream>>>(a);
        else page_bounds_kernel<uint16_t, 64><<<grid, 64, 0, stream>>>(a);
    } else if (pool_dtype == SFG_F32) {
        page_bounds_any_kernel<float><<<grid, 64, 0, stream>>>(a);
    } else {
        page_bounds_any_kernel<uint16_t><<<grid, 64, 0, stream>>>(a);
    }
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
    const bool fast = (c.head_dim == 64 || c.head_dim == 128) && (reinterpret_cast<uintptr_t>(bounds) & 15) == 0;
    // a wave takes 64 pages, fewer while that leaves CUs idle
    a.pages_per_wave = 64;
    while (a.pages_per_wave > 16 && units * ((a.max_pages + 4 * a.pages_per_wave - 1) / (4 * a.pages_per_wave)) < 512)
        a.pages_per_wave /= 2;
    const int64_t groups = (a.max_pages + 4 * a.pages_per_wave - 1) / (4 * a.pages_per_wave);
    if (fast && groups <= 65535) {
        const dim3 grid(units, static_cast<unsigned>(groups));
        if (c.kv_dtype == SFG_F32) {
            if (c.head_dim == 128) page_score_kernel<float, 128><<<grid, 256, 0, stream>>>(a);
            else page_score_kernel<float, 64><<<grid, 256, 0, stream>>>(a);
        } else {
            if (c.head_dim == 128) page_score_kernel<uint16_t, 128><<<grid, 256, 0, stream>>>(a);
            else page_score_kernel<uint16_t, 64><<<grid, 256, 0, stream>>>(a);
        }
    } else {
        const dim3 grid(units, static_cast<unsigned>(std::min<int64_t>((a.max_pages + 15) / 16, 1024)));
        if (c.kv_dtype == SFG_F32) page_score_any_kernel<float><<<grid, 256, 0, stream>>>(a);
        else page_score_any_kernel<uint16_t><<<grid, 256, 0, stream>>>(a);
    }
    by_size(a.max_pages, [&](auto nt, auto k) {
        page_select_kernel<decltype(nt)::value, decltype(k)::value><<<units, decltype(nt)::value, 0, stream>>>(a);
    });
}

void launch_kv_select(const float* weights, int64_t ld, const int32_t* seq_lens, int64_t max_context, int64_t budget,
                      int64_t recent, int32_t* keep, int32_t* kept_lens, float* kept_weights, int64_t batch,
                      int64_t kv_heads, hipStream_t stream) {
    TokenSelectArgs a{};
    a.weights = weights; a.ld = ld; a.seq_lens = seq_lens; a.max_len = static_cast<int>(max_context);
    a.budget = static_cast<int>(budget); a.recent = static_cast<int>(recent);
    a.keep = keep; a.kept_lens = kept_lens; a.kept = kept_weights; a.kv_heads = static_cast<int>(kv_heads);
    by_size(max_context, [&](auto nt, auto k) {
        kv_select_kernel<decltype(nt)::value, decltype(k)::value>
            <<<static_cast<unsigned>(batch * kv_heads), decltype(nt)::value, 0, stream>>>(a);
    });
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
