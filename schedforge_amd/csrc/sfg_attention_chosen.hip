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
#include <cfloat>

#include <algorithm>
#include <type_traits>

#include "sfg_chosen.hpp"

namespace sfg {

namespace {

// A score as the weights' end reads it: -inf is a token that the column does not see, so
// that one it does see whose score is -inf (weight 0, or NaN where all are) is the lowest number.
__device__ __forceinline__ float kept_score(float s, bool seen) { return seen && s == -INFINITY ? -FLT_MAX : s; }

// ===========================================================================
// Any head_dim up to kRowMaxD, any page size, any alignment: one wave per
// (unit column, split).  Lane j scores token j of each 64-token chunk with one
// fp32 FMA chain over the head dimension, then the wave accumulates p V, lane d
// owning dims d, d + 64, ...  Bound by its loads, K and V once per column: head_dim
// 80, 8 x 8 kv heads x up to 4096 tokens, 32 columns 0.74 ms, 4 columns with weights
// 0.205 ms (an element a load 1.53 and 0.38 ms).
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
    // splits begin at multiples of four tokens
    const int k0 = static_cast<int>(static_cast<int64_t>(u.walk) * split / p.splits) & ~3;
    const int k1 = split + 1 == p.splits ? u.walk : static_cast<int>(static_cast<int64_t>(u.walk) * (split + 1) / p.splits) & ~3;
    // K rows as 16-byte vectors, V four tokens of a dim at a time, where they lie so
    constexpr int kVec = 16 / sizeof(KvT);
    const bool k_vec = D % kVec == 0 && (reinterpret_cast<uintptr_t>(p.k_pool) & 15) == 0;
    const bool v_vec = pt % 4 == 0 && (reinterpret_cast<uintptr_t>(p.v_pool) & 15) == 0;

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
                    if (k_vec) {
#pragma unroll 4
                        for (int d = 0; d < D; d += kVec) {
                            KvT v[kVec];
                            const uint4 w = *reinterpret_cast<const uint4*>(kr + d);
                            __builtin_memcpy(v, &w, sizeof v);
#pragma unroll
                            for (int e = 0; e < kVec; ++e) dot = fmaf(sq[d + e], kv_f32(v, e), dot);
                        }
                    } else {
                        for (int d = 0; d < D; ++d) dot = fmaf(sq[d], kv_f32(kr, d), dot);
                    }
                    s = dot * p.scale_log2;
                }
            }
            if constexpr (MODE == kChosenWeights) p.scores[slot * p.scores_ld + j] = kept_score(s, page >= 0);
        }
        const float m_new = fmaxf(m, wave_max(s));
        const float pr = page < 0 ? 0.f : m_new == -INFINITY ? (s == -INFINITY ? 0.f : s) : fast_exp2(s - m_new);
        const float alpha = m == -INFINITY ? 0.f : fast_exp2(m - m_new);
        l = l * alpha + wave_sum(pr);
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[r] *= alpha;
        const int count = min(64, k1 - base);
        if (v_vec) {
            for (int t = 0; t < count; t += 4) {  // tokens of one page
                int seen[4], pg = -1;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    seen[e] = lane_bcast(page, t + e);  // (lanes past the chunk hold -1)
                    pg = max(pg, seen[e]);
                }
                if (pg < 0) continue;  // wave-uniform
                const KvT* vb = vpool + (static_cast<int64_t>(pg) * p.kv_heads + u.kvh) * D * pt + lane_bcast(at, t);
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int d = lane + 64 * r;
                    if (d >= D) continue;
                    KvT v[4];
                    __builtin_memcpy(v, __builtin_assume_aligned(vb + static_cast<int64_t>(d) * pt, 4 * sizeof(KvT)), sizeof v);
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (seen[e] >= 0) acc[r] = fmaf(lane_bcast(pr, t + e), kv_f32(v, e), acc[r]);
                }
            }
            m = m_new;
            continue;
        }
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
// head_dim 64 / 128 and 16-token pages on the matrix cores.  A workgroup owns 16
// columns of a unit and one split; its four (or eight) waves take an equal part of the
// pages each, with the next page's K and V loads behind the current page's products:
//   S^T[16 tok][16 col] = K[16 tok][D] Q^T[D][16 col]
//   O^T[D][16 col]     += V^T[D][16 tok] P^T[16 tok][16 col]
// The S^T accumulator (lane: column l & 15, tokens 4 (l >> 4) + r) is the P^T
// operand's layout, so the running maximum needs two cross-lane steps a page and the
// rescale is one factor per lane.  Bound by HBM where a unit has at most 16 columns:
// with weights, 32 x 4 kv heads x up to 8192 tokens (281 MB) 50 us from a warm cache, 62
// from HBM (a copy's rate would be 57); 64 pages of 16 x 8 heads (67 MB) 16 us.  Two
// pages in flight instead of one were no faster (53 and 17 us).
//
// FAST (bf16 queries and output over bf16 pools): Q is exact in one bf16 operand; P
// keeps 16 bits in two terms, so that what reaches the result is its own rounding (one
// rounded term made as large an error of its own, and was no faster: the loads bound
// the walk).  Otherwise Q and P keep 24 bits: three bf16 terms over bf16 pools, fp32
// matrix instructions over fp32 pools.
//
// What a column does not see reaches it neither as a score (replaced by -inf) nor as
// 0 * inf: V past the unit's end is zeroed, and a page with a hidden non-finite value
// is taken token by token.  With three terms a visible infinity would meet terms of
// zero, so a wave whose sums are not finite walks its pages once more: keys'
// non-finite elements meet the leading term only, values go token by token.
//
// Two waves a SIMD (at most 256 registers) for every variant: over fp32 pools of head_dim
// 128 the compiler would take more and leave one (8 x 8 kv heads x up to 4096 tokens, 128
// columns: 213 us so, 185 with two).
// ===========================================================================
template <typename KvT, int kD, int MODE, bool FAST, int WAVES>
__global__ __launch_bounds__(WAVES * 64, 2) void chosen_mfma_kernel(ChosenArgs p, int chunks, int xcds) {
    constexpr bool kF32 = sizeof(KvT) == 4;
    static_assert(!(FAST && kF32), "fp32 pools keep fp32 precision");
    constexpr int kTerms = FAST ? 1 : 3;
    constexpr int kStep = kF32 ? 16 : 32, kKs = kD / kStep, kDt = kD / 16;
    constexpr int kLane = kStep / 4;  // dims of a k-step per lane
    using VecV = std::conditional_t<kF32, uint4, uint2>;  // four tokens of V
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int lr = lane & 15, lg = lane >> 4;
    // consecutive workgroup ids go to the XCDs in turn: the chunks of a (unit, split) lie one
    // round of XCDs apart, so that they read its K and V through one L2 at about one time
    // (16 x 8 kv heads x 900 tokens, 32 columns: 22.8 us in plain order, 17.3 so)
    const int bid = static_cast<int>(blockIdx.x), pairs = static_cast<int>(gridDim.x) / chunks;
    const int full = pairs - pairs % xcds;
    const int in = bid < full * chunks ? bid % (xcds * chunks) : bid - full * chunks;
    const int lanes = bid < full * chunks ? xcds : pairs - full;  // (unit, split)s side by side
    const int chunk = in / lanes;
    const int pair = (bid < full * chunks ? bid / (xcds * chunks) * xcds : full) + in % lanes;
    const int split = pair % p.splits, uid = pair / p.splits;
    const int per_b = MODE == kChosenSparse ? p.rows * p.kv_heads : p.kv_heads;
    const Unit<MODE> u = unit_of<MODE>(p, uid / per_b, uid % per_b);
    const int col0 = 16 * chunk;
    const int pages = (u.walk + kPageTok - 1) / kPageTok;
    const int sp_begin = static_cast<int>(static_cast<int64_t>(pages) * split / p.splits);
    const int sp_end = static_cast<int>(static_cast<int64_t>(pages) * (split + 1) / p.splits);
    const int n_sp = sp_end - sp_begin;
    const int w_begin = sp_begin + n_sp * wave / WAVES;
    const int w_end = sp_begin + n_sp * (wave + 1) / WAVES;

    // Q^T operand: this lane's column, dims kStep s + kLane lg + [0, kLane)
    const bool has = col0 + lr < u.cols;
    int row, head;
    column_of<MODE>(p, u, has ? col0 + lr : col0, row, head);
    bf16x8 qf[kF32 ? 1 : kKs][kTerms];
    float4 qf32[kF32 ? kKs : 1];
    {
        const int64_t qo = column_offset(p, u.b, row, head) + kLane * lg;
#pragma unroll
        for (int s = 0; s < kKs; ++s) {
            if constexpr (FAST) {
                const uint4 w = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.q) + qo + kStep * s);
                qf[s][0] = as_bf16x8(has ? w : make_uint4(0, 0, 0, 0));
            } else {
                float v[kLane];
                if (p.q_f32) {
#pragma unroll
                    for (int e = 0; e < kLane; e += 4)
                        *reinterpret_cast<float4*>(v + e) = *reinterpret_cast<const float4*>(static_cast<const float*>(p.q) + qo + kStep * s + e);
                } else {
#pragma unroll
                    for (int e = 0; e < kLane; ++e) v[e] = bf16_to_f32(static_cast<const uint16_t*>(p.q)[qo + kStep * s + e]);
                }
#pragma unroll
                for (int e = 0; e < kLane; ++e) v[e] = has ? v[e] : 0.f;
                if constexpr (kF32) {
                    qf32[s] = make_float4(v[0], v[1], v[2], v[3]);
                } else {
                    uint32_t w[3][4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        uint16_t a[3], c[3];
                        split3(v[2 * e], a[0], a[1], a[2]);
                        split3(v[2 * e + 1], c[0], c[1], c[2]);
#pragma unroll
                        for (int t = 0; t < 3; ++t) w[t][e] = static_cast<uint32_t>(a[t]) | (static_cast<uint32_t>(c[t]) << 16);
                    }
#pragma unroll
                    for (int t = 0; t < kTerms; ++t) qf[s][t] = as_bf16x8(make_uint4(w[t][0], w[t][1], w[t][2], w[t][3]));
                }
            }
        }
    }

    floatx4 acc[kDt];
    float m_run, l_run;
    const int32_t* table = p.page_table + static_cast<int64_t>(u.b) * p.pages_per_seq;
    const int64_t head_stride = static_cast<int64_t>(kPageTok) * kD;
    const int64_t page_stride = head_stride * p.kv_heads;
    const KvT* kpool = static_cast<const KvT*>(p.k_pool) + u.kvh * head_stride + lr * kD + kLane * lg;
    const KvT* vpool = static_cast<const KvT*>(p.v_pool) + u.kvh * head_stride + lr * kPageTok + 4 * lg;
    float* scores = MODE == kChosenWeights ? p.scores + (u.id * u.cols + col0 + lr) * p.scores_ld : nullptr;
    uint4 kb[kKs];
    VecV vb[kDt];
    bool okb = false;
    int lpb = 0;
    // logical pages and their ids 64 at a time, one per lane, so that a page's loads
    // wait on no read of their own; an id outside the pool reads page 0 and shows no key
    int ids = 0, lps = 0, ids_base = 0;
    auto load_page = [&](int at) __attribute__((always_inline)) {
        if (at - ids_base >= 64) {  // wave-uniform
            ids_base = at;
            int lp = at + lane;
            if constexpr (MODE == kChosenSparse) lp = lp < w_end ? u.list[lp] : -1;
            lps = lp;
            ids = at + lane < w_end && lp >= 0 && lp < p.pages_per_seq ? table[lp] : -1;
        }
        const int id = __builtin_amdgcn_readlane(ids, at - ids_base);
        lpb = MODE == kChosenSparse ? __builtin_amdgcn_readlane(lps, at - ids_base) : at;
        okb = id >= 0 && id < p.num_pages;
        const int64_t base = okb ? static_cast<int64_t>(id) * page_stride : 0;
#pragma unroll
        for (int s = 0; s < kKs; ++s) kb[s] = *reinterpret_cast<const uint4*>(kpool + base + kStep * s);
#pragma unroll
        for (int dt = 0; dt < kDt; ++dt) vb[dt] = *reinterpret_cast<const VecV*>(vpool + base + dt * 16 * kPageTok);
    };
    auto walk_pages = [&](auto second_c) __attribute__((always_inline)) {
        constexpr bool kSecond = decltype(second_c)::value;
        m_run = -INFINITY;
        l_run = 0.f;
#pragma unroll
        for (int i = 0; i < kDt; ++i) acc[i] = floatx4{0.f, 0.f, 0.f, 0.f};
        ids_base = w_begin - 64;
        if (w_begin < w_end) load_page(w_begin);
        for (int at = w_begin; at < w_end; ++at) {
            uint4 kc[kKs];
            VecV vc[kDt];
#pragma unroll
            for (int s = 0; s < kKs; ++s) kc[s] = kb[s];
#pragma unroll
            for (int dt = 0; dt < kDt; ++dt) vc[dt] = vb[dt];
            const bool ok = okb;
            const int lp = lpb;
            if (at + 1 < w_end) load_page(at + 1);
            const int tok0 = lp * kPageTok + 4 * lg;  // this lane's four tokens
            const bool whole = ok && (lp + 1) * kPageTok <= u.all_see;  // wave-uniform: every column sees every token
            uint32_t vis = 15;  // bit r: the lane's column sees token tok0 + r
            bool slow = false;
            if (!whole || kSecond) {
                if (!whole) {
                    vis = 0;
                    if (ok && has)
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            if (tok0 + r < u.total && sees<MODE>(p, u, row, tok0 + r)) vis |= 1u << r;
                }
                // tokens past the end (or of no page) are not data
                bool bad = false;
#pragma unroll
                for (int dt = 0; dt < kDt; ++dt) {
                    if constexpr (kF32) {
                        uint32_t w[4] = {vc[dt].x, vc[dt].y, vc[dt].z, vc[dt].w};
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            if (!ok || tok0 + e >= u.total) w[e] = 0u;
                            bad |= (w[e] & 0x7F800000u) == 0x7F800000u;
                        }
                        vc[dt] = make_uint4(w[0], w[1], w[2], w[3]);
                    } else {
                        uint32_t w[2] = {vc[dt].x, vc[dt].y};
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const uint32_t mask = 0xFFFFu << (16 * (e & 1));
                            if (!ok || tok0 + e >= u.total) w[e >> 1] &= ~mask;
                            const uint32_t expo = (w[e >> 1] >> (16 * (e & 1))) & 0x7F80u;
                            bad |= expo == 0x7F80u;
                        }
                        vc[dt] = make_uint2(w[0], w[1]);
                    }
                }
                slow = __any(bad);
            }
            floatx4 st;
            if constexpr (kF32) {
                // two chains; a lane's four dims feed four MFMAs
                floatx4 s2[2] = {floatx4{0.f, 0.f, 0.f, 0.f}, floatx4{0.f, 0.f, 0.f, 0.f}};
#pragma unroll
                for (int s = 0; s < kKs; ++s) {
                    const float4 kf = __builtin_bit_cast(float4, kc[s]), qq = qf32[s];
                    s2[0] = __builtin_amdgcn_mfma_f32_16x16x4f32(kf.x, qq.x, s2[0], 0, 0, 0);
                    s2[1] = __builtin_amdgcn_mfma_f32_16x16x4f32(kf.y, qq.y, s2[1], 0, 0, 0);
                    s2[0] = __builtin_amdgcn_mfma_f32_16x16x4f32(kf.z, qq.z, s2[0], 0, 0, 0);
                    s2[1] = __builtin_amdgcn_mfma_f32_16x16x4f32(kf.w, qq.w, s2[1], 0, 0, 0);
                }
                st = s2[0] + s2[1];
            } else {
                // a chain per term, the small terms summed first
                floatx4 sk[kTerms];
#pragma unroll
                for (int t = 0; t < kTerms; ++t) sk[t] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int s = 0; s < kKs; ++s)
#pragma unroll
                    for (int t = 0; t < kTerms; ++t) {
                        uint4 k = kc[s];
                        if (kSecond && t > 0)
                            k = make_uint4(finite_bf16x2(k.x), finite_bf16x2(k.y), finite_bf16x2(k.z), finite_bf16x2(k.w));
                        sk[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf16x8(k), qf[s][t], sk[t], 0, 0, 0);
                    }
                if constexpr (FAST) st = sk[0];
                else st = sk[0] + (sk[1] + sk[2]);
            }
            float sv[4];
            float mx = -INFINITY;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                sv[r] = (vis >> r) & 1u ? st[r] * p.scale_log2 : -INFINITY;
                mx = fmaxf(mx, sv[r]);
            }
            if constexpr (MODE == kChosenWeights)
                if (has)
                    *reinterpret_cast<float4*>(scores + tok0) =
                        make_float4(kept_score(sv[0], vis & 1u), kept_score(sv[1], vis & 2u), kept_score(sv[2], vis & 4u), kept_score(sv[3], vis & 8u));
            mx = xor16_max(mx);
            mx = xor32_max(mx);
            const float m_new = fmaxf(m_run, mx);
            const float alpha = m_run == -INFINITY ? 0.f : fast_exp2(m_run - m_new);
            float pv[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) pv[r] = sv[r] == -INFINITY ? 0.f : fast_exp2(sv[r] - m_new);
            l_run = l_run * alpha + ((pv[0] + pv[1]) + (pv[2] + pv[3]));
            m_run = m_new;
#pragma unroll
            for (int dt = 0; dt < kDt; ++dt) acc[dt] *= alpha;
            if (!slow) {
                if constexpr (kF32) {
#pragma unroll
                    for (int t = 0; t < 4; ++t)
#pragma unroll
                        for (int dt = 0; dt < kDt; ++dt) {
                            const float4 vf = __builtin_bit_cast(float4, vc[dt]);
                            const float vt = t == 0 ? vf.x : t == 1 ? vf.y : t == 2 ? vf.z : vf.w;
                            acc[dt] = __builtin_amdgcn_mfma_f32_16x16x4f32(vt, pv[t], acc[dt], 0, 0, 0);
                        }
                } else if constexpr (FAST) {
                    uint2 hi, lo;
                    split2_weights(pv[0], pv[1], hi.x, lo.x);
                    split2_weights(pv[2], pv[3], hi.y, lo.y);
#pragma unroll
                    for (int dt = 0; dt < kDt; ++dt)
                        acc[dt] = __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(as_short4(vc[dt]), as_short4(lo), acc[dt], 0, 0, 0);
#pragma unroll
                    for (int dt = 0; dt < kDt; ++dt)
                        acc[dt] = __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(as_short4(vc[dt]), as_short4(hi), acc[dt], 0, 0, 0);
                } else {
                    uint16_t w[3][4];
#pragma unroll
                    for (int r = 0; r < 4; ++r) split3(pv[r], w[0][r], w[1][r], w[2][r]);
#pragma unroll
                    for (int t = 2; t >= 0; --t) {
                        const short4v pb = as_short4(make_uint2(static_cast<uint32_t>(w[t][0]) | (static_cast<uint32_t>(w[t][1]) << 16),
                                                                static_cast<uint32_t>(w[t][2]) | (static_cast<uint32_t>(w[t][3]) << 16)));
#pragma unroll
                        for (int dt = 0; dt < kDt; ++dt)
                            acc[dt] = __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(as_short4(vc[dt]), pb, acc[dt], 0, 0, 0);
                    }
                }
            } else {
                // token by token: lane (lr, t / 4) holds its probability and whether the
                // column sees it, lane (4 lg + r, t / 4) V of this lane's dims
#pragma unroll 1
                for (int t = 0; t < kPageTok; ++t) {
                    const float mine = (t & 3) == 0 ? pv[0] : (t & 3) == 1 ? pv[1] : (t & 3) == 2 ? pv[2] : pv[3];
                    const float pt = __shfl(mine, 16 * (t >> 2) + lr, 64);
                    const bool seen = (__shfl(static_cast<int>(vis), 16 * (t >> 2) + lr, 64) >> (t & 3)) & 1;
#pragma unroll
                    for (int dt = 0; dt < kDt; ++dt) {
                        // (masked, not selected: a select between the words is turned into
                        // a load from scratch memory, which would hold V for every page)
                        const uint32_t hi = 0u - static_cast<uint32_t>((t >> 1) & 1);
                        uint32_t word;
                        if constexpr (kF32) {
                            const uint32_t odd = 0u - static_cast<uint32_t>(t & 1);
                            const uint32_t lo2 = vc[dt].x ^ ((vc[dt].x ^ vc[dt].y) & odd), hi2 = vc[dt].z ^ ((vc[dt].z ^ vc[dt].w) & odd);
                            word = lo2 ^ ((lo2 ^ hi2) & hi);
                        } else {
                            word = vc[dt].x ^ ((vc[dt].x ^ vc[dt].y) & hi);
                        }
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            const uint32_t w = __shfl(static_cast<int>(word), 16 * (t >> 2) + 4 * lg + r, 64);
                            const float v = kF32 ? __uint_as_float(w) : bf16_to_f32(static_cast<uint16_t>(w >> (16 * (t & 1))));
                            if (seen) acc[dt][r] = fmaf(pt, v, acc[dt][r]);
                        }
                    }
                }
            }
        }
    };
    walk_pages(std::false_type{});
    if constexpr (!kF32 && !FAST) {
        float t = l_run * 0.f;  // NaN unless every sum is finite
#pragma unroll
        for (int dt = 0; dt < kDt; ++dt)
#pragma unroll
            for (int r = 0; r < 4; ++r) t = fmaf(acc[dt][r], 0.f, t);
        if (__any(has && t != 0.f)) walk_pages(std::true_type{});
    }
    // the waves merged in LDS: acc[dt][r] = O^T[dim 16 dt + 4 lg + r][column lr]
    __shared__ float s_m[WAVES][16], s_l[WAVES][16];
    __shared__ float s_acc[WAVES][16][kD];
    const float l_sum = xor32_sum(xor16_sum(l_run));
#pragma unroll
    for (int dt = 0; dt < kDt; ++dt) *reinterpret_cast<floatx4*>(&s_acc[wave][lr][16 * dt + 4 * lg]) = acc[dt];
    if (lg == 0) {
        s_m[wave][lr] = m_run;
        s_l[wave][lr] = l_sum;
    }
    __syncthreads();
    for (int o = threadIdx.x; o < min(16, u.cols - col0) * kD; o += WAVES * 64) {
        const int c = o / kD, d = o % kD;
        float M = -INFINITY;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) M = fmaxf(M, s_m[w][c]);
        float L = 0.f, a = 0.f;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) {
            const float f = split_weight(s_m[w][c], M);
            L = fmaf(s_l[w][c], f, L);
            a = fmaf(s_acc[w][c][d], f, a);
        }
        if (MODE != kChosenWeights && p.splits == 1) {
            int ro, he;
            column_of<MODE>(p, u, col0 + c, ro, he);
            const int64_t o0 = column_offset(p, u.b, ro, he) + d;
            const float v = a / L;  // nothing visible: 0 / 0
            if (p.out_f32) static_cast<float*>(p.out)[o0] = v;
            else static_cast<uint16_t*>(p.out)[o0] = f32_to_bf16(v);
        } else {
            const int64_t part = (u.id * u.cols + col0 + c) * p.splits + split;
            p.part_acc[part * kD + d] = a;
            if (d == 0) {
                p.part_ml[2 * part] = M;
                p.part_ml[2 * part + 1] = L;
            }
        }
    }
}

// ===========================================================================
// The splits of a column merged: weights 2^(m_s - M), output sum / L.
// ===========================================================================
// One wave a column.  kV: dims a lane holds side by side (head_dim 64 kV), 0: any head_dim.
template <int MODE, int kV>
__device__ __forceinline__ void merge_dims(const ChosenArgs& p, const Unit<MODE>& u, int col, int lane) {
    constexpr int kW = kV ? kV : 1;
    const int64_t slot = u.id * u.cols + col;
    const float2* ml = reinterpret_cast<const float2*>(p.part_ml) + slot * p.splits;
    const float* pa = p.part_acc + slot * p.splits * p.head_dim;
    int row, head;
    column_of<MODE>(p, u, col, row, head);
    const int64_t o0 = column_offset(p, u.b, row, head);
    // eight splits at a time, their loads all issued before the ordered sum (slots past
    // the count re-read the last split and are left out)
    constexpr int kBatch = 8;
    for (int d = lane * kW; d < p.head_dim; d += 64 * kW) {
        float M = -INFINITY, L = 0.f, o[kW];
#pragma unroll
        for (int i = 0; i < kW; ++i) o[i] = 0.f;
        for (int s0 = 0; s0 < p.splits; s0 += kBatch) {
            float2 x[kBatch];
            float av[kBatch][kW];
#pragma unroll
            for (int e = 0; e < kBatch; ++e) {
                const int64_t sc = min(s0 + e, p.splits - 1);
                x[e] = ml[sc];
                const float* at = pa + sc * p.head_dim + d;
                if constexpr (kV == 2) {
                    const float2 v = *reinterpret_cast<const float2*>(at);
                    av[e][0] = v.x;
                    av[e][kW - 1] = v.y;
                } else {
                    av[e][0] = *at;
                }
            }
            float m = M;
#pragma unroll
            for (int e = 0; e < kBatch; ++e) m = fmaxf(m, x[e].x);
            const float f = split_weight(M, m);
            L *= f;
#pragma unroll
            for (int i = 0; i < kW; ++i) o[i] *= f;
#pragma unroll
            for (int e = 0; e < kBatch; ++e) {
                if (s0 + e >= p.splits) continue;
                const float w = split_weight(x[e].x, m);
                L = fmaf(x[e].y, w, L);
#pragma unroll
                for (int i = 0; i < kW; ++i) o[i] = fmaf(w, av[e][i], o[i]);
            }
            M = m;
        }
#pragma unroll
        for (int i = 0; i < kW; ++i) {
            const float v = o[i] / L;  // nothing visible: 0 / 0
            if (p.out_f32) static_cast<float*>(p.out)[o0 + d + i] = v;
            else static_cast<uint16_t*>(p.out)[o0 + d + i] = f32_to_bf16(v);
        }
    }
}

template <int MODE>
__device__ __forceinline__ void merge_column(const ChosenArgs& p, const Unit<MODE>& u, int col, int lane) {
    if (p.head_dim == 128) merge_dims<MODE, 2>(p, u, col, lane);
    else merge_dims<MODE, 0>(p, u, col, lane);
}

// Four columns a workgroup, one a wave.  3.9 us for 256 columns of 8 splits, most of it
// the launch and two dependent loads.
template <int MODE>
__global__ __launch_bounds__(256) void chosen_combine_kernel(ChosenArgs p, int columns) {
    const int slot = blockIdx.x * 4 + (threadIdx.x >> 6);
    if (slot >= columns) return;
    int col;
    const Unit<MODE> u = unit_of_slot<MODE>(p, slot, col);
    merge_column<MODE>(p, u, col, threadIdx.x & 63);
}

// The weights' end, one wave per 256 tokens of a (sequence, kv head): four columns at a
// time, their scores and (m, l) loaded together, lane s merging split s (and s + 64, ...);
// the wave adds sum_columns 2^(s - M) / L to its tokens' accumulators.  The workgroups past
// the tokens merge the output columns.  A column that sees nothing adds nothing.  Latency,
// not bytes (4 G of scores and 8 of accumulator a token), bounds it: 7.0 us for 32 x 4
// heads x up to 8192 tokens, 5.8 for 8 heads x 4096.
__global__ __launch_bounds__(64) void chosen_weights_kernel(ChosenArgs p, float* weights, int64_t ld, int chunks) {
    constexpr int kTok = 4, kCols = 4;  // tokens a lane, columns at a time
    const Unit<kChosenWeights> u = unit_of<kChosenWeights>(p, blockIdx.x / p.kv_heads, blockIdx.x % p.kv_heads);
    const int lane = threadIdx.x, tok0 = blockIdx.y * 256 + lane;
    if (static_cast<int>(blockIdx.y) >= chunks) {
        for (int c = blockIdx.y - chunks; c < u.cols; c += gridDim.y - chunks) merge_column<kChosenWeights>(p, u, c, lane);
        return;
    }
    if (static_cast<int>(blockIdx.y) * 256 >= u.total) return;
    const float* scores = p.scores + u.id * u.cols * p.scores_ld;
    const float2* ml = reinterpret_cast<const float2*>(p.part_ml) + u.id * u.cols * p.splits;
    int at[kTok];
    float sum[kTok], was[kTok];
#pragma unroll
    for (int t = 0; t < kTok; ++t) {
        at[t] = min(tok0 + 64 * t, u.total - 1);
        sum[t] = 0.f;
        was[t] = weights[u.id * ld + at[t]];
    }
    for (int c0 = 0; c0 < u.cols; c0 += kCols) {
        float2 x[kCols];
        float s[kCols][kTok];
#pragma unroll
        for (int c = 0; c < kCols; ++c) {
            const int64_t col = min(c0 + c, u.cols - 1);
            x[c] = ml[col * p.splits + min(lane, p.splits - 1)];
            if (lane >= p.splits) x[c] = make_float2(-INFINITY, 0.f);
#pragma unroll
            for (int t = 0; t < kTok; ++t) s[c][t] = scores[col * p.scores_ld + at[t]];
        }
#pragma unroll
        for (int c = 0; c < kCols; ++c) {
            if (c0 + c >= u.cols) continue;
            for (int i = lane + 64; i < p.splits; i += 64) {
                const float2 y = ml[static_cast<int64_t>(c0 + c) * p.splits + i];
                const float m = fmaxf(x[c].x, y.x);
                x[c] = make_float2(m, x[c].y * split_weight(x[c].x, m) + y.y * split_weight(y.x, m));
            }
            const float M = wave_max(x[c].x), L = wave_sum(x[c].y * split_weight(x[c].x, M));
            const float R = L == 0.f ? NAN : 1.f / L;  // (0: every score it sees is -inf)
#pragma unroll
            for (int t = 0; t < kTok; ++t)
                if (s[c][t] != -INFINITY) sum[t] = fmaf(fast_exp2(s[c][t] - M), R, sum[t]);
        }
    }
#pragma unroll
    for (int t = 0; t < kTok; ++t)
        if (tok0 + 64 * t < u.total) weights[u.id * ld + at[t]] = was[t] + sum[t];
}

constexpr int64_t kMaxGroups = 1 << 23;  // workgroups of 256 threads in a launch

size_t up256(size_t v) { return (v + 255) / 256 * 256; }

template <int MODE, int kD, int WAVES>
void launch_mfma(const ChosenLaunch& a, const ChosenArgs& p, unsigned grid, int chunks, hipStream_t stream) {
    const int xcds = device_xcds(stream);
    if (a.kv_dtype == SFG_F32) chosen_mfma_kernel<float, kD, MODE, false, WAVES><<<grid, WAVES * 64, 0, stream>>>(p, chunks, xcds);
    else if (a.q_dtype == SFG_BF16 && a.out_dtype == SFG_BF16)
        chosen_mfma_kernel<uint16_t, kD, MODE, true, WAVES><<<grid, WAVES * 64, 0, stream>>>(p, chunks, xcds);
    else chosen_mfma_kernel<uint16_t, kD, MODE, false, WAVES><<<grid, WAVES * 64, 0, stream>>>(p, chunks, xcds);
}

template <int MODE>
void launch_mode(const ChosenLaunch& a, const ChosenArgs& p, const ChosenPlan& plan, void* workspace, hipStream_t stream) {
    const unsigned columns = static_cast<unsigned>(a.batch * a.rows * a.q_heads);
    const int64_t units = a.batch * a.kv_heads * (MODE == kChosenSparse ? a.rows : 1);
    const int64_t chunks = (columns / units + 15) / 16;
    // Q, K and V are read as 16-byte vectors; rows of 64 or 128 elements keep a base's boundary
    const bool aligned = ((reinterpret_cast<uintptr_t>(a.q) | reinterpret_cast<uintptr_t>(a.k_pool) | reinterpret_cast<uintptr_t>(a.v_pool)) & 15) == 0;
    if (plan.tiles && aligned && (reinterpret_cast<uintptr_t>(a.out) & 7) == 0) {
        launch_tree_tiles(p, plan_tree_tiles(a.batch, a.kv_heads, columns / units, a.head_dim, a.max_context + a.rows, a.kv_splits),
                          a.batch, workspace, stream);
        return;
    }
    if (plan.mfma && aligned && units * chunks * plan.splits <= kMaxGroups) {
        const unsigned grid = static_cast<unsigned>(units * chunks * plan.splits);
        const int n = static_cast<int>(chunks);
        if constexpr (MODE == kChosenWeights) {
            if (a.head_dim == 128) launch_mfma<MODE, 128, 4>(a, p, grid, n, stream);
            else launch_mfma<MODE, 64, 4>(a, p, grid, n, stream);
        } else if (plan.waves == 8) {
            if (a.head_dim == 128) launch_mfma<MODE, 128, 8>(a, p, grid, n, stream);
            else launch_mfma<MODE, 64, 8>(a, p, grid, n, stream);
        } else {
            if (a.head_dim == 128) launch_mfma<MODE, 128, 4>(a, p, grid, n, stream);
            else launch_mfma<MODE, 64, 4>(a, p, grid, n, stream);
        }
    } else {
        const dim3 grid(columns, static_cast<unsigned>(plan.splits));
        if (a.kv_dtype == SFG_F32) chosen_any_kernel<float, MODE><<<grid, 64, 0, stream>>>(p);
        else chosen_any_kernel<uint16_t, MODE><<<grid, 64, 0, stream>>>(p);
    }
    if constexpr (MODE == kChosenWeights) {
        const int tokens = static_cast<int>((a.max_context + 255) / 256);
        const unsigned merges = static_cast<unsigned>(std::min<int64_t>(columns / units, 64));
        chosen_weights_kernel<<<dim3(static_cast<unsigned>(units), tokens + merges), 64, 0, stream>>>(p, a.weights, a.weights_ld, tokens);
    }
    else if (plan.splits > 1) chosen_combine_kernel<MODE><<<(columns + 3) / 4, 256, 0, stream>>>(p, static_cast<int>(columns));
}

}  // namespace

ChosenPlan plan_chosen(int mode, bool bf16, bool ragged, int64_t batch, int64_t q_heads, int64_t kv_heads, int64_t rows, int64_t head_dim,
                       int64_t page_tokens, int64_t keys, int32_t requested) {
    ChosenPlan plan{};
    const int64_t columns = batch * rows * q_heads;
    plan.mfma = (head_dim == 64 || head_dim == 128) && page_tokens == kPageTok;
    const int64_t units = batch * kv_heads * (mode == kChosenSparse ? rows : 1);
    const int64_t cols = columns / units;
    const int64_t base = plan.mfma ? units * ((cols + 15) / 16) : columns;
    const int64_t most = plan.mfma ? (keys + kPageTok - 1) / kPageTok : keys;
    int64_t s = 1;
    plan.waves = 4;
    if (requested > 0) {
        s = std::min<int64_t>(requested, std::max<int64_t>(most, 1));
    } else if (!plan.mfma) {
        // >= 1024 waves while a split keeps >= 256 tokens
        while (base * s < 1024 && most / (s * 2) >= 256) s *= 2;
    } else if (mode != kChosenWeights && most <= 64 && base >= 128) {
        // half of the CUs busy and up to eight pages a wave: no splits to merge, one launch
        // less.  Whole sparse calls so and with splits, us: 128 units of 16 pages 16.4 and 18.7,
        // of 64 26.8 and 29.6, of 128 38.8 and 40.3, of 192 52.3 and 52.1; 96 units of 64 27.0 and
        // 27.9, 64 units 26.1 and 23.8, 32 units 24.0 and 18.3; 256 units 37.0 and 41.1, 512
        // units 67.0 and 63.6
        plan.waves = 8;
    } else {
        // two workgroups per CU while a split keeps 8 pages, two per wave (tree: 4; 1 x 8 kv
        // heads x 900 tokens 12.3 us at 4 splits, 11.2 at 8); sequences with lengths of their
        // own leave their last splits short or empty, so up to eight per CU while a split
        // keeps 32 (32 x 4 kv heads x up to 8192 tokens: 65 us at 4 splits, 58 at 16)
        while (base * s < 512 && most / (s * 2) >= (mode == kChosenTree ? 4 : 8)) s *= 2;
        while (ragged && mode != kChosenSparse && base * s < 2048 && most / (s * 2) >= 32) s *= 2;
    }
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
    if (mode == kChosenTree && plan.mfma && bf16) {
        const TreeTiles t = plan_tree_tiles(batch, kv_heads, cols, head_dim, keys, requested);
        plan.tiles = t.groups > 0;
        plan.tile_bytes = t.bytes();
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
    if (a.mode == kChosenTree) launch_mode<kChosenTree>(a, p, plan, workspace, stream);
    else if (a.mode == kChosenWeights) launch_mode<kChosenWeights>(a, p, plan, workspace, stream);
    else launch_mode<kChosenSparse>(a, p, plan, workspace, stream);
}

}  // namespace sfg
