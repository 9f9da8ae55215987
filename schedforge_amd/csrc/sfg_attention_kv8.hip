// sfg_attention_kv8.hip -- causal attention of each sequence's newest rows over a paged
// cache held in 8 bits (codes with a scale for each page, kv head and pool).
#include <math.h>

#include <algorithm>

#include "sfg_kernels.hpp"
#include "sfg_kv8.hpp"

namespace sfg {
namespace {

struct Kv8Args {
    const void* q; int64_t q_stride; int q_f32;
    void* out; int64_t out_stride; int out_f32;
    const uint8_t* k_pool; const uint8_t* v_pool; const float* scales;
    const int32_t* page_table; const int32_t* seq_lens; const int32_t* starts;
    int batch, tokens, max_rows, q_heads, kv_heads, dim, pt, per, pages, max_context;
    float scale;
    // the matrix-core kernels'
    int group, slots, share, fixed, least, direct, width;  // (as in Kv8Plan)
    int vec, out_vec;                                      // rows begin on 16-byte boundaries
    int2* slot_of; int* sequence_of; float2* part_ml; float* part_acc;
    // Rows [t0, t0 + rows) of a sequence and its tokens.
    __device__ __forceinline__ void sequence(int b, int& t0, int& rows, int& len) const {
        t0 = b * max_rows;
        int t1 = t0 + max_rows;
        if (starts) {
            t0 = min(max(starts[b], 0), tokens);
            t1 = min(max(starts[b + 1], t0), tokens);
        }
        rows = t1 - t0;
        len = seq_lens ? min(max(seq_lens[b], 0), max_context) : max_context;
    }
};

__device__ __forceinline__ float kv8_load(const void* p, int f32, int64_t i) {
    return f32 ? static_cast<const float*>(p)[i] : bf16_to_f32(static_cast<const uint16_t*>(p)[i]);
}
__device__ __forceinline__ void kv8_store(void* p, int f32, int64_t i, float v) {
    if (f32) static_cast<float*>(p)[i] = v;
    else static_cast<uint16_t*>(p)[i] = static_cast<uint16_t>(cvt_pk_bf16(v, v));  // (a NaN stays one)
}
// Four values of a row over their sum of weights (nothing seen: 0 / 0).
__device__ __forceinline__ void kv8_store4(const Kv8Args& a, int64_t i, const float4& v, float sum) {
    const float4 y = make_float4(v.x / sum, v.y / sum, v.z / sum, v.w / sum);
    if (!a.out_vec) {
        kv8_store(a.out, a.out_f32, i, y.x);
        kv8_store(a.out, a.out_f32, i + 1, y.y);
        kv8_store(a.out, a.out_f32, i + 2, y.z);
        kv8_store(a.out, a.out_f32, i + 3, y.w);
    } else if (a.out_f32) {
        *reinterpret_cast<float4*>(static_cast<float*>(a.out) + i) = y;
    } else {
        *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.out) + i) = make_uint2(cvt_pk_bf16(y.x, y.y), cvt_pk_bf16(y.z, y.w));
    }
}

}  // namespace

// Any head dim up to kRowMaxD and any page size: a wave a row and query head, 64 tokens at a
// time with a token a lane for the scores and a dim a lane for the values.
template <bool FP8>
__global__ __launch_bounds__(64) void attn_kv8_rows_kernel(Kv8Args a) {
    __shared__ float sq[kRowMaxD];
    const int lane = threadIdx.x, t = blockIdx.x, h = blockIdx.y;
    int b = t / a.max_rows;
    if (a.starts) {
        int hi = a.batch;
        b = 0;
        while (hi - b > 1) {
            const int mid = (b + hi) >> 1;
            if (a.starts[mid] <= t) b = mid;
            else hi = mid;
        }
    }
    int t0, rows, len;
    a.sequence(b, t0, rows, len);
    const int i = t - t0;
    if (i < 0 || i >= rows || i >= a.max_rows) return;
    const int D = a.dim, kvh = h / (a.q_heads / a.kv_heads);
    const int end = min(max(len - rows + i + 1, 0), len);
    for (int d = lane; d < D; d += 64) sq[d] = kv8_load(a.q, a.q_f32, t * a.q_stride + static_cast<int64_t>(h) * D + d);
    __syncthreads();
    const int32_t* table = a.page_table + static_cast<int64_t>(b) * a.per;
    float m = -INFINITY, l = 0.f;
    float acc[kRowMaxD / 64] = {};
    for (int base = 0; base < end; base += 64) {
        const int j = base + lane;
        float s = -INFINITY, sv = 0.f;
        int page = -1;
        if (j < end) {
            const int id = table[j / a.pt];
            if (id >= 0 && id < a.pages) {
                page = id;
                const int64_t unit = static_cast<int64_t>(id) * a.kv_heads + kvh;
                const uint8_t* k = a.k_pool + (unit * a.pt + j % a.pt) * D;
                float dot = 0.f;
                for (int d = 0; d < D; ++d) dot = fmaf(sq[d], kv8_value<FP8>(k[d]), dot);
                s = dot * (a.scales[2 * unit] * a.scale);
                sv = a.scales[2 * unit + 1];
            }
        }
        const bool nan = __any(s != s);
        const float m_new = nan ? __uint_as_float(0x7FC00000u) : fmaxf(m, wave_max(s));
        if (m_new == -INFINITY) continue;  // wave-uniform: nothing seen so far
        const float alpha = m == -INFINITY ? 0.f : expf(m - m_new);
        const float p = page >= 0 ? expf(s - m_new) : 0.f;
        l = l * alpha + wave_sum(p);
#pragma unroll
        for (int r = 0; r < kRowMaxD / 64; ++r) acc[r] *= alpha;
        const float w = page >= 0 ? p * sv : 0.f;
        for (int c = 0; c < min(64, end - base); ++c) {
            const int pg = lane_bcast(page, c);
            const float wc = lane_bcast(w, c);
            if (pg < 0) continue;  // wave-uniform
            const uint8_t* v = a.v_pool + (static_cast<int64_t>(pg) * a.kv_heads + kvh) * D * a.pt + (base + c) % a.pt;
#pragma unroll
            for (int r = 0; r < kRowMaxD / 64; ++r) {
                const int d = lane + 64 * r;
                if (d < D) acc[r] = fmaf(wc, kv8_value<FP8>(v[static_cast<int64_t>(d) * a.pt]), acc[r]);
            }
        }
        m = m_new;
    }
#pragma unroll
    for (int r = 0; r < kRowMaxD / 64; ++r) {
        const int d = lane + 64 * r;
        if (d < D) kv8_store(a.out, a.out_f32, t * a.out_stride + static_cast<int64_t>(h) * D + d, acc[r] / l);  // (nothing seen: 0 / 0)
    }
}

// ===========================================================================
// Head dim 64 and 128, pages of whole 16 tokens, on the matrix cores.
//
// The rows x group query columns of a (sequence, kv head) fill columns of 16; a wave holds NT
// of those.  It walks tiles of 64 tokens, four runs of 16 that lie on a page each:
//   S^T[64 tok][16 q] = K[64 tok][D] Q^T[D][16 q]       4 x D/32 x mfma_16x16x32_bf16
//   O^T[D][16 q]     += V^T[D][64 tok] P^T[64 tok][16 q]  D/16 x 2 x mfma_16x16x32_bf16
// Codes become bf16 exactly (int8: 8 bits, e4m3: 4), so the products run over codes and the
// scales go where they are one number a lane.  Which token a row of K's operand is and which
// dims a lane's k-slice holds is free as long as Q and V agree, and is chosen so that every
// load is 16 bytes and nothing crosses lanes between the two products: row r of the
// i-th operand is token 4 i + (r & 3) of run r >> 2, so lane (q, g) ends up with all 16 scores
// of run g in token order -- which is what the second product's operand wants of it, its
// k-slices being tokens 0 .. 7 and 8 .. 15 of run g, the two halves of the 16 bytes that a V
// row holds of that run.  K's scale of run g then multiplies the lane's scores, V's its weights.
//
// Weights (times V's scale) enter the second product as two bf16 terms (PT = 2: 16 bits) or
// three (24); fp32 queries as three (QT = 3).  Scores, softmax statistics and sums are fp32.
//
// Bound by HBM: a tile is 64 tokens x 2 D bytes, against 4 x (16 + 8 PT x 2) MFMA cycles and the
// codes' conversion.  K's registers are loaded again as soon as the first product has read
// them, V's after the second: a wave has up to 16 KB in flight.
//
// A workgroup is four waves: one column group, its tiles split four ways, for up to 16 NT
// columns; two by two for twice that; else four column groups over the same tiles.
// ===========================================================================
namespace {

constexpr int kTile = 64;

__device__ __forceinline__ int ceil_div(int a, int b) { return (a + b - 1) / b; }

// Columns that a workgroup takes of a sequence: its waves' tiles split four ways, two ways or
// not at all.
__device__ __forceinline__ int ways_of(int cols, int width) { return cols > 2 * width ? 1 : cols > width ? 2 : 4; }
__device__ __forceinline__ int blocks_of(int cols, int width) { return cols > 4 * width ? ceil_div(cols, 4 * width) : cols > 0; }

// A slot of the grid: block `block` of a sequence's columns, split `split` of its tiles, of which
// each split has `each`.  Its slots begin at `first`, splits of a block side by side.
struct Slot {
    int b, block, split, splits, each, first;
};

// Sequences are split so that every workgroup has about the same number of tiles: all blocks'
// tiles over `share`; share and the blocks together bound the slots.  Each wave works it out for
// itself from the lengths.
template <int WIDTH>
__device__ bool find_slot(const Kv8Args& a, int slot, Slot& s) {
    if (a.direct) {  // a slot a sequence
        int t0, rows, len;
        a.sequence(slot, t0, rows, len);
        s = {slot, 0, 0, 1, 0x3FFFFFFF, slot};
        return rows > 0;
    }
    const int lane = threadIdx.x & 63;
    int tiles = 0, blocks = 0;
    auto load = [&](int b) {  // a sequence's tiles (at least one) and blocks, none without rows
        tiles = blocks = 0;
        if (b < a.batch) {
            int t0, rows, len;
            a.sequence(b, t0, rows, len);
            blocks = blocks_of(min(rows, a.max_rows) * a.group, WIDTH);
            tiles = max(ceil_div(len, kTile), 1);
        }
    };
    int each = 0x3FFFFFFF;
    load(lane);
    if (a.share) {
        int64_t all = 0;
        for (int base = 0;;) {
            // (64 sequences' tiles times blocks may pass 32 bits)
            int64_t n = static_cast<int64_t>(tiles) * blocks;
#pragma unroll
            for (int off = 32; off > 0; off >>= 1) n += __shfl_xor(n, off, kWave);
            all += n;
            if ((base += kWave) >= a.batch) break;
            load(base + lane);
        }
        each = static_cast<int>(max((all + a.share - 1) / a.share, static_cast<int64_t>(a.least)));
        if (a.batch > kWave) load(lane);
    }
    int before = 0;
    for (int base = 0;;) {
        const int mine_each = a.fixed ? ceil_div(tiles, a.fixed) : each;
        const int splits = blocks > 0 ? ceil_div(tiles, mine_each) : 0;
        const int upto = wave_inclusive(splits * blocks) + before;
        const uint64_t behind = __ballot(upto > slot);
        if (behind) {
            const int l = __builtin_ctzll(behind);
            s.b = base + l;
            s.splits = __builtin_amdgcn_readlane(splits, l);
            s.each = __builtin_amdgcn_readlane(mine_each, l);
            s.first = __builtin_amdgcn_readlane(upto - splits * blocks, l);
            s.block = (slot - s.first) / s.splits;
            s.split = slot - s.first - s.block * s.splits;
            return true;
        }
        before = __builtin_amdgcn_readlane(upto, 63);
        if ((base += kWave) >= a.batch) return false;
        load(base + lane);
    }
}

// 8 codes as an MFMA operand.
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
template <bool FP8>
__device__ __forceinline__ bf16x8 kv8_operand(uint32_t lo, uint32_t hi) {
    if constexpr (FP8) {
        uint4 r;
        r.x = __builtin_bit_cast(uint32_t, (bf16x2)__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, false));
        r.y = __builtin_bit_cast(uint32_t, (bf16x2)__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, true));
        r.z = __builtin_bit_cast(uint32_t, (bf16x2)__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, false));
        r.w = __builtin_bit_cast(uint32_t, (bf16x2)__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, true));
        return as_bf16x8(r);
    } else {
        return as_bf16x8(i8x8_to_bf16x8(lo, hi));
    }
}

// Two weights as PT bf16 terms, packed (each truncated, the last of two rounded).
template <int PT>
__device__ __forceinline__ void weight_terms(float p0, float p1, uint32_t* t) {
    if constexpr (PT == 2) {
        split2_weights(p0, p1, t[0], t[1]);
    } else {
        const uint32_t u0 = __float_as_uint(p0), u1 = __float_as_uint(p1);
        t[0] = __builtin_amdgcn_perm(u1, u0, 0x07060302u);
        const uint32_t r0 = __float_as_uint(p0 - __uint_as_float(u0 & 0xFFFF0000u)), r1 = __float_as_uint(p1 - __uint_as_float(u1 & 0xFFFF0000u));
        t[1] = __builtin_amdgcn_perm(r1, r0, 0x07060302u);
        t[2] = cvt_pk_bf16(__uint_as_float(r0) - __uint_as_float(r0 & 0xFFFF0000u), __uint_as_float(r1) - __uint_as_float(r1 & 0xFFFF0000u));
    }
}

}  // namespace

template <bool FP8, int D, int QT, int PT, int NT>
__global__ __launch_bounds__(256) void attn_kv8_kernel(Kv8Args a) {
    static_assert(D == 64 || D == 128, "16 bytes of 4 lanes make a k-step");
    constexpr int kF = D / 32, kDt = D / 16, kLd = D + 4, kCols = 16 * NT;
    __shared__ float so[4][kCols][kLd];
    __shared__ float sm[4][kCols], sl[4][kCols];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, lr = lane & 15, lg = lane >> 4;
    const int slot = blockIdx.x / a.kv_heads, kvh = blockIdx.x - slot * a.kv_heads;
    Slot at;
    int t0, rows, len;
    if (!find_slot<kCols>(a, slot, at)) return;
    a.sequence(at.b, t0, rows, len);
    const int cols = min(rows, a.max_rows) * a.group;
    const int ways = ways_of(cols, kCols), groups = 4 / ways, col0 = at.block * groups * kCols;
    const int wcol = col0 + wave % groups * kCols;  // (may lie behind the columns)
    // tokens that all of the wave's columns see, and that any does
    const int seen_all = max(len - rows + wcol / a.group + 1, 0);
    const int seen_any = wcol < cols ? max(len - rows + min(wcol + kCols - 1, cols - 1) / a.group + 1, 0) : 0;
    const int64_t from = static_cast<int64_t>(at.split) * at.each;
    const int tile0 = static_cast<int>(min(from, static_cast<int64_t>(0x3FFFFFFF)));
    const int span = max(static_cast<int>(min(from + at.each, static_cast<int64_t>(ceil_div(seen_any, kTile)))) - tile0, 0);
    const int way = wave / groups;
    const int begin = tile0 + static_cast<int>(static_cast<int64_t>(span) * way / ways), end = tile0 + static_cast<int>(static_cast<int64_t>(span) * (way + 1) / ways);

    // Q^T: lane (q, g) holds dims 64 (f / 2) + 16 g + 8 (f % 2) + [0, 8) of column q
    bf16x8 qf[NT][kF][QT];
    int seen[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        const int c = wcol + 16 * n + lr, i = c / a.group;
        const bool live = c < cols;
        seen[n] = live ? max(len - rows + i + 1, 0) : 0;
        const int64_t row = static_cast<int64_t>(t0 + (live ? i : 0)) * a.q_stride + static_cast<int64_t>(kvh * a.group + (live ? c - i * a.group : 0)) * D + 16 * lg;
#pragma unroll
        for (int f = 0; f < kF; ++f) {
            const int64_t o = row + 64 * (f >> 1) + 8 * (f & 1);
            if constexpr (QT == 1) {
                const uint16_t* p = static_cast<const uint16_t*>(a.q) + o;
                uint4 w;
                if (a.vec) w = *reinterpret_cast<const uint4*>(p);
                else w = make_uint4(p[0] | p[1] << 16, p[2] | p[3] << 16, p[4] | p[5] << 16, p[6] | p[7] << 16);
                qf[n][f][0] = as_bf16x8(live ? w : make_uint4(0, 0, 0, 0));
            } else {
                uint16_t t[3][8];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float v = live ? kv8_load(a.q, a.q_f32, o + e) : 0.f;
                    split3(v, t[0][e], t[1][e], t[2][e]);
                }
#pragma unroll
                for (int s = 0; s < QT; ++s) qf[n][f][s] = __builtin_bit_cast(bf16x8, t[s]);
            }
        }
    }
    const float scale = a.scale * kLog2e;
    const int runs = a.pt >> 4;  // 16-token runs of a page
    const int32_t* table = a.page_table + static_cast<int64_t>(at.b) * a.per;
    // run s of the sequence (at most the last tile's): its page, and where it lies there
    auto page_of = [&](int s, int& sub) {
        const int page = runs == 1 ? s : s / runs;
        sub = runs == 1 ? 0 : s - page * runs;
        return table[min(page, a.per - 1)];
    };
    uint4 kr[4][D / 64], vr[kDt];
    float2 sc;
    bool vok;
    auto load_k = [&](int page, int sub) {
        const bool ok = static_cast<uint32_t>(page) < static_cast<uint32_t>(a.pages);
        const int64_t u = (static_cast<int64_t>(ok ? page : 0) * a.kv_heads + kvh) * (a.pt * D) + (sub * 16 + (lr & 3)) * D + 16 * lg;
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < D / 64; ++j) kr[i][j] = *reinterpret_cast<const uint4*>(a.k_pool + u + i * 4 * D + j * 64);
    };
    auto load_v = [&](int page, int sub) {
        vok = static_cast<uint32_t>(page) < static_cast<uint32_t>(a.pages);
        const int64_t u = static_cast<int64_t>(vok ? page : 0) * a.kv_heads + kvh;
        sc = reinterpret_cast<const float2*>(a.scales)[u];
        const uint8_t* p = a.v_pool + u * (a.pt * D) + static_cast<int64_t>(lr) * a.pt + sub * 16;
#pragma unroll
        for (int i = 0; i < kDt; ++i) vr[i] = *reinterpret_cast<const uint4*>(p + static_cast<int64_t>(i) * 16 * a.pt);
    };
    floatx4 o[NT][kDt] = {};
    float m[NT], l[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        m[n] = -INFINITY;
        l[n] = 0.f;
    }
    if (begin < end) {
        int sub_k, sub_v;
        int page_k = page_of(4 * begin + (lr >> 2), sub_k), page_v = page_of(4 * begin + lg, sub_v);
        load_k(page_k, sub_k);
        load_v(page_v, sub_v);
        // the pages of the tile behind the one in flight
        int next = min(begin + 1, end - 1);
        page_k = page_of(4 * next + (lr >> 2), sub_k);
        page_v = page_of(4 * next + lg, sub_v);
        for (int t = begin; t < end; ++t) {
            floatx4 s[NT][4] = {};
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int f = 0; f < kF; ++f) {
                    const uint4& w = kr[i][f >> 1];
                    const bf16x8 k = f & 1 ? kv8_operand<FP8>(w.z, w.w) : kv8_operand<FP8>(w.x, w.y);
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int e = QT - 1; e >= 0; --e) s[n][i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k, qf[n][f][e], s[n][i], 0, 0, 0);
                }
            if (t + 1 < end) load_k(page_k, sub_k);
            const int base = t * kTile + lg * 16;  // the lane's run
            const float fk = sc.x * scale, fv = sc.y;
            const bool part = t * kTile + kTile > seen_all || __any(!vok);
            uint32_t pw[NT][PT][8];
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const int live = vok ? min(max(seen[n] - base, 0), 16) : 0;  // tokens of the run that the column sees
                float top = -INFINITY;
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        s[n][i][r] *= fk;
                        if (part && 4 * i + r >= live) s[n][i][r] = -INFINITY;
                        top = fmaxf(top, s[n][i][r]);
                    }
                top = xor32_max(xor16_max(top));
                // the running maximum moves only when a score is 2^8 above it
                if (__any(top > m[n] + 8.0f)) {
                    const float to = fmaxf(m[n], top);
                    const float alpha = to == m[n] ? 1.0f : __builtin_amdgcn_exp2f(m[n] - to);
                    m[n] = to;
                    l[n] *= alpha;
#pragma unroll
                    for (int d = 0; d < kDt; ++d)
#pragma unroll
                        for (int r = 0; r < 4; ++r) o[n][d][r] *= alpha;
                }
                const float ref = m[n] == -INFINITY ? 0.0f : m[n];
                float w[16];
                float sum = 0.f;
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const float p = __builtin_amdgcn_exp2f(s[n][i][r] - ref);
                        sum += p;
                        w[4 * i + r] = part && 4 * i + r >= live ? 0.0f : p * fv;
                    }
                l[n] += sum;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    uint32_t e[PT];
                    weight_terms<PT>(w[2 * i], w[2 * i + 1], e);
#pragma unroll
                    for (int x = 0; x < PT; ++x) pw[n][x][i] = e[x];
                }
            }
            if (FP8 && part) {  // codes that no row sees may be NaN: 0 * NaN
                const int held = vok ? min(max(len - base, 0), 16) : 0;
#pragma unroll
                for (int i = 0; i < kDt; ++i) {
                    uint32_t* w = &vr[i].x;
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const int k = min(max(held - 4 * j, 0), 4);
                        w[j] = k == 4 ? w[j] : w[j] & ((1u << (8 * k)) - 1u);
                    }
                }
            }
#pragma unroll
            for (int d = 0; d < kDt; ++d) {
                const bf16x8 v0 = kv8_operand<FP8>(vr[d].x, vr[d].y), v1 = kv8_operand<FP8>(vr[d].z, vr[d].w);
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int x = PT - 1; x >= 0; --x) {
                        const uint32_t* p = pw[n][x];
                        o[n][d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v0, as_bf16x8(make_uint4(p[0], p[1], p[2], p[3])), o[n][d], 0, 0, 0);
                        o[n][d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v1, as_bf16x8(make_uint4(p[4], p[5], p[6], p[7])), o[n][d], 0, 0, 0);
                    }
            }
            if (t + 1 < end) {
                load_v(page_v, sub_v);
                next = min(t + 2, end - 1);
                page_k = page_of(4 * next + (lr >> 2), sub_k);
                page_v = page_of(4 * next + lg, sub_v);
            }
        }
    }
    // the waves of a column group, joined in LDS
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        l[n] = xor32_sum(xor16_sum(l[n]));
        if (lg == 0) {
            sm[wave][16 * n + lr] = m[n];
            sl[wave][16 * n + lr] = l[n];
        }
    }
    __syncthreads();
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        float top = -INFINITY;
        for (int w = wave % groups; w < 4; w += groups) top = fmaxf(top, sm[w][16 * n + lr]);
        const float f = m[n] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m[n] - top);
#pragma unroll
        for (int d = 0; d < kDt; ++d) {
            float4 v = make_float4(o[n][d][0] * f, o[n][d][1] * f, o[n][d][2] * f, o[n][d][3] * f);
            *reinterpret_cast<float4*>(&so[wave][16 * n + lr][16 * d + 4 * lg]) = v;
        }
    }
    __syncthreads();
    const int64_t part = static_cast<int64_t>(blockIdx.x) * a.width;
    for (int e = threadIdx.x; e < groups * kCols * (D / 4); e += 256) {
        const int c = e / (D / 4), d = e % (D / 4) * 4, gr = c / kCols, cc = c % kCols;
        const int col = col0 + c;
        if (col >= cols) break;
        float top = -INFINITY, sum = 0.f;
        for (int w = gr; w < 4; w += groups) top = fmaxf(top, sm[w][cc]);
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int w = gr; w < 4; w += groups) {
            sum += sl[w][cc] * (sm[w][cc] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(sm[w][cc] - top));
            const float4 x = *reinterpret_cast<const float4*>(&so[w][cc][d]);
            v.x += x.x; v.y += x.y; v.z += x.z; v.w += x.w;
        }
        const int i = col / a.group;
        if (at.splits == 1) {
            kv8_store4(a, static_cast<int64_t>(t0 + i) * a.out_stride + static_cast<int64_t>(kvh * a.group + col - i * a.group) * D + d, v, sum);
        } else {
            *reinterpret_cast<float4*>(a.part_acc + (part + c) * D + d) = v;
            if (d == 0) a.part_ml[part + c] = make_float2(top, sum);
        }
    }
    // where the join finds a row's sequence, and the sequence's slots
    if (a.slot_of && at.split == 0 && kvh == 0) {
        if (at.block == 0 && threadIdx.x == 0) a.slot_of[at.b] = make_int2(at.first, at.splits);
        for (int e = threadIdx.x; e < groups * kCols; e += 256)
            if (col0 + e < cols) a.sequence_of[t0 + (col0 + e) / a.group] = at.b;
    }
}

// The splits of a row and kv head: weights 2^(m_s - M), a sum in the splits' order.
template <int D, int WIDTH>
__global__ __launch_bounds__(128) void attn_kv8_join_kernel(Kv8Args a) {
    const int t = blockIdx.x, kvh = blockIdx.y;
    if (a.starts && t >= a.starts[a.batch]) return;
    const int b = min(max(a.sequence_of[t], 0), a.batch - 1);
    int t0, rows, len;
    a.sequence(b, t0, rows, len);
    const int i = t - t0;
    rows = min(rows, a.max_rows);
    if (i < 0 || i >= rows) return;  // (a row that no sequence computes)
    const int2 at = a.slot_of[b];
    const int cols = rows * a.group, wide = 4 / ways_of(cols, WIDTH) * WIDTH;
    if (at.y <= 1) return;
    for (int e = threadIdx.x; e < a.group * (D / 4); e += 128) {
        const int g = e / (D / 4), d = e % (D / 4) * 4;
        const int c = i * a.group + g, block = c / wide;
        const int64_t slot = at.x + static_cast<int64_t>(block) * at.y;
        if (slot < 0 || slot + at.y > a.slots) return;
        const int64_t col = (slot * a.kv_heads + kvh) * a.width + c - block * wide, step = static_cast<int64_t>(a.kv_heads) * a.width;
        float top = -INFINITY;
        for (int s = 0; s < at.y; ++s) top = fmaxf(top, a.part_ml[col + s * step].x);
        float sum = 0.f;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
        for (int s = 0; s < at.y; ++s) {
            const float2 ml = a.part_ml[col + s * step];
            const float4 x = *reinterpret_cast<const float4*>(a.part_acc + (col + s * step) * D + d);
            const float f = ml.x == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(ml.x - top);
            sum = fmaf(ml.y, f, sum);
            v.x = fmaf(x.x, f, v.x); v.y = fmaf(x.y, f, v.y); v.z = fmaf(x.z, f, v.z); v.w = fmaf(x.w, f, v.w);
        }
        kv8_store4(a, static_cast<int64_t>(t) * a.out_stride + static_cast<int64_t>(kvh * a.group + g) * D + d, v, sum);
    }
}

namespace {

size_t up256(size_t n) { return (n + 255) & ~static_cast<size_t>(255); }

size_t kv8_bytes(const sfg_kv8_attn_args& a, int64_t slots, int width) {
    const size_t columns = static_cast<size_t>(slots) * a.kv_heads * width;
    return up256(a.batch * sizeof(int2)) + up256(a.tokens * sizeof(int)) + up256(columns * sizeof(float2)) + up256(columns * a.head_dim * sizeof(float));
}

constexpr int64_t kMostSlots = 1 << 22;  // workgroups of a launch: 256 threads each

}  // namespace

Kv8Plan plan_attn_kv8(const sfg_kv8_attn_args& a) {
    Kv8Plan p{};
    if ((a.head_dim != 64 && a.head_dim != 128) || a.page_tokens % 16) return p;
    const bool narrow = a.q_dtype == SFG_BF16 && a.out_dtype == SFG_BF16;
    const int64_t group = a.q_heads / a.kv_heads, cols = a.max_rows * group;
    const int64_t tiles = std::max<int64_t>((a.max_context + kTile - 1) / kTile, 1);
    p.nt = narrow && cols > 16 ? 2 : 1;
    p.width = 16 * p.nt * (cols > 32 * p.nt ? 4 : cols > 16 * p.nt ? 2 : 1);
    const int64_t blocks = a.tokens * group / (64 * p.nt) + a.batch;  // of all sequences, at most
    if (blocks * a.kv_heads > kMostSlots) return p;
    p.mfma = true;
    p.least = 4;
    p.slots = static_cast<int>(blocks);
    p.direct = cols <= 64 * p.nt;
    if (p.direct) p.slots = static_cast<int>(a.batch);
    if (a.kv_splits > 0) {
        const int64_t fixed = std::min<int64_t>({a.kv_splits, tiles, kMostSlots / (blocks * a.kv_heads)});
        if (fixed > 1) {
            p.fixed = static_cast<int>(fixed);
            p.slots = static_cast<int>(blocks * fixed);
        }
    } else {
        const int64_t share = 1024 / a.kv_heads;
        const int64_t slots = std::min(share + blocks, blocks * ((tiles + p.least - 1) / p.least));
        if (share > blocks && slots > blocks && kv8_bytes(a, slots, p.width) <= (size_t{128} << 20)) {
            p.share = static_cast<int>(share);
            p.slots = static_cast<int>(slots);
        }
    }
    if (p.share || p.fixed) {
        p.direct = false;
        p.bytes = kv8_bytes(a, p.slots, p.width);
    }
    return p;
}

namespace {

template <bool FP8, int D>
void launch_kv8_mfma(const Kv8Args& a, const Kv8Plan& p, bool narrow, hipStream_t stream) {
    const dim3 grid(static_cast<unsigned>(p.slots * a.kv_heads));
    if (!narrow) attn_kv8_kernel<FP8, D, 3, 3, 1><<<grid, 256, 0, stream>>>(a);
    else if (p.nt == 2) attn_kv8_kernel<FP8, D, 1, 2, 2><<<grid, 256, 0, stream>>>(a);
    else attn_kv8_kernel<FP8, D, 1, 2, 1><<<grid, 256, 0, stream>>>(a);
    if (!p.bytes) return;
    const dim3 joins(static_cast<unsigned>(a.tokens), static_cast<unsigned>(a.kv_heads));
    if (p.nt == 2) attn_kv8_join_kernel<D, 32><<<joins, 128, 0, stream>>>(a);
    else attn_kv8_join_kernel<D, 16><<<joins, 128, 0, stream>>>(a);
}

}  // namespace

void launch_attn_kv8(const sfg_kv8_attn_args& s, const Kv8Plan& plan, void* workspace, hipStream_t stream) {
    Kv8Args a{};
    a.q = s.q; a.q_stride = s.q_stride; a.q_f32 = s.q_dtype == SFG_F32;
    a.out = s.out; a.out_stride = s.out_stride; a.out_f32 = s.out_dtype == SFG_F32;
    a.k_pool = static_cast<const uint8_t*>(s.k_pool); a.v_pool = static_cast<const uint8_t*>(s.v_pool); a.scales = s.scales;
    a.page_table = s.page_table; a.seq_lens = s.seq_lens; a.starts = s.starts;
    a.batch = static_cast<int>(s.batch); a.tokens = static_cast<int>(s.tokens); a.max_rows = static_cast<int>(s.max_rows);
    a.q_heads = static_cast<int>(s.q_heads); a.kv_heads = static_cast<int>(s.kv_heads); a.dim = static_cast<int>(s.head_dim);
    a.pt = static_cast<int>(s.page_tokens); a.per = static_cast<int>(s.pages_per_seq); a.pages = static_cast<int>(s.num_pages);
    a.max_context = static_cast<int>(s.max_context);
    a.scale = s.scale > 0.0f ? s.scale : 1.0f / sqrtf(static_cast<float>(s.head_dim));
    const bool narrow = s.q_dtype == SFG_BF16 && s.out_dtype == SFG_BF16;
    // codes are read 16 bytes at a time, scales in pairs
    const bool aligned = ((reinterpret_cast<uintptr_t>(s.k_pool) | reinterpret_cast<uintptr_t>(s.v_pool)) & 15) == 0 &&
                         (reinterpret_cast<uintptr_t>(s.scales) & 7) == 0;
    if (plan.mfma && aligned) {
        a.group = a.q_heads / a.kv_heads;
        a.slots = plan.slots; a.share = plan.share; a.fixed = plan.fixed; a.least = plan.least;
        a.direct = plan.direct; a.width = plan.width;
        a.vec = (reinterpret_cast<uintptr_t>(s.q) & 15) == 0 && s.q_stride % 8 == 0;
        a.out_vec = (reinterpret_cast<uintptr_t>(s.out) & 15) == 0 && s.out_stride % 4 == 0;
        if (plan.bytes) {
            char* at = static_cast<char*>(workspace);
            const size_t columns = static_cast<size_t>(plan.slots) * a.kv_heads * plan.width;
            a.slot_of = reinterpret_cast<int2*>(at); at += up256(a.batch * sizeof(int2));
            a.sequence_of = reinterpret_cast<int*>(at); at += up256(a.tokens * sizeof(int));
            a.part_ml = reinterpret_cast<float2*>(at); at += up256(columns * sizeof(float2));
            a.part_acc = reinterpret_cast<float*>(at);
        }
        if (s.pool_dtype == SFG_FP8) {
            if (a.dim == 128) launch_kv8_mfma<true, 128>(a, plan, narrow, stream);
            else launch_kv8_mfma<true, 64>(a, plan, narrow, stream);
        } else {
            if (a.dim == 128) launch_kv8_mfma<false, 128>(a, plan, narrow, stream);
            else launch_kv8_mfma<false, 64>(a, plan, narrow, stream);
        }
        return;
    }
    const dim3 grid(static_cast<unsigned>(a.tokens), static_cast<unsigned>(a.q_heads));
    if (s.pool_dtype == SFG_FP8) attn_kv8_rows_kernel<true><<<grid, 64, 0, stream>>>(a);
    else attn_kv8_rows_kernel<false><<<grid, 64, 0, stream>>>(a);
}

}  // namespace sfg
