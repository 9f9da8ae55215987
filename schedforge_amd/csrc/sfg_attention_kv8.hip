// sfg_attention_kv8.hip -- causal attention of each sequence's newest rows over a paged
// cache held in 8 bits (codes with a scale for each page, kv head and pool).
#include <math.h>

#include <algorithm>
#include <bit>

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
    int group;
    // the matrix-core kernels' (the rows kernel: fixed)
    int slots, share, quads, fixed, least, few, width, row_shift;  // (as in Kv8Plan)
    int vec, out_vec;                                      // rows begin on 16-byte boundaries
    int4* slot_of; int* sequence_of; float2* part_ml; float* part_acc;
    // A column's row (single rows without the division).
    __device__ __forceinline__ int row_of(int col) const { return col < group ? 0 : col / group; }
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
    const float inv = 1.0f / sum;  // (0 times its infinity is NaN)
    const float4 y = make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv);
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

// Any head dim up to kRowMaxD and any page size: a wave a row, query head and split of its
// tokens, 64 of those at a time with a token a lane for the scores and a dim a lane for the
// values.  WORDS: head dim and page are multiples of 4, codes are read four at a time.  16 sequences
// of up to 4096 tokens, 32 heads of 80 over 8: 197 us (without splits and words 1220).
template <bool FP8, bool WORDS>
__global__ __launch_bounds__(64) void attn_kv8_rows_kernel(Kv8Args a) {
    __shared__ float sq[kRowMaxD];
    const int lane = threadIdx.x, t = blockIdx.x, h = blockIdx.y, split = blockIdx.z;
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
    const int D = a.dim, kvh = h / a.group;
    const int seen = min(max(len - rows + i + 1, 0), len), chunks = (seen + 63) / 64;
    const int begin = static_cast<int>(static_cast<int64_t>(chunks) * split / a.fixed) * 64;
    const int end = min(static_cast<int>(static_cast<int64_t>(chunks) * (split + 1) / a.fixed) * 64, seen);
    for (int d = lane; d < D; d += 64) sq[d] = kv8_load(a.q, a.q_f32, t * a.q_stride + static_cast<int64_t>(h) * D + d);
    __syncthreads();
    const int32_t* table = a.page_table + static_cast<int64_t>(b) * a.per;
    float m = -INFINITY, l = 0.f;
    float acc[kRowMaxD / 64] = {};
    for (int base = begin; base < end; base += 64) {
        const int j = base + lane, count = min(64, end - base);
        float s = -INFINITY, sv = 0.f;
        int page = -1;
        if (j < end) {
            const int id = table[j / a.pt];
            if (id >= 0 && id < a.pages) {
                page = id;
                const int64_t unit = static_cast<int64_t>(id) * a.kv_heads + kvh;
                const uint8_t* k = a.k_pool + (unit * a.pt + j % a.pt) * D;
                float dot = 0.f;
                if constexpr (WORDS) {
#pragma unroll 4
                    for (int d = 0; d < D; d += 4) {
                        const uint32_t w = *reinterpret_cast<const uint32_t*>(k + d);
#pragma unroll
                        for (int e = 0; e < 4; ++e) dot = fmaf(sq[d + e], kv8_value<FP8>(static_cast<uint8_t>(w >> (8 * e))), dot);
                    }
                } else {
                    for (int d = 0; d < D; ++d) dot = fmaf(sq[d], kv8_value<FP8>(k[d]), dot);
                }
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
        constexpr int kStep = WORDS ? 4 : 1;
        for (int c = 0; c < count; c += kStep) {
            const int pg = lane_bcast(page, c);  // (of all kStep tokens)
            if (pg < 0) continue;                // wave-uniform
            const uint8_t* v = a.v_pool + (static_cast<int64_t>(pg) * a.kv_heads + kvh) * D * a.pt + (base + c) % a.pt;
#pragma unroll
            for (int r = 0; r < kRowMaxD / 64; ++r) {
                const int d = lane + 64 * r;
                if (d >= D) continue;
                if constexpr (WORDS) {
                    const uint32_t x = *reinterpret_cast<const uint32_t*>(v + static_cast<int64_t>(d) * a.pt);
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (c + e < count) acc[r] = fmaf(lane_bcast(w, c + e), kv8_value<FP8>(static_cast<uint8_t>(x >> (8 * e))), acc[r]);
                } else {
                    acc[r] = fmaf(lane_bcast(w, c), kv8_value<FP8>(v[static_cast<int64_t>(d) * a.pt]), acc[r]);
                }
            }
        }
        m = m_new;
    }
    const int64_t part = (static_cast<int64_t>(t) * a.q_heads + h) * a.fixed + split;
    if (a.part_ml && lane == 0) a.part_ml[part] = make_float2(m, l);
#pragma unroll
    for (int r = 0; r < kRowMaxD / 64; ++r) {
        const int d = lane + 64 * r;
        if (d >= D) continue;
        if (a.part_ml) a.part_acc[part * D + d] = acc[r];
        else kv8_store(a.out, a.out_f32, t * a.out_stride + static_cast<int64_t>(h) * D + d, acc[r] / l);  // (nothing seen: 0 / 0)
    }
    if (a.part_ml && h == 0 && split == 0 && lane == 0) a.sequence_of[t] = 1;  // (a row that is computed)
}

// The splits of a row and query head.
__global__ __launch_bounds__(64) void attn_kv8_rows_join_kernel(Kv8Args a) {
    const int lane = threadIdx.x, t = blockIdx.x, h = blockIdx.y, D = a.dim;
    if (a.sequence_of[t] == 0) return;
    const int64_t part = (static_cast<int64_t>(t) * a.q_heads + h) * a.fixed;
    float top = -INFINITY;
    bool nan = false;
    for (int s = 0; s < a.fixed; ++s) {
        top = fmaxf(top, a.part_ml[part + s].x);
        nan |= a.part_ml[part + s].x != a.part_ml[part + s].x;
    }
    float sum = nan ? __uint_as_float(0x7FC00000u) : 0.f;
    float acc[kRowMaxD / 64] = {};
#pragma unroll 4
    for (int s = 0; s < a.fixed; ++s) {
        const float2 ml = a.part_ml[part + s];
        const float f = ml.x == -INFINITY ? 0.f : expf(ml.x - top);
        sum = fmaf(ml.y, f, sum);
#pragma unroll
        for (int r = 0; r < kRowMaxD / 64; ++r)
            if (lane + 64 * r < D) acc[r] = fmaf(a.part_acc[(part + s) * D + lane + 64 * r], f, acc[r]);
    }
#pragma unroll
    for (int r = 0; r < kRowMaxD / 64; ++r)
        if (lane + 64 * r < D) kv8_store(a.out, a.out_f32, t * a.out_stride + static_cast<int64_t>(h) * D + lane + 64 * r, acc[r] / sum);
}

// Which rows a call computes (the join's others stay as they were).
__global__ __launch_bounds__(256) void attn_kv8_rows_begin_kernel(int* computed, int tokens) {
    const int t = blockIdx.x * 256 + threadIdx.x;
    if (t < tokens) computed[t] = 0;
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
// them, V's after the second: a wave has up to 16 KB in flight.  64 sequences of up to 8192 tokens, 32
// heads of 128 over 8, int8: 103 us (540 MB at 5.3 TB/s).  With many rows (four column groups over
// the same tiles) by the units: beside one wave's matrix instructions of 16 cycles another one's
// vector instructions get 6, and the clock is near 2 GHz.  4096 rows over 4096 tokens, e4m3:
// 254 us, 540 TFLOP/s (32 x 32 x 16 products, which leave more to the other wave: 265; int8 301 and 292).
//
// A workgroup is four waves: one column group, its tiles split four ways, for up to 16 NT
// columns; two by two for twice that; else four column groups over the same tiles.  (Eight waves
// where that makes a split and its join unnecessary.)
// ===========================================================================
namespace {

constexpr int kTile = 64;

__device__ __forceinline__ int ceil_div(int a, int b) { return (a + b - 1) / b; }

// Column groups of `width` that a workgroup has of a sequence: each has its share of the waves, which
// split the tiles.
__device__ __forceinline__ int groups_of(int cols, int width) { return cols > 2 * width ? 4 : cols > width ? 2 : 1; }
__device__ __forceinline__ int blocks_of(int cols, int width) { return cols > 4 * width ? ceil_div(cols, 4 * width) : cols > 0; }

// A sequence's blocks of columns, the tiles that each walks and what it costs.  A block walks up to
// the last token that a row of it sees.  Where it has a whole number of rows, 2^row_shift, that and
// its sums are in closed form; else every block counts the sequence's tiles.  Costs: a tile 1, or
// 2 where each wave walks all of them (1.4 us for 3.5 with two workgroups a compute unit); a
// block's queries and sums two tiles', or four (10 us or more).  A prompt of 4096 rows: 254 us, dealt
// as if every block walked all tiles 342.  MANY: a sequence may have several blocks (for one, and 16
// columns, the code that is left out costs 0.3 us of 11.5).
template <bool MANY>
struct Blocks {
    int count, tiles;   // blocks, and tiles of the sequence (of the last block, where steps are known)
    int before, shift;  // tokens before the first row; rows of a block (-1: steps are not known)
    int twice;          // 1: a tile costs 2
    template <int WIDTH>
    __device__ __forceinline__ static Blocks of(const Kv8Args& a, int rows, int len) {
        const int live = min(rows, a.max_rows), cols = live * a.group;
        Blocks x{MANY ? blocks_of(cols, WIDTH) : cols > 0, max(ceil_div(len, kTile), 1), len - rows, -1, MANY && cols > 2 * WIDTH};
        if (MANY && x.count > 1 && x.before >= 0) {
            x.shift = a.row_shift;
            if (x.shift >= 0) x.tiles = max(ceil_div(x.before + live, kTile), 1);
        }
        return x;
    }
    __device__ __forceinline__ int tiles_of(int block) const {
        return MANY && shift >= 0 && block + 1 < count ? ceil_div(before + ((block + 1) << shift), kTile) : tiles;
    }
    // Tiles of the first n blocks, n < count.
    __device__ __forceinline__ int64_t sum(int n) const {
        if (shift < 0) return static_cast<int64_t>(n) * tiles;
        const int64_t pairs = static_cast<int64_t>(n) * (n - 1) / 2;
        if (shift >= 6) return static_cast<int64_t>(n) * ceil_div(before + (1 << shift), kTile) + (pairs << (shift - 6));
        // sums of floor((at + i) / 2^k)
        const int k = 6 - shift, at = (before + (1 << shift) + kTile - 1) >> shift;
        return upto(at + n, k) - upto(at, k);
    }
    __device__ __forceinline__ static int64_t upto(int m, int k) {
        const int64_t q = m >> k;
        return ((q * (q - 1) / 2) << k) + (m & ((1 << k) - 1)) * q;
    }
    // Costs: of a block's own work, of the first n blocks, n < count, and of all.
    __device__ __forceinline__ int own() const { return 2 + 2 * twice; }
    __device__ __forceinline__ int64_t cost(int n) const { return (sum(n) + static_cast<int64_t>(n) * own()) << twice; }
    __device__ __forceinline__ int64_t cost() const {
        if (!MANY) return count * (tiles + own());
        return ((count > 1 ? sum(count - 1) : 0) + (count > 0 ? tiles : 0) + static_cast<int64_t>(count) * own()) << twice;
    }
    // Where a block's tile begins among its costs.
    __device__ __forceinline__ int at(int tile) const { return (tile + own()) << twice; }
    // Its tiles that begin before a cost.
    __device__ __forceinline__ int tiles_before(int cost) const { return max(((cost + twice) >> twice) - own(), 0); }
};

// A unit of work: a block of a sequence's columns over its tiles.
template <bool MANY>
struct Unit {
    int b, block, tiles, t0, rows, len;
    Blocks<MANY> of;
    int ord;    // units before it
    int begin;  // costs before it, where tiles are dealt; else the pieces of the sequences before
};
// Starts and lengths that a caller left in disorder may give any cost: what the host has checked
// never reaches the cuts, and with them 64 of these and the sum before them fit 32 bits.
constexpr int kMostCost = 1 << 23, kMostCosts = 1 << 29;
__device__ __forceinline__ int cut(int64_t n) { return static_cast<int>(min(n, static_cast<int64_t>(kMostCost))); }
template <int WIDTH, bool MANY>
__device__ __forceinline__ void load_unit(const Kv8Args& a, int b, Unit<MANY>& u) {
    u.tiles = u.t0 = u.rows = u.len = 0;
    u.of = {};
    if (b >= a.batch) return;
    a.sequence(b, u.t0, u.rows, u.len);
    u.of = Blocks<MANY>::template of<WIDTH>(a, u.rows, u.len);
    u.tiles = u.of.tiles_of(0);
}

// How the units' tiles are given to workgroups, which each one works out from the lengths.
// Dealt (each 0): in units' order, the same cost to each of `groups`, across units: with a
// round of workgroups as long as the work, none waits for another's longer share.  Split: a unit
// into pieces of `each` tiles (of the sequence's, for each of its blocks), a workgroup a piece, where
// there are few: a second unit would double a workgroup's time.  64 sequences of up to 8192 tokens:
// dealt 103 us, split into 1280 pieces 129; 32 of up to 2000: 30 and 27.
struct Shares {
    int cost, groups, each, fixed;
    bool quads;  // a workgroup's waves take four kv heads, not a fourth of the tiles each
    // n: the sequences' tiles for each of their blocks
    __device__ Shares(const Kv8Args& a, int n, int of_all) : cost(of_all), groups(a.share), each(0), fixed(a.fixed) {
        quads = !fixed && a.quads && static_cast<int64_t>(n) * a.kv_heads >= a.quads;
        if (quads) groups *= 4;
        if (fixed || n <= groups * a.few) each = max(ceil_div(n, max(groups, 1)), a.least);
    }
    __device__ int pieces(int tiles) const { return ceil_div(tiles, fixed ? ceil_div(tiles, fixed) : each); }
    __device__ int begin(int w) const { return static_cast<int>(static_cast<int64_t>(cost) * w / groups); }
    __device__ int of(int at) const { return static_cast<int>((static_cast<int64_t>(at + 1) * groups - 1) / cost); }
};

// The unit that `at` of all costs belongs to (where units are split: piece `at`), and its place
// there.  first: the lane's sequence of the first 64.
template <int WIDTH, bool MANY>
__device__ __forceinline__ bool find_unit(const Kv8Args& a, const Shares& how, const Unit<MANY>& first, int at, Unit<MANY>& u, int& place) {
    const int lane = threadIdx.x & 63;
    int sum = 0, ord = 0;
    Unit<MANY> v = first;
    for (int base = 0;;) {
        const int mine = v.of.count == 0 ? 0 : cut(how.each ? static_cast<int64_t>(how.pieces(v.of.tiles)) * v.of.count : v.of.cost());
        const int upto = wave_inclusive(mine) + sum, units = wave_inclusive(v.of.count) + ord;
        const uint64_t behind = __ballot(upto > at);
        if (behind) {
            const int l = __builtin_ctzll(behind);
            u.b = base + l;
            u.of.count = __builtin_amdgcn_readlane(v.of.count, l);
            u.of.tiles = __builtin_amdgcn_readlane(v.of.tiles, l);
            u.of.before = __builtin_amdgcn_readlane(v.of.before, l);
            u.of.shift = __builtin_amdgcn_readlane(v.of.shift, l);
            u.t0 = __builtin_amdgcn_readlane(v.t0, l);
            u.rows = __builtin_amdgcn_readlane(v.rows, l);
            u.len = __builtin_amdgcn_readlane(v.len, l);
            u.of.twice = __builtin_amdgcn_readlane(v.of.twice, l);
            u.begin = __builtin_amdgcn_readlane(upto - mine, l);
            const int rest = at - u.begin;
            u.block = 0;
            place = rest;
            if (MANY && how.each) {
                const int of_block = how.pieces(u.of.tiles);
                u.block = rest / of_block;
                place = rest - u.block * of_block;
            } else if (MANY && u.of.count > 1) {  // the last block that begins there or before
                for (int from = 0; from < u.of.count; from += kWave) {
                    const uint64_t behind_it = __ballot(from + lane >= u.of.count || u.of.cost(from + lane) > rest);
                    u.block = max(from + (behind_it ? __builtin_ctzll(behind_it) : kWave) - 1, 0);
                    if (behind_it) break;
                }
                const int begin = static_cast<int>(u.of.cost(u.block));
                place = rest - begin;
                u.begin += begin;
            }
            u.ord = __builtin_amdgcn_readlane(units - v.of.count, l) + u.block;
            u.tiles = how.each ? u.of.tiles : u.of.tiles_of(u.block);
            return true;
        }
        sum = __builtin_amdgcn_readlane(upto, 63);
        ord = __builtin_amdgcn_readlane(units, 63);
        if ((base += kWave) >= a.batch) return false;
        load_unit<WIDTH>(a, base + lane, v);
    }
}

// Memory operations before it stay before those behind it.
__device__ __forceinline__ void in_order() { asm volatile("" ::: "memory"); }

// (the same in all lanes: kept in scalar registers)
__device__ __forceinline__ void same(int& x) { x = __builtin_amdgcn_readfirstlane(x); }
template <bool MANY>
__device__ __forceinline__ void same(Unit<MANY>& u) {
    same(u.b); same(u.block); same(u.tiles); same(u.t0); same(u.rows); same(u.len); same(u.ord); same(u.begin);
    same(u.of.count); same(u.of.tiles); same(u.of.before); same(u.of.shift); same(u.of.twice);
}

// The unit behind u, if there is one, where tiles are dealt.
template <int WIDTH, bool MANY>
__device__ __forceinline__ void next_unit(const Kv8Args& a, Unit<MANY>& u) {
    ++u.ord;
    u.begin += u.of.at(u.tiles);
    if (MANY && ++u.block < u.of.count) {
        u.tiles = u.of.tiles_of(u.block);
        return;
    }
    u.block = 0;
    do {
        load_unit<WIDTH>(a, ++u.b, u);
    } while (u.of.count == 0 && u.b < a.batch);
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

// 16 bytes of codes; ONCE: read by this workgroup alone, so not kept in the caches (64
// sequences of up to 8192 tokens: 112.5 us -> 102.9, two of 131072: 75.9 -> 70.3).
typedef uint32_t uint32x4 __attribute__((ext_vector_type(4)));
template <bool ONCE>
__device__ __forceinline__ uint4 kv8_fetch(const uint8_t* p) {
    if constexpr (ONCE) return __builtin_bit_cast(uint4, __builtin_nontemporal_load(reinterpret_cast<const uint32x4*>(p)));
    else return *reinterpret_cast<const uint4*>(p);
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

template <bool FP8, int D, int QT, int PT, int NT, bool P16, int WAVES>
__global__ __launch_bounds__(64 * WAVES, WAVES == 8 || NT == 2 ? 2 : QT == 3 ? (D == 64 ? 3 : 2) : D == 64 ? 4 : 3) void attn_kv8_kernel(Kv8Args a) {
    static_assert(D == 64 || D == 128, "16 bytes of 4 lanes make a k-step");
    constexpr int kF = D / 32, kDt = D / 16, kLd = D + 4, kCols = 16 * NT;
    // a wave's queries as operands, which the loop reads again for each tile; then its sums
    union Wave {
        uint4 q[NT][kF][QT][kWave];
        float o[kCols][kLd];
    };
    __shared__ Wave sw[WAVES];
    __shared__ float sm[WAVES][kCols], sl[WAVES][kCols];
    const int lane = threadIdx.x & 63, lr = lane & 15, lg = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const float scale = a.scale * kLog2e;
    const int pt = P16 ? 16 : a.pt, runs = pt >> 4;  // 16-token runs of a page

    // what this workgroup walks: a piece of a unit, or tiles of one unit after the other
    Unit<(NT == 2 || QT == 3)> first, u;  // (a row's 16 columns: one block)
    load_unit<kCols>(a, lane, first);
    int all = 0, cost = 0;
    if (!a.fixed) {
        u = first;
        for (int base = 0;;) {
            const int64_t n = static_cast<int64_t>(u.of.tiles) * u.of.count;
            all = min(all + __builtin_amdgcn_readlane(wave_inclusive(cut(n)), 63), kMostCosts);
            cost = min(cost + __builtin_amdgcn_readlane(wave_inclusive(cut(u.of.cost())), 63), kMostCosts);
            if ((base += kWave) >= a.batch) break;
            load_unit<kCols>(a, base + lane, u);
        }
    }
    Shares how(a, all, cost);
    same(how.each);
    const bool quads = WAVES == 4 && NT == 1 && how.quads;
    const int across = quads ? a.kv_heads >> 2 : a.kv_heads, group = blockIdx.x / across;
    const int kvh = quads ? 4 * (blockIdx.x - group * across) + wave : blockIdx.x - group * across;
    int tile0, count, until = 0;
    if (how.each) {
        if (!find_unit<kCols>(a, how, first, group, u, tile0)) return;
        const int each = how.fixed ? ceil_div(u.tiles, how.fixed) : how.each;
        tile0 *= each;
        count = min(each, u.tiles - tile0);
    } else {
        if (group >= how.groups) return;
        const int from = how.begin(group);
        until = how.begin(group + 1);
        if (!find_unit<kCols>(a, how, first, from, u, tile0)) return;
        tile0 = u.of.tiles_before(tile0);
        if (tile0 >= u.tiles) {
            next_unit<kCols>(a, u);
            tile0 = 0;
        }
        count = min(u.of.tiles_before(until - u.begin), u.tiles) - tile0;
    }
    same(until);
    for (;;) {
        same(u);
        same(tile0);
        same(count);
        if (count <= 0 || u.b >= a.batch) return;
        const int cols = min(u.rows, a.max_rows) * a.group;
        const int groups = quads ? 1 : groups_of(cols, kCols), ways = quads ? 1 : WAVES / groups, col0 = u.block * groups * kCols;
        const int wcol = col0 + wave % groups * kCols;  // (may lie behind the columns)
        // tokens that all of the wave's columns see, and that any does
        const int seen_all = max(u.len - u.rows + a.row_of(wcol) + 1, 0);
        const int seen_any = wcol < cols ? max(u.len - u.rows + a.row_of(min(wcol + kCols - 1, cols - 1)) + 1, 0) : 0;
        const int span = max(min(tile0 + count, ceil_div(seen_any, kTile)) - tile0, 0), way = quads ? 0 : wave / groups;
        const int begin = tile0 + static_cast<int>(static_cast<int64_t>(span) * way / ways);
        const int end = tile0 + static_cast<int>(static_cast<int64_t>(span) * (way + 1) / ways);
        const int32_t* table = a.page_table + static_cast<int64_t>(u.b) * a.per;
        // run s of the sequence (at most the last tile's): its page, and where it lies there
        auto page_of = [&](int s, int& sub) {
            const int page = P16 ? s : s / runs;
            sub = P16 ? 0 : s - page * runs;
            return table[min(page, a.per - 1)];
        };
        int sub_k, sub_v, page_k = -1, page_v = -1;
        if (begin < end) {
            page_k = page_of(4 * begin + (lr >> 2), sub_k);
            page_v = page_of(4 * begin + lg, sub_v);
        }
        // Q^T: lane (q, g) holds dims 64 (f / 2) + 16 g + 8 (f % 2) + [0, 8) of column q
        int seen[NT];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const int c = wcol + 16 * n + lr;
            const bool live = c < cols;
            const int i = live ? a.row_of(c) : 0;
            seen[n] = live ? max(u.len - u.rows + i + 1, 0) : 0;
            const int64_t row = static_cast<int64_t>(u.t0 + i) * a.q_stride + static_cast<int64_t>(kvh * a.group + (live ? c - i * a.group : 0)) * D + 16 * lg;
#pragma unroll
            for (int f = 0; f < kF; ++f) {
                const int64_t at = row + 64 * (f >> 1) + 8 * (f & 1);
                if constexpr (QT == 1) {
                    const uint16_t* p = static_cast<const uint16_t*>(a.q) + at;
                    uint4 w;
                    if (a.vec) w = *reinterpret_cast<const uint4*>(p);
                    else w = make_uint4(p[0] | p[1] << 16, p[2] | p[3] << 16, p[4] | p[5] << 16, p[6] | p[7] << 16);
                    sw[wave].q[n][f][0][lane] = live ? w : make_uint4(0, 0, 0, 0);
                } else {
                    uint16_t t[3][8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const float v = live ? kv8_load(a.q, a.q_f32, at + e) : 0.f;
                        split3(v, t[0][e], t[1][e], t[2][e]);
                    }
#pragma unroll
                    for (int s = 0; s < QT; ++s) sw[wave].q[n][f][s][lane] = __builtin_bit_cast(uint4, t[s]);
                }
            }
        }
        uint4 kr[4][D / 64], vr[kDt];
        float2 sc;
        bool vok;
        auto load_k = [&](int page, int sub) {
            const bool ok = static_cast<uint32_t>(page) < static_cast<uint32_t>(a.pages);
            const int64_t at = (static_cast<int64_t>(ok ? page : 0) * a.kv_heads + kvh) * (pt * D) + (sub * 16 + (lr & 3)) * D + 16 * lg;
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < D / 64; ++j) kr[i][j] = kv8_fetch<QT == 1 && NT == 1>(a.k_pool + at + i * 4 * D + j * 64);
        };
        const uint8_t* v_at;
        const float2* s_at;
        auto find_v = [&](int page, int sub) {
            vok = static_cast<uint32_t>(page) < static_cast<uint32_t>(a.pages);
            const int64_t at = static_cast<int64_t>(vok ? page : 0) * a.kv_heads + kvh;
            s_at = reinterpret_cast<const float2*>(a.scales) + at;
            v_at = a.v_pool + at * (pt * D) + static_cast<int64_t>(lr) * pt + sub * 16;
        };
        auto load_v = [&]() {
            sc = *s_at;
            in_order();
#pragma unroll
            for (int i = 0; i < kDt; ++i) vr[i] = kv8_fetch<QT == 1 && NT == 1>(v_at + static_cast<int64_t>(i) * 16 * pt);
        };
        floatx4 o[NT][kDt] = {};
        float m[NT], l[NT];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            m[n] = -INFINITY;
            l[n] = 0.f;
        }
        // A loop that waits for no load but the one it uses: loads are counted in order, so they are issued
        // in one order on every path into it, K among them without a branch (behind the last tile a page that
        // the caches hold), and page ids before the loads that may stay in flight.
        auto pages = [&](int t) {
            in_order();
            page_k = page_of(4 * t + (lr >> 2), sub_k);
            page_v = page_of(4 * t + lg, sub_v);
            in_order();
        };
        if (begin < end) {
            load_k(page_k, sub_k);
            find_v(page_v, sub_v);
            pages(min(begin + 1, end - 1));
            load_v();
            for (int t = begin;; ++t) {
                in_order();  // (and the queries stay in LDS: in registers they cost a wave a SIMD)
                floatx4 s[NT][4] = {};
                __builtin_amdgcn_s_setprio(1);  // (matrix work of one wave beside the softmax of another)
#pragma unroll
                for (int f = 0; f < kF; ++f) {
                    bf16x8 q[NT][QT];
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int e = 0; e < QT; ++e) q[n][e] = as_bf16x8(sw[wave].q[n][f][e][lane]);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const uint4& w = kr[i][f >> 1];
                        const bf16x8 k = f & 1 ? kv8_operand<FP8>(w.z, w.w) : kv8_operand<FP8>(w.x, w.y);
#pragma unroll
                        for (int n = 0; n < NT; ++n)
#pragma unroll
                            for (int e = QT - 1; e >= 0; --e) s[n][i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k, q[n][e], s[n][i], 0, 0, 0);
                    }
                }
                __builtin_amdgcn_s_setprio(0);
                const int base = t * kTile + lg * 16;  // the lane's run
                const float fk = sc.x * scale, fv = sc.y;
                in_order();
                load_k(t + 1 < end ? page_k : -1, sub_k);
                in_order();
                const bool part = t * kTile + kTile > seen_all || __any(!vok);
                uint32_t pw[NT][PT][8];
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    int live = 0;  // tokens of the run that the column sees
                    if (part) {
                        live = vok ? min(max(seen[n] - base, 0), 16) : 0;
                        asm volatile("" : "+v"(live));  // (its comparisons are not made for the tiles that need none)
#pragma unroll
                        for (int i = 0; i < 16; ++i) s[n][i / 4][i % 4] = i < live ? s[n][i / 4][i % 4] : -INFINITY;
                    }
                    float top = -INFINITY;
#pragma unroll
                    for (int i = 0; i < 16; ++i) top = fmaxf(top, s[n][i / 4][i % 4]);
                    top = top == -INFINITY ? top : top * fk;  // (nothing seen, and fk may be 0)
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
                    for (int i = 0; i < 16; ++i) w[i] = __builtin_amdgcn_exp2f(fmaf(s[n][i / 4][i % 4], fk, -ref));
                    if (part) {  // (0 * -inf, or a scale that is NaN, where nothing is seen)
#pragma unroll
                        for (int i = 0; i < 16; ++i) w[i] = i < live ? w[i] : 0.0f;
                    }
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        sum += w[i];
                        w[i] *= fv;
                    }
                    if (part) {
#pragma unroll
                        for (int i = 0; i < 16; ++i) w[i] = i < live ? w[i] : 0.0f;
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
                    const int held = vok ? min(max(u.len - base, 0), 16) : 0;
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
                __builtin_amdgcn_s_setprio(1);
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
                __builtin_amdgcn_s_setprio(0);
                if (t + 1 >= end) break;
                find_v(page_v, sub_v);
                pages(min(t + 2, end - 1));
                load_v();
            }
        }
        // the waves of a column group, joined in LDS (of four heads: each one alone, laid out for its stores)
        const int step = quads ? WAVES : groups;  // from one wave of a group to the next
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            l[n] = xor32_sum(xor16_sum(l[n]));
            if (lg == 0) sm[wave][16 * n + lr] = m[n];
        }
        __syncthreads();
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            float top = -INFINITY;
            for (int w = wave % step; w < WAVES; w += step) top = fmaxf(top, sm[w][16 * n + lr]);
            const float f = m[n] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m[n] - top);
            if (lg == 0) sl[wave][16 * n + lr] = l[n] * f;
#pragma unroll
            for (int d = 0; d < kDt; ++d) {
                const float4 v = make_float4(o[n][d][0] * f, o[n][d][1] * f, o[n][d][2] * f, o[n][d][3] * f);
                *reinterpret_cast<float4*>(&sw[wave].o[16 * n + lr][16 * d + 4 * lg]) = v;
            }
        }
        __syncthreads();
        const bool whole = count == u.tiles;
        const int slot = how.each ? group : group + u.ord;
        const int64_t part = (static_cast<int64_t>(slot) * a.kv_heads + kvh) * a.width;
        const int begin_e = quads ? lane : threadIdx.x, step_e = quads ? kWave : 64 * WAVES;
        for (int e = begin_e; e < groups * kCols * (D / 4); e += step_e) {
            const int c = e / (D / 4), d = e % (D / 4) * 4, gr = quads ? wave : c / kCols, cc = c % kCols;
            const int col = col0 + c;
            if (col >= cols) break;
            float top = -INFINITY, sum = 0.f;
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
            for (int w = gr; w < WAVES; w += step) {
                top = fmaxf(top, sm[w][cc]);
                sum += sl[w][cc];
                const float4 x = *reinterpret_cast<const float4*>(&sw[w].o[cc][d]);
                v.x += x.x; v.y += x.y; v.z += x.z; v.w += x.w;
            }
            const int i = a.row_of(col);
            if (whole) {
                kv8_store4(a, static_cast<int64_t>(u.t0 + i) * a.out_stride + static_cast<int64_t>(kvh * a.group + col - i * a.group) * D + d, v, sum);
            } else if (slot < a.slots) {  // (it is, of sequences in order)
                *reinterpret_cast<float4*>(a.part_acc + (part + c) * D + d) = v;
                if (d == 0) a.part_ml[part + c] = make_float2(top, sum);
            }
        }
        // where the join finds a row's sequence, and the sequence's pieces or tiles among all
        if (a.slot_of && tile0 == 0 && kvh == 0) {
            if (u.block == 0 && threadIdx.x == 0) a.slot_of[u.b] = make_int4(u.begin, how.each ? how.pieces(u.tiles) : u.ord, cost, how.each ? 0 : all);
            for (int e = begin_e; e < groups * kCols; e += step_e)
                if (col0 + e < cols) a.sequence_of[u.t0 + a.row_of(col0 + e)] = u.b;
        }
        if (how.each) return;
        next_unit<kCols>(a, u);
        tile0 = 0;
        count = min(u.of.tiles_before(until - u.begin), u.tiles);
        __syncthreads();  // (the sums have been read: the queries of the next unit go there)
    }
}

// The splits of a row and query head: weights 2^(m_s - M), sums in a fixed order.  D / 4 lanes to a
// split.  TOGETHER: all of a workgroup's for one row and head, so many splits at a time; else
// each D / 4 lanes for one of their own, which pays where there are many rows (519 of 32 heads,
// about 5 splits: 9 us, 30 together) and not where there are few (2 of 32 heads, 90 splits: 45 one
// after the other, 5 together).
template <int D, int WIDTH, bool TOGETHER>
__global__ __launch_bounds__(256) void attn_kv8_join_kernel(Kv8Args a) {
    constexpr int kLanes = D / 4, kWays = TOGETHER ? 256 / kLanes : 1;
    __shared__ float4 sv[kWays][kLanes];
    __shared__ float ssum[kWays], stop[kWays];
    const int at_once = TOGETHER ? 1 : 256 / kLanes;
    const int way = TOGETHER ? threadIdx.x / kLanes : 0, d = threadIdx.x % kLanes;
    const int t = blockIdx.x, h = blockIdx.y * at_once + (TOGETHER ? 0 : threadIdx.x / kLanes), kvh = h / a.group;
    if (h >= a.q_heads || (a.starts && t >= a.starts[a.batch])) return;  // (uniform where lanes work together)
    const int b = min(max(a.sequence_of[t], 0), a.batch - 1);
    const int4 at = a.slot_of[b];
    int t0, rows, len;
    a.sequence(b, t0, rows, len);
    const int i = t - t0, all_rows = rows;
    rows = min(rows, a.max_rows);
    if (i < 0 || i >= rows) return;  // (a row that no sequence computes)
    const int wide = groups_of(rows * a.group, WIDTH) * WIDTH;
    const int c = i * a.group + h - kvh * a.group, block = c / wide;
    int slot = at.x + block * at.y, splits = at.y;
    if (at.w) {
        const Shares how(a, at.w, at.z);
        const auto of = Blocks<true>::of<WIDTH>(a, all_rows, len);
        const int from = at.x + static_cast<int>(of.cost(block));
        slot = how.of(from + of.at(0));
        splits = how.of(from + of.at(of.tiles_of(block) - 1)) - slot + 1;
        slot += at.y + block;
    }
    if (splits <= 1 || slot < 0 || slot > a.slots - splits) return;
    const int64_t col = (static_cast<int64_t>(slot) * a.kv_heads + kvh) * a.width + c - block * wide, step = static_cast<int64_t>(a.kv_heads) * a.width;
    // a running maximum: the splits' own are not known before
    float top = -INFINITY, sum = 0.f;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int s = way; s < splits; s += kWays) {
        const float2 ml = a.part_ml[col + s * step];
        const float4 x = reinterpret_cast<const float4*>(a.part_acc + (col + s * step) * D)[d];
        const float to = fmaxf(top, ml.x);
        const float keep = top == to ? 1.0f : __builtin_amdgcn_exp2f(top - to);  // (-infinity for both: nothing yet)
        const float f = ml.x == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(ml.x - to);  // (NaN sums stay NaN)
        top = to;
        sum = fmaf(ml.y, f, sum * keep);
        v.x = fmaf(x.x, f, v.x * keep); v.y = fmaf(x.y, f, v.y * keep); v.z = fmaf(x.z, f, v.z * keep); v.w = fmaf(x.w, f, v.w * keep);
    }
    if constexpr (TOGETHER) {
        sv[way][d] = v;
        if (d == 0) {
            ssum[way] = sum;
            stop[way] = top;
        }
        __syncthreads();
        if (way) return;
        float all = -INFINITY;
#pragma unroll
        for (int w = 0; w < kWays; ++w) all = fmaxf(all, stop[w]);
        sum = 0.f;
        v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < kWays; ++w) {
            const float f = stop[w] == all ? 1.0f : __builtin_amdgcn_exp2f(stop[w] - all);
            const float4 x = sv[w][d];
            sum = fmaf(ssum[w], f, sum);
            v.x = fmaf(x.x, f, v.x); v.y = fmaf(x.y, f, v.y); v.z = fmaf(x.z, f, v.z); v.w = fmaf(x.w, f, v.w);
        }
    }
    kv8_store4(a, static_cast<int64_t>(t) * a.out_stride + static_cast<int64_t>(h) * D + 4 * d, v, sum);
}

namespace {

size_t up256(size_t n) { return (n + 255) & ~static_cast<size_t>(255); }

size_t kv8_bytes(const sfg_kv8_attn_args& a, int64_t slots, int width) {
    const size_t columns = static_cast<size_t>(slots) * a.kv_heads * width;
    return up256(a.batch * sizeof(int4)) + up256(a.tokens * sizeof(int)) + up256(columns * sizeof(float2)) + up256(columns * a.head_dim * sizeof(float));
}

size_t parts_bytes(const sfg_kv8_attn_args& a, size_t parts) {
    return up256(a.tokens * sizeof(int)) + up256(parts * sizeof(float2)) + up256(parts * a.head_dim * sizeof(float));
}
size_t rows_bytes(const sfg_kv8_attn_args& a, int64_t splits) { return parts_bytes(a, static_cast<size_t>(a.tokens) * a.q_heads * splits); }

constexpr int64_t kMostSlots = 1 << 22;  // workgroups of a launch: 256 threads each
constexpr size_t kMostBytes = size_t{128} << 20;  // partial results, unless the caller says how many splits
// Workgroups that tiles are dealt to: two a compute unit, all of them resident at once.  (768, where
// registers allow three: 64 sequences of up to 8192 tokens 120 us for 103, 64 with 8 rows
// 158 for 135.)  Fewer than 16 tiles for each: pieces (32 sequences of up to 2000 tokens 27 us,
// dealt 30; 64 of up to 1000 27 and 31).  A piece is a tile a wave, and two tiles where each wave walks
// them all: 256 rows over 300 tokens 25.4 us (four tiles 29.2, one 28.0), 16 fp32 rows over 8192
// 16.8 (18.6, 18.9), 64 over 3000 21.5 (19.3, 21.3).
constexpr int64_t kRound = 512;
constexpr int kFew = 16;
// Tiles of all heads from which a workgroup takes four heads, its waves never waiting for each other
// over a tile: 64 sequences of up to 2000 tokens 37.0 us for 41.3, 256 of up to 500 47.4 for 54.8, 64
// of up to 8192, 16 heads of 64 over 4, 31.6 for 36.6; with fewer the waves' share is too long: 64
// of up to 1000 29.7 for 27.6.  Few long sequences have more pieces to join for it (two of
// 131072 tokens 74.1 for 70.9), so it takes a fourth as many sequences as shares.
constexpr int kQuads = 8192;
constexpr int64_t kManyRows = 4096;  // rows by heads from which a join's lanes have one each
// Tiles up to which eight waves take a unit whole, a tile each, if every one of them has a compute
// unit: one sequence of 500 tokens 10.1 us for 11.2, 32 of up to 500 11.9 for 15.6; 64 21.3 for 21.9.
constexpr int64_t kShort = 8;

}  // namespace

// The rows kernel: splits of 128 tokens or more until there are 2048 waves.
Kv8Plan plan_rows(const sfg_kv8_attn_args& a) {
    Kv8Plan p{};
    const int64_t waves = a.tokens * a.q_heads, chunks = std::max<int64_t>((a.max_context + 63) / 64, 1);
    int64_t splits = 1;
    if (a.kv_splits > 0) splits = std::min<int64_t>({a.kv_splits, chunks, 65535});
    else
        while (waves * splits < 2048 && chunks / (2 * splits) >= 2) splits *= 2;
    // (a launch's threads and the workspace stay within bounds)
    while (splits > 1 && (waves * splits > (1 << 25) || rows_bytes(a, splits) > kMostBytes)) splits /= 2;
    p.fixed = static_cast<int>(splits);
    p.bytes = splits > 1 ? rows_bytes(a, splits) : 0;
    return p;
}

namespace {

bool mfma_dims(const sfg_kv8_attn_args& a) { return (a.head_dim == 64 || a.head_dim == 128) && a.page_tokens % 16 == 0; }
// What the matrix-core kernels' plan and the workspace follow from.
struct Kv8Sizes {
    bool narrow;
    int64_t group, cols, tiles, blocks, share;
    int nt, width;
    explicit Kv8Sizes(const sfg_kv8_attn_args& a) {
        narrow = a.q_dtype == SFG_BF16 && a.out_dtype == SFG_BF16;
        group = a.q_heads / a.kv_heads;
        cols = a.max_rows * group;
        tiles = std::max<int64_t>((a.max_context + kTile - 1) / kTile, 1);
        nt = narrow && cols > 16 ? 2 : 1;
        width = 16 * nt * (cols > 32 * nt ? 4 : cols > 16 * nt ? 2 : 1);
        blocks = a.batch + (cols > 64 * nt ? a.tokens * group / (64 * nt) : 0);  // of all sequences, at most
        share = std::max<int64_t>(kRound / a.kv_heads, 1);
    }
};

}  // namespace

Kv8Plan plan_attn_kv8(const sfg_kv8_attn_args& a) {
    if (!mfma_dims(a)) return plan_rows(a);
    Kv8Plan p{};
    const Kv8Sizes z(a);
    const bool narrow = z.narrow;
    const int64_t group = z.group, cols = z.cols, tiles = z.tiles, blocks = z.blocks;
    p.nt = z.nt;
    p.width = z.width;
    const int64_t cost = 2 * (tiles + 4);  // of a block, at most
    if (blocks * a.kv_heads > kMostSlots) return plan_rows(a);
    p.mfma = true;
    // tiles are dealt by sums of costs in 32 bits; where those of the bounds pass them, units run whole
    const bool summed = (cols / (64 * p.nt) + 1) * cost <= kMostCost && blocks * cost <= kMostCosts;
    const int64_t wide = 64 * p.nt;  // columns of a block where a sequence has several
    p.row_shift = wide % group == 0 ? std::countr_zero(static_cast<uint64_t>(wide / group)) : -1;
    p.least = std::max(64 * p.nt / p.width, 2);  // (a tile a wave; two where each walks them all)
    p.few = kFew;
    p.fixed = static_cast<int>(std::min<int64_t>({std::max(a.kv_splits, 0), tiles, kMostSlots / (blocks * a.kv_heads)}));
    p.waves = 4;
    if (!p.fixed && narrow && p.nt == 1 && tiles <= kShort && tiles > p.least && blocks * a.kv_heads <= 256) {
        p.waves = 8;
        p.fixed = 1;
    }
    if (!p.fixed && summed && tiles > p.least) {
        p.share = static_cast<int>(z.share);
        p.quads = narrow && p.nt == 1 && a.kv_heads % 4 == 0 && 4 * a.batch >= p.share ? kQuads : 0;
        const int64_t most = blocks * ((tiles + p.least - 1) / p.least);  // the shortest pieces
        p.slots = static_cast<int>(std::min(p.share * (p.quads ? 4 : 1) + blocks, most));
        p.groups = static_cast<int>(std::min(p.share + blocks, most) * a.kv_heads);
        if (kv8_bytes(a, p.slots, p.width) > kMostBytes) p.share = 0;  // (more rows: units run whole)
    }
    if (!p.share) {
        p.fixed = std::max(p.fixed, 1);
        p.slots = static_cast<int>(blocks * p.fixed);
        p.groups = static_cast<int>(p.slots * a.kv_heads);
    }
    if (p.fixed != 1) p.bytes = kv8_bytes(a, p.slots, p.width);
    return p;
}

// Plans do not grow with their bounds: fewer columns take narrower blocks and other kernels, many rows
// run whole.  The workspace does: it is what no plan of these or shorter bounds passes, each term
// growing with tokens, max_rows and max_context.  (64 sequences of up to 131072 tokens, 32 + 8 heads of
// 128: one row each 20 MiB, up to 2048 rows 98 MiB, 4096 and more 128 MiB, of which they take none.)
size_t workspace_attn_kv8(const sfg_kv8_attn_args& a) {
    const Kv8Sizes z(a);
    const bool mfma = mfma_dims(a);
    const int64_t splits = std::max(a.kv_splits, 0), units = kMostSlots / a.kv_heads;
    size_t most = 0;
    if (mfma && splits) {
        const int64_t each = std::min(splits, z.tiles);
        if (each > 1) most = kv8_bytes(a, std::min(z.blocks * each, units), z.width);
    } else if (mfma && z.tiles > 2) {
        most = kv8_bytes(a, std::min(z.share + z.blocks, z.blocks * ((z.tiles + 1) / 2)), z.width);
        if (z.narrow && z.group <= 16 && a.kv_heads % 4 == 0 && 4 * a.batch >= z.share)  // (four heads a workgroup)
            most = std::max(most, kv8_bytes(a, std::min(4 * z.share + a.batch, a.batch * ((z.tiles + 3) / 4)), 16));
        most = std::min(most, kMostBytes);
    }
    if (mfma && z.blocks * a.kv_heads <= kMostSlots) return most;
    // the rows kernel: as many splits as asked for, or until there are 2048 waves
    const int64_t chunks = (a.max_context + 63) / 64, each = splits ? std::min(splits, chunks) : chunks / 2;
    if (each < 2) return most;
    const int64_t parts = std::min<int64_t>(a.tokens * a.q_heads * each, splits ? 1 << 25 : 4096);
    return std::max(most, std::min(parts_bytes(a, parts), kMostBytes));
}

namespace {

template <int D, int WIDTH>
void launch_kv8_join(const Kv8Args& a, hipStream_t stream) {
    constexpr int kAtOnce = 256 / (D / 4);
    if (static_cast<int64_t>(a.tokens) * a.q_heads >= kManyRows)
        attn_kv8_join_kernel<D, WIDTH, false><<<dim3(static_cast<unsigned>(a.tokens), static_cast<unsigned>((a.q_heads + kAtOnce - 1) / kAtOnce)), 256, 0, stream>>>(a);
    else
        attn_kv8_join_kernel<D, WIDTH, true><<<dim3(static_cast<unsigned>(a.tokens), static_cast<unsigned>(a.q_heads)), 256, 0, stream>>>(a);
}

template <bool FP8, int D, bool P16>
void launch_kv8_mfma(const Kv8Args& a, const Kv8Plan& p, bool narrow, hipStream_t stream) {
    const dim3 grid(static_cast<unsigned>(p.groups));
    if (!narrow) attn_kv8_kernel<FP8, D, 3, 3, 1, P16, 4><<<grid, 256, 0, stream>>>(a);
    else if (p.nt == 2) attn_kv8_kernel<FP8, D, 1, 2, 2, P16, 4><<<grid, 256, 0, stream>>>(a);
    else if (p.waves == 8) attn_kv8_kernel<FP8, D, 1, 2, 1, P16, 8><<<grid, 512, 0, stream>>>(a);
    else attn_kv8_kernel<FP8, D, 1, 2, 1, P16, 4><<<grid, 256, 0, stream>>>(a);
    if (!p.bytes) return;
    if (p.nt == 2) launch_kv8_join<D, 32>(a, stream);
    else launch_kv8_join<D, 16>(a, stream);
}

template <bool FP8, int D>
void launch_kv8_pages(const Kv8Args& a, const Kv8Plan& p, bool narrow, hipStream_t stream) {
    if (a.pt == kPageTok) launch_kv8_mfma<FP8, D, true>(a, p, narrow, stream);
    else launch_kv8_mfma<FP8, D, false>(a, p, narrow, stream);
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
    a.group = a.q_heads / a.kv_heads;
    a.fixed = plan.fixed;
    if (plan.mfma && aligned) {
        a.slots = plan.slots; a.share = plan.share; a.least = plan.least; a.few = plan.few; a.quads = plan.quads;
        a.width = plan.width; a.row_shift = plan.row_shift;
        a.vec = (reinterpret_cast<uintptr_t>(s.q) & 15) == 0 && s.q_stride % 8 == 0;
        a.out_vec = (reinterpret_cast<uintptr_t>(s.out) & 15) == 0 && s.out_stride % 4 == 0;
        if (plan.bytes) {
            char* at = static_cast<char*>(workspace);
            const size_t columns = static_cast<size_t>(plan.slots) * a.kv_heads * plan.width;
            a.slot_of = reinterpret_cast<int4*>(at); at += up256(a.batch * sizeof(int4));
            a.sequence_of = reinterpret_cast<int*>(at); at += up256(a.tokens * sizeof(int));
            a.part_ml = reinterpret_cast<float2*>(at); at += up256(columns * sizeof(float2));
            a.part_acc = reinterpret_cast<float*>(at);
        }
        if (s.pool_dtype == SFG_FP8) {
            if (a.dim == 128) launch_kv8_pages<true, 128>(a, plan, narrow, stream);
            else launch_kv8_pages<true, 64>(a, plan, narrow, stream);
        } else {
            if (a.dim == 128) launch_kv8_pages<false, 128>(a, plan, narrow, stream);
            else launch_kv8_pages<false, 64>(a, plan, narrow, stream);
        }
        return;
    }
    // (pools off their boundaries: whole, in the plan's place)
    if (plan.mfma) a.fixed = 1;
    if (a.fixed > 1) {
        const size_t parts = static_cast<size_t>(a.tokens) * a.q_heads * a.fixed;
        char* at = static_cast<char*>(workspace);
        a.sequence_of = reinterpret_cast<int*>(at); at += up256(a.tokens * sizeof(int));
        a.part_ml = reinterpret_cast<float2*>(at); at += up256(parts * sizeof(float2));
        a.part_acc = reinterpret_cast<float*>(at);
        attn_kv8_rows_begin_kernel<<<dim3(static_cast<unsigned>((a.tokens + 255) / 256)), 256, 0, stream>>>(a.sequence_of, a.tokens);
    }
    const dim3 grid(static_cast<unsigned>(a.tokens), static_cast<unsigned>(a.q_heads), static_cast<unsigned>(a.fixed));
    const bool words = a.dim % 4 == 0 && a.pt % 4 == 0 && ((reinterpret_cast<uintptr_t>(s.k_pool) | reinterpret_cast<uintptr_t>(s.v_pool)) & 3) == 0;
    if (s.pool_dtype == SFG_FP8) {
        if (words) attn_kv8_rows_kernel<true, true><<<grid, 64, 0, stream>>>(a);
        else attn_kv8_rows_kernel<true, false><<<grid, 64, 0, stream>>>(a);
    } else {
        if (words) attn_kv8_rows_kernel<false, true><<<grid, 64, 0, stream>>>(a);
        else attn_kv8_rows_kernel<false, false><<<grid, 64, 0, stream>>>(a);
    }
    if (a.fixed > 1) attn_kv8_rows_join_kernel<<<dim3(static_cast<unsigned>(a.tokens), static_cast<unsigned>(a.q_heads)), 64, 0, stream>>>(a);
}

}  // namespace sfg
