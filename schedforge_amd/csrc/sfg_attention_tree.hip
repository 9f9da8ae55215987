// sfg_attention_tree.hip -- tree attention of many columns over a paged bf16 cache.
//
// The rows x group query columns of a (sequence, kv head) read the same K and V.  A
// workgroup takes up to 256 of them (32 a wave) through tiles of 64 tokens -- four pages
// -- which its waves bring into LDS by DMA, the next tiles in flight while the current
// one is multiplied:
//   S^T[64 tok][32 col] = K Q^T     2 x D/16 mfma_f32_32x32x16_bf16 (Q in registers)
//   O^T[D][32 col]     += V^T P^T   8 x D/32 of them (P in two terms)
// K row order inside a 32-token block (bits 2 and 3 of the row exchanged) makes the
// S^T accumulator the P^T operand: register r of lane l holds token 16 (r / 8) + 8 (l / 32)
// + r % 8, so a V^T fragment is eight consecutive tokens of one page's dim -- 16 bytes of
// the page as it lies in the pool.  LDS 16-byte slots are XOR-swizzled so that 16
// consecutive lanes read 16 distinct ones.
// Up to 64 columns four waves and two LDS stages, two workgroups a CU; else eight waves and
// three stages.  With up to 64, and with 65 to 128, columns two waves share each 32 and take
// every other 32-token block.
// The running maximum moves only when a tile exceeds it by more than 8 (p <= 2^8): the
// rescale of O^T runs only then.  P keeps 16 bits (split2_weights): with one rounded bf16
// term outputs were off by 2.4e-3 rms where their own rounding is 1.7e-3, at 116 us instead
// of 138 on the shape below.
//
// Sequences have lengths of their own, so the tiles of all of them are dealt evenly:
// counted through (sequence, kv head, column chunk, tile), each (sequence, kv head,
// chunk) as long as its tiles and kStart more for its start, workgroup w of W takes the
// range [N w / W, N (w + 1) / W), at most two of whose runs are parts of a longer one;
// those leave (m, l, acc) partials, and a second kernel joins them in tile order.
// 64 drafts x 4 heads a kv head, 16 x 8 kv heads x up to 8192 tokens: 121 us and 15 of the
// join once the clock has settled (up to 170 in the first milliseconds of a run).  That
// is 260 thousand cycles for 36 tiles a workgroup and its starts: the matrix pipe is 43% busy,
// and a tile's fragments, 256 KB at 128 bytes a cycle, take LDS 2048 cycles.  32 drafts,
// 8 x 8 x up to 4096: 29 and 9 us for 80 MB, the starts more of it.
//
// Tokens that some column does not see (drafts, the end, pages of no id) sit in the
// last tiles: there each lane builds the 64 bits of what its column sees, and non-finite
// values of V are replaced by zero in LDS, so that nothing hidden spreads by 0 * inf; such
// a run is marked, and the join adds those values to the columns that see them.
#include <algorithm>
#include <type_traits>

#include "sfg_chosen.hpp"

namespace sfg {

namespace {

constexpr int kTileTok = 64;
// What starting a (sequence, kv head, chunk) costs, in tiles: its queries, mask and first
// tiles are waited for, the sums before it are written (at 0, 16 x 8 heads x up to 8192
// tokens with 64 drafts take 169 us, where one workgroup has five short sequences; 138 so,
// both with the join).
constexpr int kStart = 6;
// The least length of a workgroup's range: shorter ones cost more in starts, and in parts
// to join, than they give (us at 2, 4, 5, 6 and 8; 2 x 8 heads x 8000 tokens, 64 columns:
// 40, 40, 38, 37, 38; 16 x 8 x up to 900: 27.2, 26.2, 26.3, 27.9, 30.5; 4 x 8 x up to 2000, 128
// columns: 29.3, 28.8, 27.8, 29.1, 30.9).
constexpr int kLeast = 5;

__device__ __forceinline__ int swap_bits23(int i) { return (i & ~12) | ((i & 4) << 1) | ((i & 8) >> 1); }

// The swizzle of K's 16-byte slots by row, of V's halves by dim.
template <int kD>
__device__ __forceinline__ int k_swizzle(int row) { return kD == 128 ? swap_bits23(row & 15) : (row >> 1) & 7; }
__device__ __forceinline__ int v_swizzle(int d) { return (d >> 3) & 1; }

// The value, computed where it is used: what follows from it is not hoisted out of the
// walk, whose registers it would take.
__device__ __forceinline__ int here_only(int v) {
    asm volatile("" : "+v"(v));
    return v;
}

// kStart and the tiles of sequence b (at least one).
__device__ __forceinline__ int sequence_length(const ChosenArgs& p, int b) {
    const int len = p.seq_lens ? min(max(p.seq_lens[b], 0), p.max_len) : p.max_len;
    return kStart + (len + p.rows + kTileTok - 1) / kTileTok;
}

// Where workgroup w's range begins among `total`.
__device__ __forceinline__ int64_t run_begin(int64_t total, int w, int groups) { return total * w / groups; }

// Words of a query row's mask: the first two, which most trees fit, loaded early.
__device__ __forceinline__ uint2 first_words(const ChosenArgs& p, int b, int row) {
    const uint32_t* mask = p.mask + b * p.mask_stride + static_cast<int64_t>(row) * p.mask_words;
    return make_uint2(mask[0], mask[p.mask_words > 1 ? 1 : 0]);
}

// Which of the 64 tokens from tok0 on query row `row` sees; ok: which of their pages hold tokens.
__device__ __forceinline__ uint64_t seen_bits(const ChosenArgs& p, const Unit<kChosenTree>& u, uint2 first, int row, int tok0, uint32_t ok) {
    const int t0 = tok0 - u.all_see;  // draft index of the first token
    uint64_t bits = 0;
    const int w0 = t0 >> 5;  // (rounds down)
    for (int w = w0; w <= ((t0 + 63) >> 5); ++w) {
        uint32_t word = w < 0 ? 0xFFFFFFFFu : w >= p.mask_words ? 0u : w == 0 ? first.x : w == 1 ? first.y :
                        (p.mask + u.b * p.mask_stride + static_cast<int64_t>(row) * p.mask_words)[w];
        if (w == p.mask_words - 1 && (p.rows & 31)) word &= (1u << (p.rows & 31)) - 1u;
        const int at = 32 * w - t0;
        bits |= at >= 0 ? static_cast<uint64_t>(word) << at : static_cast<uint64_t>(word) >> -at;
    }
#pragma unroll
    for (int w = 0; w < 4; ++w)
        if (!((ok >> w) & 1u)) bits &= ~(0xFFFFull << (16 * w));
    return bits;
}

template <int kD, int WC, int WAVES>
__global__ __launch_bounds__(WAVES * 64) __attribute__((amdgpu_waves_per_eu(2, 2)))
void tree_tile_kernel(ChosenArgs p, TreeRuns runs, int xcds) {
    static_assert(kD == 64 || kD == 128, "head_dim 64 or 128");
    static_assert((WAVES == 4 || WAVES == 8) && (WC == WAVES || WC == WAVES / 2), "columns over all waves or half of them");
    constexpr int kGroups = WAVES / WC;         // waves that share columns
    constexpr int kBlocks = 2 / kGroups;        // 32-token blocks of a tile per wave
    constexpr int kDb = kD / 32;                // 32-dim blocks of O^T
    constexpr int kPage = kPageTok * kD;        // elements of a page's K (or V)
    constexpr int kDma = kPage * 2 / 1024;      // 1 KB DMAs of a page
    constexpr int kSlots = kD / 8;              // 16-byte slots of a K row
    constexpr int kPart = 4 * kDma / WAVES;     // DMAs of K (and of V) per wave and tile
    constexpr int kStages = WAVES == 8 ? 3 : 2; // eight waves: the next two tiles in flight
    constexpr int kThird = kStages == 3 ? 4 * kPage : 8;
    // (an array a stage: the compiler then knows that reading one does not wait for the
    // DMAs into the others)
    __shared__ __attribute__((aligned(1024))) uint16_t sK0[4 * kPage], sK1[4 * kPage], sK2[kThird];
    __shared__ __attribute__((aligned(1024))) uint16_t sV0[4 * kPage], sV1[4 * kPage], sV2[kThird];

    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int hl = lane >> 5, l32 = lane & 31;
    const int group = wave / WC;

    // The length before each sequence (every wave counts it, 64 sequences at a time;
    // workgroup 0 leaves them for the join), then this workgroup's run.
    int total_seq = 0;
    for (int b0 = 0; b0 < runs.batch; b0 += 64) {
        const int b = b0 + lane;
        const int n = b < runs.batch ? sequence_length(p, b) : 0;
        const int upto = wave_inclusive(n) + total_seq;
        if (blockIdx.x == 0 && wave == 0 && b < runs.batch) runs.before[b + 1] = upto;
        total_seq = __builtin_amdgcn_readlane(upto, 63);
    }
    if (blockIdx.x == 0 && threadIdx.x == 0) runs.before[0] = 0;
    const int per_seq = p.kv_heads * runs.chunks;  // (kv head, chunk) pairs
    const int64_t total = static_cast<int64_t>(total_seq) * per_seq;
    const int groups = static_cast<int>(min<int64_t>(runs.groups, max<int64_t>(total / runs.least, 1)));
    // consecutive workgroup ids go to the XCDs in turn: each XCD gets consecutive runs, so
    // that the chunks of a (sequence, kv head) read K and V through one L2
    const int grid = static_cast<int>(gridDim.x), bid = static_cast<int>(blockIdx.x);
    const int full = grid - grid % xcds;
    const int w = bid < full ? (bid % xcds) * (full / xcds) + bid / xcds : bid;
    if (w >= groups) return;
    int64_t x = run_begin(total, w, groups);
    const int64_t x_end = run_begin(total, w + 1, groups);
    // its first sequence: the last one with no more length before it than x / per_seq
    int b = 0, pair, skip;
    {
        const int y = static_cast<int>(x / per_seq);
        int before = 0, base = 0;
        for (int b0 = 0; b0 < runs.batch; b0 += 64) {
            const int bb = b0 + lane;
            const int n = bb < runs.batch ? sequence_length(p, bb) : 0;
            const int upto = wave_inclusive(n) + base;
            const uint64_t here = __ballot(bb < runs.batch && upto - n <= y && y < upto);
            if (here) {
                const int at = __ffsll(static_cast<unsigned long long>(here)) - 1;
                b = b0 + at;
                before = __builtin_amdgcn_readlane(upto - n, at);
                break;
            }
            base = __builtin_amdgcn_readlane(upto, 63);
        }
        const int64_t rest = x - static_cast<int64_t>(before) * per_seq;
        const int n = sequence_length(p, b);
        pair = static_cast<int>(rest / n);
        skip = static_cast<int>(rest % n);  // of that (sequence, kv head, chunk)'s length
    }

    for (int run = 0; x < x_end;) {
    const Unit<kChosenTree> u = unit_of<kChosenTree>(p, b, pair / runs.chunks);
    const int chunk = pair % runs.chunks;
    const int col = chunk * (32 * WC) + (wave % WC) * 32 + l32;
    const bool has = col < u.cols;
    int row, head;
    column_of<kChosenTree>(p, u, has ? col : 0, row, head);

    const int pages = (u.walk + kPageTok - 1) / kPageTok;
    const int all_tiles = (pages + 3) / 4;
    const int upto = static_cast<int>(min<int64_t>(all_tiles + kStart, skip + (x_end - x)));
    const int tile = max(skip - kStart, 0), tiles = upto - kStart - tile;
    x += upto - skip;
    if (tiles <= 0) break;  // the range ends within a start
    const int begin = 4 * tile, end = min(pages, begin + 4 * tiles);
    const bool whole = tiles == all_tiles;

    const uint2 mask2 = first_words(p, u.b, row);
    // Q^T fragments: this lane's column, dims 16 s + 8 hl + [0, 8)
    bf16x8 qf[kD / 16];
    {
        const uint16_t* qr = static_cast<const uint16_t*>(p.q) + column_offset(p, u.b, row, head) + 8 * hl;
#pragma unroll
        for (int s = 0; s < kD / 16; ++s) qf[s] = as_bf16x8(*reinterpret_cast<const uint4*>(qr + 16 * s));
    }

    const int32_t* table = p.page_table + static_cast<int64_t>(u.b) * p.pages_per_seq;
    const int64_t page_stride = static_cast<int64_t>(kPage) * p.kv_heads;
    const uint16_t* kpool = static_cast<const uint16_t*>(p.k_pool) + static_cast<int64_t>(u.kvh) * kPage;
    const uint16_t* vpool = static_cast<const uint16_t*>(p.v_pool) + static_cast<int64_t>(u.kvh) * kPage;
    // byte offsets inside a page of what this wave's DMAs' lanes bring: K slot s of a row
    // holds its vector s ^ swizzle, V's two halves of a dim lie in swizzled order
    const int my_page = wave * kPart / kDma, first_dma = wave * kPart % kDma;
    uint32_t k_off[kPart], v_off[kPart];
#pragma unroll
    for (int n = 0; n < kPart; ++n) {
        const int r = (first_dma + n) * (64 / kSlots) + lane / kSlots, slot = lane % kSlots;
        k_off[n] = static_cast<uint32_t>(r * kD + (slot ^ k_swizzle<kD>(r)) * 8) * 2;
        const int d = 32 * (first_dma + n) + (lane >> 1);
        v_off[n] = static_cast<uint32_t>(d * kPageTok + ((lane & 1) ^ v_swizzle(d)) * 8) * 2;
    }
    // page ids 64 at a time, one per lane, and which of them are in the pool; the others
    // read page 0 and are hidden
    int ids = 0, ids_base = begin - 64;
    uint64_t ids_ok = 0;
    // This wave's share of a tile (past the last one: of the last one again, into a stage
    // nobody reads, so that every tile issues the same number of loads).  Returns which of
    // its four pages hold tokens.
    auto issue = [&](uint16_t* dk, uint16_t* dv, int tile_at) __attribute__((always_inline)) {
        const int pg = begin + 4 * min(tile_at, tiles - 1);
        if (pg - ids_base >= 64) {  // wave-uniform; a tile's four pages never straddle this
            ids_base = pg;
            const int id = table[min(pg + lane, end - 1)];
            const bool good = pg + lane < end && id >= 0 && id < p.num_pages;
            ids = good ? id : 0;
            ids_ok = __ballot(good);
        }
        const uint32_t ok = static_cast<uint32_t>(ids_ok >> (pg - ids_base)) & 15u;
        const int mine = __builtin_amdgcn_readlane(ids, pg - ids_base + my_page);
        const buf_rsrc rk = make_rsrc(kpool + mine * page_stride, kPage * 2), rv = make_rsrc(vpool + mine * page_stride, kPage * 2);
#pragma unroll
        for (int n = 0; n < kPart; ++n) lds_dma16_buf(rk, k_off[n], dk + (wave * kPart + n) * 512);
#pragma unroll
        for (int n = 0; n < kPart; ++n) lds_dma16_buf(rv, v_off[n], dv + (wave * kPart + n) * 512);
        return ok;
    };

    floatx16 acc[kDb];
#pragma unroll
    for (int i = 0; i < kDb; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[i][r] = 0.f;
    float m_run = -INFINITY, l_run = 0.f;
    uint32_t non_finite = 0;  // non-zero: some were left out
    const float c = p.scale_log2;
    // a tile with tokens that some column does not see; the same for all waves
    auto is_partial = [&](int tile_at, uint32_t ok) { return ok != 15u || (begin + 4 * tile_at + 4) * kPageTok > u.all_see; };
    // Non-finite values of a partial tile become zero, and are marked: each lane looks at
    // what its own DMAs brought, before the barrier that lets the other waves read it.
    auto clean = [&](uint16_t* tv) __attribute__((always_inline)) {
#pragma unroll
        for (int n = 0; n < kPart; ++n) {
            uint4* at = reinterpret_cast<uint4*>(tv + (wave * kPart + n) * 512) + here_only(lane);
            const uint4 v = *at;
            const uint4 f = make_uint4(finite_bf16x2(v.x), finite_bf16x2(v.y), finite_bf16x2(v.z), finite_bf16x2(v.w));
            non_finite |= (f.x ^ v.x) | (f.y ^ v.y) | (f.z ^ v.z) | (f.w ^ v.w);
            *at = f;
        }
        wait_lds();
    };
    auto compute = [&](const uint16_t* tk, const uint16_t* tv, int tile_at, uint32_t ok) __attribute__((always_inline)) {
        const int tok0 = (begin + 4 * tile_at) * kPageTok;
        const bool partial = is_partial(tile_at, ok);
        uint64_t bits = ~0ull;
        if (partial) bits = seen_bits(p, u, mask2, here_only(row), tok0, ok);
        floatx16 s[kBlocks];
#pragma unroll
        for (int j = 0; j < kBlocks; ++j) {
            const int blk = kGroups == 1 ? j : group;
#pragma unroll
            for (int r = 0; r < 16; ++r) s[j][r] = 0.f;
            const int kr = 32 * blk + swap_bits23(l32);
#pragma unroll
            for (int st = 0; st < kD / 16; ++st) {
                const bf16x8 kf = as_bf16x8(*reinterpret_cast<const uint4*>(
                    &tk[kr * kD + ((2 * st + hl) ^ k_swizzle<kD>(kr & 15)) * 8]));
                s[j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf, qf[st], s[j], 0, 0, 0);
            }
        }
        if (partial)
#pragma unroll
            for (int j = 0; j < kBlocks; ++j) {
                const uint32_t mine = static_cast<uint32_t>(bits >> (kGroups == 1 ? 32 * j : 32 * group)) >> here_only(8 * hl);
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    if (!((mine >> (16 * (r >> 3) + (r & 7))) & 1u)) s[j][r] = -INFINITY;
            }
        float tmax = s[0][0];
#pragma unroll
        for (int j = 0; j < kBlocks; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) tmax = fmaxf(tmax, s[j][r]);
        tmax = xor32_max(tmax) * c;
        const bool upd = tmax > m_run + 8.0f;
        if (__builtin_amdgcn_ballot_w64(upd)) {
            const float m_new = upd ? tmax : m_run;
            const float alpha = upd ? fast_exp2(m_run - m_new) : 1.0f;
            l_run *= alpha;
#pragma unroll
            for (int i = 0; i < kDb; ++i)
#pragma unroll
                for (int r = 0; r < 16; ++r) acc[i][r] *= alpha;
            m_run = m_new;
        }
        const float nm = m_run == -INFINITY ? 0.f : -m_run;
        bf16x8 pf[kBlocks][2][2];
#pragma unroll
        for (int j = 0; j < kBlocks; ++j)
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                float pv[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    pv[e] = fast_exp2(fmaf(s[j][8 * t + e], c, nm));
                    l_run += pv[e];
                }
                uint4 hi, lo;
                split2_weights(pv[0], pv[1], hi.x, lo.x);
                split2_weights(pv[2], pv[3], hi.y, lo.y);
                split2_weights(pv[4], pv[5], hi.z, lo.z);
                split2_weights(pv[6], pv[7], hi.w, lo.w);
                pf[j][t][0] = as_bf16x8(hi);
                pf[j][t][1] = as_bf16x8(lo);
            }
#pragma unroll
        for (int j = 0; j < kBlocks; ++j)
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const int pg = 2 * (kGroups == 1 ? j : group) + t;
                bf16x8 vf[kDb];
#pragma unroll
                for (int i = 0; i < kDb; ++i) {
                    const int d = 32 * i + l32;
                    vf[i] = as_bf16x8(*reinterpret_cast<const uint4*>(
                        &tv[pg * kPage + d * kPageTok + (hl ^ v_swizzle(d)) * 8]));
                }
#pragma unroll
                for (int x = 1; x >= 0; --x)  // (the smaller terms first)
#pragma unroll
                    for (int i = 0; i < kDb; ++i)
                        acc[i] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf[i], pf[j][t][x], acc[i], 0, 0, 0);
            }
    };

    if constexpr (kStages == 3) {
        // Tile t: its own loads are done (tile t + 1's stay in flight), every wave is past
        // tile t - 1, whose stage the loads of tile t + 2 then take.
        uint32_t ok0 = issue(sK0, sV0, 0), ok1 = issue(sK1, sV1, 1), ok2 = 0;
        auto step = [&](const uint16_t* tk, uint16_t* tv, uint16_t* nk, uint16_t* nv, int t, uint32_t ok, uint32_t& next) __attribute__((always_inline)) {
            wait_vmem_lds<2 * kPart>();
            if (is_partial(t, ok)) clean(tv);
            barrier_no_fence();
            next = issue(nk, nv, t + 2);
            compute(tk, tv, t, ok);
            return t + 1 < tiles;
        };
        for (int t = 0;; t += 3) {
            if (!step(sK0, sV0, sK2, sV2, t, ok0, ok2)) break;
            if (!step(sK1, sV1, sK0, sV0, t + 1, ok1, ok0)) break;
            if (!step(sK2, sV2, sK1, sV1, t + 2, ok2, ok1)) break;
        }
    } else {
        uint32_t ok0 = issue(sK0, sV0, 0), ok1 = 0;
        for (int t = 0;; t += 2) {
            wait_vmem_lds<0>();
            if (is_partial(t, ok0)) clean(sV0);
            barrier_no_fence();
            ok1 = issue(sK1, sV1, t + 1);
            compute(sK0, sV0, t, ok0);
            if (t + 1 >= tiles) break;
            wait_vmem_lds<0>();
            if (is_partial(t + 1, ok1)) clean(sV1);
            barrier_no_fence();
            ok0 = issue(sK0, sV0, t + 2);
            compute(sK1, sV1, t + 1, ok1);
            if (t + 2 >= tiles) break;
        }
    }
    wait_vmem_all();
    __syncthreads();
    l_run += __shfl_xor(l_run, 32, 64);
    // acc: this lane's column, dims 32 i + 8 cc + 4 hl + [0, 4)
    const int at = here_only(lane);
    if constexpr (kGroups == 2) {
        // the second wave of a column block hands its sums over
        // (a stage's K or V holds the sums of one block: 32 columns x D, 4 bytes each)
        static_assert(sizeof sK0 == 32 * kD * 4 && sizeof sV0 == sizeof sK0, "a block's sums fit a stage");
        const int cb = wave % WC;
        float* hand = reinterpret_cast<float*>(cb == 0 ? sK0 : cb == 1 ? sK1 : cb == 2 ? sV0 : sV1);
        __shared__ float ml[2 * WC * 64];
        if (group == 1) {
#pragma unroll
            for (int i = 0; i < kDb; ++i)
#pragma unroll
                for (int r = 0; r < 16; ++r) hand[(16 * i + r) * 64 + at] = acc[i][r];
            ml[(2 * cb) * 64 + at] = m_run;
            ml[(2 * cb + 1) * 64 + at] = l_run;
        }
        __syncthreads();
        if (group == 0) {
            const float m2 = ml[(2 * cb) * 64 + at], l2 = ml[(2 * cb + 1) * 64 + at];
            const float M = fmaxf(m_run, m2);
            const float f1 = split_weight(m_run, M), f2 = split_weight(m2, M);
            l_run = l_run * f1 + l2 * f2;
            m_run = M;
#pragma unroll
            for (int i = 0; i < kDb; ++i)
#pragma unroll
                for (int r = 0; r < 16; ++r) acc[i][r] = acc[i][r] * f1 + hand[(16 * i + r) * 64 + at] * f2;
        }
        __syncthreads();  // (the next run's DMA lands here)
    }
    non_finite = __syncthreads_or(non_finite != 0);
    if (threadIdx.x == 0) {
        if (whole) runs.unit_flags[u.id * runs.chunks + chunk] = non_finite;
        else runs.part_flags[2 * w + (run > 0 ? 1 : 0)] = non_finite;
    }
    if (has && group == 0 && whole) {
        const float inv = 1.0f / l_run;  // nothing visible: 0 * inf
        uint16_t* o = static_cast<uint16_t*>(p.out) + column_offset(p, u.b, here_only(row), here_only(head));
#pragma unroll
        for (int i = 0; i < kDb; ++i)
#pragma unroll
            for (int cc = 0; cc < 4; ++cc)
                *reinterpret_cast<uint2*>(o + 32 * i + 8 * cc + 4 * (at >> 5)) =
                    make_uint2(cvt_pk_bf16(acc[i][4 * cc] * inv, acc[i][4 * cc + 1] * inv),
                               cvt_pk_bf16(acc[i][4 * cc + 2] * inv, acc[i][4 * cc + 3] * inv));
    } else if (has && group == 0) {
        // part 0 of the workgroup: its first run, part 1: its last
        const int64_t part = (2 * static_cast<int64_t>(w) + (run > 0 ? 1 : 0)) * (32 * WC) + (wave % WC) * 32 + (at & 31);
#pragma unroll
        for (int i = 0; i < kDb; ++i)
#pragma unroll
            for (int cc = 0; cc < 4; ++cc)
                *reinterpret_cast<float4*>(p.part_acc + part * kD + 32 * i + 8 * cc + 4 * (at >> 5)) =
                    make_float4(acc[i][4 * cc], acc[i][4 * cc + 1], acc[i][4 * cc + 2], acc[i][4 * cc + 3]);
        if (at < 32) reinterpret_cast<float2*>(p.part_ml)[part] = make_float2(m_run, l_run);
    }
    ++run;
    skip = 0;
    if (++pair == per_seq) {
        pair = 0;
        ++b;
    }
    }  // runs
}

// Infinities and NaN among the values of tiles that not every column sees whole: a
// positive weight times one is that value, whatever the weight.
template <int kD>
__device__ __forceinline__ float2 add_non_finite(const ChosenArgs& p, const Unit<kChosenTree>& u, int row, int lane, float2 o) {
    constexpr int kW = kD / 64;
    const int32_t* table = p.page_table + static_cast<int64_t>(u.b) * p.pages_per_seq;
    const int pages = (u.walk + kPageTok - 1) / kPageTok;
    for (int pg = 0; pg < pages; pg += 4) {
        uint32_t ok = 0;
        for (int w = 0; w < 4 && pg + w < pages; ++w) {
            const int id = table[pg + w];
            ok |= id >= 0 && id < p.num_pages ? 1u << w : 0u;
        }
        if (ok == 15u && pg * kPageTok + kTileTok <= u.all_see) continue;
        const uint64_t bits = seen_bits(p, u, first_words(p, u.b, row), row, pg * kPageTok, ok);
        for (int x = 0; x < kTileTok; ++x) {
            if (!((bits >> x) & 1u)) continue;
            const uint16_t* v = static_cast<const uint16_t*>(p.v_pool) +
                                ((static_cast<int64_t>(table[pg + (x >> 4)]) * p.kv_heads + u.kvh) * kD + kW * lane) * kPageTok + (x & 15);
            if ((v[0] & 0x7F80u) == 0x7F80u) o.x += bf16_to_f32(v[0]);
            if (kW == 2 && (v[kPageTok] & 0x7F80u) == 0x7F80u) o.y += bf16_to_f32(v[kPageTok]);
        }
    }
    return o;
}

// Joins the parts of the (sequence, kv head, chunk)s that more than one workgroup
// walked, in tile order: a wave takes four columns side by side (their loads together in
// flight), lane l the dims kD / 64 l + [0, kD / 64).  Four parts a batch: eight load more
// than the usual two or three (30 us against 19 on the shape above).
template <int kD>
__global__ __launch_bounds__(256) void tree_join_kernel(ChosenArgs p, TreeRuns runs, int col_groups) {
    constexpr int kW = kD / 64, kCols = 4, kBatch = 4;
    const int lane = threadIdx.x & 63;
    const int item = blockIdx.x * 4 + (threadIdx.x >> 6);  // (sequence, kv head, four columns)
    if (item >= col_groups * p.kv_heads * runs.batch) return;
    const int uid = item / col_groups, col0 = item % col_groups * kCols;
    const int per_seq = p.kv_heads * runs.chunks;
    const Unit<kChosenTree> u = unit_of<kChosenTree>(p, uid / p.kv_heads, uid % p.kv_heads);
    const int chunk = col0 / runs.cols;  // (a chunk is a multiple of four columns)
    const int64_t total = static_cast<int64_t>(runs.before[runs.batch]) * per_seq;
    const int groups = static_cast<int>(min<int64_t>(runs.groups, max<int64_t>(total / runs.least, 1)));
    const int before = runs.before[u.b], n = runs.before[u.b + 1] - before;
    const int64_t first = static_cast<int64_t>(before) * per_seq + static_cast<int64_t>(u.kvh * runs.chunks + chunk) * n;
    // the workgroup of position x: the last whose range begins at or before it
    const int w0 = static_cast<int>(((first + kStart + 1) * groups - 1) / total);
    const int w1 = static_cast<int>(((first + n) * groups - 1) / total);
    const bool direct = w0 == w1;  // written where it was walked
    int flag = direct ? runs.unit_flags[u.id * runs.chunks + chunk] : 0;
    if (direct && !flag) return;
    float M[kCols], L[kCols];
    float2 o[kCols];
#pragma unroll
    for (int c = 0; c < kCols; ++c) {
        M[c] = -INFINITY;
        L[c] = 0.f;
        o[c] = make_float2(0.f, 0.f);
    }
    if (!direct)
        for (int wb = w0; wb <= w1; wb += kBatch) {
            float2 ml[kBatch][kCols], av[kBatch][kCols];
#pragma unroll
            for (int e = 0; e < kBatch; ++e) {
                const int w = min(wb + e, w1);
                // its last run where it begins before this unit, else its first
                const int64_t run = 2 * static_cast<int64_t>(w) + (run_begin(total, w, groups) < first ? 1 : 0);
                const int64_t part = run * runs.cols + col0 % runs.cols;
                flag |= runs.part_flags[run];
#pragma unroll
                for (int c = 0; c < kCols; ++c) {  // (columns past the unit's are parts that nobody wrote, and are not kept)
                    ml[e][c] = reinterpret_cast<const float2*>(p.part_ml)[part + c];
                    if constexpr (kW == 2) av[e][c] = reinterpret_cast<const float2*>(p.part_acc)[(part + c) * 64 + lane];
                    else av[e][c] = make_float2(p.part_acc[(part + c) * 64 + lane], 0.f);
                }
            }
#pragma unroll
            for (int c = 0; c < kCols; ++c) {
                float m = M[c];
#pragma unroll
                for (int e = 0; e < kBatch; ++e) m = fmaxf(m, ml[e][c].x);
                const float f = split_weight(M[c], m);
                L[c] *= f;
                o[c].x *= f;
                o[c].y *= f;
#pragma unroll
                for (int e = 0; e < kBatch; ++e) {
                    if (wb + e > w1) continue;
                    const float g = split_weight(ml[e][c].x, m);
                    L[c] = fmaf(ml[e][c].y, g, L[c]);
                    o[c].x = fmaf(g, av[e][c].x, o[c].x);
                    o[c].y = fmaf(g, av[e][c].y, o[c].y);
                }
                M[c] = m;
            }
        }
#pragma unroll
    for (int c = 0; c < kCols; ++c) {
        if (col0 + c >= u.cols) continue;
        int row, head;
        column_of<kChosenTree>(p, u, col0 + c, row, head);
        uint16_t* out = static_cast<uint16_t*>(p.out) + column_offset(p, u.b, row, head) + kW * lane;
        float2 v = make_float2(o[c].x / L[c], o[c].y / L[c]);  // nothing visible: 0 / 0
        if (direct) v = make_float2(bf16_to_f32(out[0]), bf16_to_f32(out[kW - 1]));
        if (flag) v = add_non_finite<kD>(p, u, row, lane, v);
        if constexpr (kW == 2) *reinterpret_cast<uint32_t*>(out) = cvt_pk_bf16(v.x, v.y);
        else *out = f32_to_bf16(v.x);
    }
}

}  // namespace

TreeTiles plan_tree_tiles(int64_t batch, int64_t kv_heads, int64_t cols, int64_t head_dim, int64_t keys, int32_t requested) {
    TreeTiles t{};
    t.waves = cols <= 64 ? 4 : 8;
    t.col_waves = cols <= 64 ? 2 : cols <= 128 ? 4 : 8;
    t.cols = 32 * t.col_waves;
    t.chunks = (cols + t.cols - 1) / t.cols;
    const int64_t units = batch * kv_heads * t.chunks, tiles = (keys + kTileTok - 1) / kTileTok;
    // Against the 16-column kernel, which reads K and V once per 16 columns but starts sooner:
    // by the bytes that one reads.  64 columns: 1 x 8 kv heads x 8000 tokens 23 us there,
    // 36 here, 2 x 8 x 8000 32 and 38; 16 x 8 x up to 900 31 and 26; 128 columns: 4 x 8 x up to
    // 2000 33 and 28, 16 x 4 heads of 64 dims x up to 900 17 and 21, 16 x 8 x up to 8000 224 and
    // 83.  Over 516 random trees of 150 K to 6 M such reads the choice is 4% slower than the
    // better kernel of each on average (3% from 500 K on), 2.0 times at worst; by the tile
    // kernel alone 18%, by the other alone 21%.
    if (cols < 8) return t;
    const int64_t reads = (cols + 15) / 16 * batch * kv_heads * tiles * head_dim;
    if (requested <= 0 && reads < 960 * 1024) return t;
    if ((tiles + kStart) * batch > 0x7FFFFFFF || units * tiles > (int64_t{1} << 40)) return t;  // 64-bit products with groups
    // eight waves fill a CU (two a SIMD), four half of one; a requested count is that many a unit
    t.least = requested > 0 ? 1 : kLeast;
    t.groups = std::min<int64_t>(requested > 0 ? std::min<int64_t>(units * requested, 1024) : t.waves == 8 ? 256 : 512, units * tiles);
    const size_t parts = 2 * static_cast<size_t>(t.groups) * t.cols;
    // the length before each sequence; marks of the whole units and of the parts
    t.before_bytes = (static_cast<size_t>(batch + 1 + units + 2 * t.groups) * sizeof(int32_t) + 255) / 256 * 256;
    t.ml_bytes = (parts * 2 * sizeof(float) + 255) / 256 * 256;
    t.acc_bytes = parts * head_dim * sizeof(float);
    return t;
}

void launch_tree_tiles(ChosenArgs p, const TreeTiles& t, int64_t batch, void* workspace, hipStream_t stream) {
    char* ws = static_cast<char*>(workspace);
    TreeRuns r{};
    r.before = reinterpret_cast<int32_t*>(ws);
    r.unit_flags = r.before + batch + 1;
    r.part_flags = r.unit_flags + batch * p.kv_heads * t.chunks;
    r.batch = static_cast<int>(batch);
    r.chunks = static_cast<int>(t.chunks);
    r.cols = t.cols;
    r.groups = static_cast<int>(t.groups);
    r.least = t.least;
    p.part_ml = reinterpret_cast<float*>(ws + t.before_bytes);
    p.part_acc = reinterpret_cast<float*>(ws + t.before_bytes + t.ml_bytes);
    const unsigned grid = static_cast<unsigned>(t.groups);
    const int xcds = device_xcds(stream);
    const int64_t cols = static_cast<int64_t>(p.q_heads / p.kv_heads) * p.rows, col_groups = (cols + 3) / 4;
    const unsigned joins = static_cast<unsigned>((batch * p.kv_heads * col_groups + 3) / 4);
    if (p.head_dim == 128) {
        if (t.col_waves == 8) tree_tile_kernel<128, 8, 8><<<grid, 512, 0, stream>>>(p, r, xcds);
        else if (t.col_waves == 4) tree_tile_kernel<128, 4, 8><<<grid, 512, 0, stream>>>(p, r, xcds);
        else tree_tile_kernel<128, 2, 4><<<grid, 256, 0, stream>>>(p, r, xcds);
        tree_join_kernel<128><<<joins, 256, 0, stream>>>(p, r, static_cast<int>(col_groups));
    } else {
        if (t.col_waves == 8) tree_tile_kernel<64, 8, 8><<<grid, 512, 0, stream>>>(p, r, xcds);
        else if (t.col_waves == 4) tree_tile_kernel<64, 4, 8><<<grid, 512, 0, stream>>>(p, r, xcds);
        else tree_tile_kernel<64, 2, 4><<<grid, 256, 0, stream>>>(p, r, xcds);
        tree_join_kernel<64><<<joins, 256, 0, stream>>>(p, r, static_cast<int>(col_groups));
    }
}

}  // namespace sfg
