// sfg_attention_tree.hip -- tree attention of many columns over a paged bf16 cache.
//
// The rows x group query columns of a (sequence, kv head) read the same K and V.  A
// workgroup of four waves owns up to 128 of them (32 a wave) and one split of the
// tokens, and walks tiles of 64 tokens -- four pages -- which its waves bring into LDS
// by DMA, one page's K and V each, the next tile in flight while the current one is
// multiplied:
//   S^T[64 tok][32 col] = K Q^T     2 x D/16 mfma_f32_32x32x16_bf16 (Q in registers)
//   O^T[D][32 col]     += V^T P^T   4 x D/32 of them
// K row order inside a 32-token block (bits 2 and 3 of the row exchanged) makes the
// S^T accumulator the P^T operand: register r of lane l holds token 16 (r / 8) + 8 (l / 32)
// + r % 8, so a V^T fragment is eight consecutive tokens of one page's dim -- 16 bytes of
// the page as it lies in the pool.  LDS 16-byte slots are XOR-swizzled so that 16
// consecutive lanes read 16 distinct ones.
// With at most 64 columns, two waves share each 32 and take every other 32-token block.
// The running maximum moves only when a tile exceeds it by more than 8 (p <= 2^8): the
// rescale of O^T runs only then.  P is rounded to bf16 once (2^-8 of each weight).
//
// Tokens that some column does not see (drafts, the end, pages of no id) sit in the
// last tiles: there each lane builds the 64 bits of what its column sees, V past the
// end is zeroed in LDS, and a tile with a non-finite value left is taken token by token,
// so that nothing hidden is multiplied, not even by zero.
#include "sfg_chosen.hpp"

namespace sfg {

namespace {

constexpr int kTileTok = 64;

__device__ __forceinline__ int swap_bits23(int i) { return (i & ~12) | ((i & 4) << 1) | ((i & 8) >> 1); }

// The swizzle of K's 16-byte slots by row, of V's halves by dim.
template <int kD>
__device__ __forceinline__ int k_swizzle(int row) { return kD == 128 ? swap_bits23(row & 15) : (row >> 1) & 7; }
__device__ __forceinline__ int v_swizzle(int d) { return (d >> 3) & 1; }

template <int kD, int WC>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2, 2)))
void tree_tile_kernel(ChosenArgs p, int chunks, int xcds) {
    static_assert(kD == 64 || kD == 128, "head_dim 64 or 128");
    static_assert(WC == 4 || WC == 2, "columns over four waves or two");
    constexpr int kGroups = 4 / WC;             // waves that share columns
    constexpr int kBlocks = 2 / kGroups;        // 32-token blocks of a tile per wave
    constexpr int kDb = kD / 32;                // 32-dim blocks of O^T
    constexpr int kPage = kPageTok * kD;        // elements of a page's K (or V)
    constexpr int kDma = kPage * 2 / 1024;      // 1 KB DMAs of a page
    constexpr int kSlots = kD / 8;              // 16-byte slots of a K row
    __shared__ __attribute__((aligned(1024))) uint16_t sK[2][4 * kPage];
    __shared__ __attribute__((aligned(1024))) uint16_t sV[2][4 * kPage];

    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int hl = lane >> 5, l32 = lane & 31;
    // consecutive workgroup ids go to the XCDs in turn: each XCD gets a contiguous run of
    // (unit, split, chunk), so that the chunks of a split read K and V through one L2
    const int total_groups = static_cast<int>(gridDim.x), bid = static_cast<int>(blockIdx.x);
    const int full = total_groups - total_groups % xcds;
    const int item = bid < full ? (bid % xcds) * (full / xcds) + bid / xcds : bid;
    const int chunk = item % chunks, split = item / chunks % p.splits, uid = item / chunks / p.splits;
    const Unit<kChosenTree> u = unit_of<kChosenTree>(p, uid / p.kv_heads, uid % p.kv_heads);
    const int col = chunk * (32 * WC) + (wave % WC) * 32 + l32;
    const int group = wave / WC;
    const bool has = col < u.cols;
    int row, head;
    column_of<kChosenTree>(p, u, has ? col : 0, row, head);

    const int pages = (u.walk + kPageTok - 1) / kPageTok;
    const int begin = static_cast<int>(static_cast<int64_t>(pages) * split / p.splits);
    const int end = static_cast<int>(static_cast<int64_t>(pages) * (split + 1) / p.splits);
    const int tiles = (end - begin + 3) / 4;

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
    // byte offsets inside a page of what each DMA's lanes bring: K slot s of a row holds
    // its vector s ^ swizzle, V's two halves of a dim lie in swizzled order
    uint32_t k_off[kDma], v_off[kDma];
#pragma unroll
    for (int n = 0; n < kDma; ++n) {
        const int r = n * (64 / kSlots) + lane / kSlots, slot = lane % kSlots;
        k_off[n] = static_cast<uint32_t>(r * kD + (slot ^ k_swizzle<kD>(r)) * 8) * 2;
        const int d = 32 * n + (lane >> 1);
        v_off[n] = static_cast<uint32_t>(d * kPageTok + ((lane & 1) ^ v_swizzle(d)) * 8) * 2;
    }
    // page ids 64 at a time, one per lane; ids outside the pool read page 0 and are hidden
    int ids = 0, ids_base = begin - 64;
    auto page_id = [&](int pg) __attribute__((always_inline)) {
        if (pg - ids_base >= 64) {  // wave-uniform; tiles start at multiples of four pages from ids_base
            ids_base = begin + (pg - begin) / 4 * 4;
            ids = ids_base + lane < end ? table[ids_base + lane] : -1;
        }
        return __builtin_amdgcn_readlane(ids, pg - ids_base);
    };
    // wave w brings page w of the tile; returns which of its four pages hold tokens
    auto issue = [&](int stage, int tile) __attribute__((always_inline)) {
        const int pg = begin + 4 * tile;
        uint32_t ok = 0;
        int mine = 0;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const int id = pg + w < end ? page_id(pg + w) : -1;
            const bool good = id >= 0 && id < p.num_pages;
            ok |= good ? 1u << w : 0u;
            if (w == wave) mine = good ? id : 0;
        }
        const buf_rsrc rk = make_rsrc(kpool + mine * page_stride, kPage * 2), rv = make_rsrc(vpool + mine * page_stride, kPage * 2);
#pragma unroll
        for (int n = 0; n < kDma; ++n) lds_dma16_buf(rk, k_off[n], sK[stage] + wave * kPage + n * 512);
#pragma unroll
        for (int n = 0; n < kDma; ++n) lds_dma16_buf(rv, v_off[n], sV[stage] + wave * kPage + n * 512);
        return ok;
    };

    floatx16 acc[kDb];
#pragma unroll
    for (int i = 0; i < kDb; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[i][r] = 0.f;
    float m_run = -INFINITY, l_run = 0.f;
    const float c = p.scale_log2;
    const uint32_t* mask = p.mask + u.b * p.mask_stride + static_cast<int64_t>(row) * p.mask_words;

    // which of a tile's 64 tokens the lane's column sees
    auto seen_bits = [&](int tok0, uint32_t ok) {
        const int t0 = tok0 - u.all_see;  // draft index of the tile's first token
        uint64_t bits = 0;
        const int w0 = t0 >> 5;  // (rounds down)
        for (int w = w0; w <= ((t0 + 63) >> 5); ++w) {
            uint32_t word = w < 0 ? 0xFFFFFFFFu : w < p.mask_words ? mask[w] : 0u;
            if (w == p.mask_words - 1 && (p.rows & 31)) word &= (1u << (p.rows & 31)) - 1u;
            const int at = 32 * w - t0;
            bits |= at >= 0 ? static_cast<uint64_t>(word) << at : static_cast<uint64_t>(word) >> -at;
        }
#pragma unroll
        for (int w = 0; w < 4; ++w)
            if (!((ok >> w) & 1u)) bits &= ~(0xFFFFull << (16 * w));
        return bits;
    };

    auto compute = [&](int stage, int tile, uint32_t ok) __attribute__((always_inline)) {
        const int tok0 = (begin + 4 * tile) * kPageTok;
        const bool partial = ok != 15u || tok0 + kTileTok > u.all_see;  // the same for all waves
        uint64_t bits = ~0ull;
        bool slow = false;
        if (partial) {
            bool bad = false;
            uint4* v4 = reinterpret_cast<uint4*>(sV[stage]);
            for (int e = threadIdx.x; e < 4 * kPage / 8; e += 256) {
                // 16-byte chunk e: page, dim, swizzled half
                const int pg = e / (2 * kD), d = e / 2 % kD;
                const int first = tok0 + 16 * pg + 8 * ((e & 1) ^ v_swizzle(d));
                const int keep = (ok >> pg) & 1u ? min(max(u.total - first, 0), 8) : 0;  // tokens that exist
                uint4 v = v4[e];
                uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if (2 * j >= keep) w[j] = 0u;
                    else if (2 * j + 1 >= keep) w[j] &= 0xFFFFu;
                    bad |= finite_bf16x2(w[j]) != w[j];
                }
                v4[e] = make_uint4(w[0], w[1], w[2], w[3]);
            }
            slow = __syncthreads_or(bad);
            bits = seen_bits(tok0, ok);
        }
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
                    &sK[stage][kr * kD + ((2 * st + hl) ^ k_swizzle<kD>(kr & 15)) * 8]));
                s[j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf, qf[st], s[j], 0, 0, 0);
            }
            if (partial) {
                const uint64_t mine = bits >> (32 * blk + 8 * hl);
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    if (!((mine >> (16 * (r >> 3) + (r & 7))) & 1u)) s[j][r] = -INFINITY;
            }
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
        bf16x8 pf[kBlocks][2];
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
                pf[j][t] = as_bf16x8(make_uint4(cvt_pk_bf16(pv[0], pv[1]), cvt_pk_bf16(pv[2], pv[3]),
                                                cvt_pk_bf16(pv[4], pv[5]), cvt_pk_bf16(pv[6], pv[7])));
            }
        if (!slow) {
#pragma unroll
            for (int j = 0; j < kBlocks; ++j)
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    const int pg = 2 * (kGroups == 1 ? j : group) + t;
#pragma unroll
                    for (int i = 0; i < kDb; ++i) {
                        const int d = 32 * i + l32;
                        const bf16x8 vf = as_bf16x8(*reinterpret_cast<const uint4*>(
                            &sV[stage][pg * kPage + d * kPageTok + (hl ^ v_swizzle(d)) * 8]));
                        acc[i] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf, pf[j][t], acc[i], 0, 0, 0);
                    }
                }
        } else {
            // token by token: lanes l and l ^ 32 hold a column's rounded weights, eight
            // tokens of every sixteen each
#pragma unroll
            for (int j = 0; j < kBlocks; ++j)
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    const int pg = 2 * (kGroups == 1 ? j : group) + t;
                    const uint4 w = __builtin_bit_cast(uint4, pf[j][t]);
                    const uint32_t own[4] = {w.x, w.y, w.z, w.w};
#pragma unroll 1
                    for (int x = 0; x < kPageTok; ++x) {
                        const int e = x & 7;
                        const uint32_t pair = (e >> 1) == 0 ? own[0] : (e >> 1) == 1 ? own[1] : (e >> 1) == 2 ? own[2] : own[3];
                        const uint32_t from = __shfl(static_cast<int>(pair), 32 * (x >> 3) + l32, 64);
                        const float pt = bf16_to_f32(static_cast<uint16_t>(from >> (16 * (e & 1))));
                        const bool seen = (bits >> (16 * pg + x)) & 1u;
#pragma unroll
                        for (int i = 0; i < kDb; ++i)
#pragma unroll
                            for (int r = 0; r < 16; ++r) {
                                const int d = 32 * i + 8 * (r >> 2) + 4 * hl + (r & 3);
                                const float v = bf16_to_f32(sV[stage][pg * kPage + d * kPageTok + ((x >> 3) ^ v_swizzle(d)) * 8 + e]);
                                if (seen) acc[i][r] = fmaf(pt, v, acc[i][r]);
                            }
                    }
                }
        }
    };

    if (tiles > 0) {
        uint32_t ok = issue(0, 0);
        wait_vmem_all();
        __syncthreads();
        for (int t = 0; t < tiles; ++t) {
            uint32_t next = 0;
            if (t + 1 < tiles) next = issue((t + 1) & 1, t + 1);
            compute(t & 1, t, ok);
            ok = next;
            wait_vmem_all();
            __syncthreads();
        }
    }
    l_run += __shfl_xor(l_run, 32, 64);
    // acc: this lane's column, dims 32 i + 8 cc + 4 hl + [0, 4)
    if constexpr (kGroups == 2) {
        // the second wave of a column block hands its sums over
        float* hand = reinterpret_cast<float*>(&sK[0][0]);                  // 2 x 32 columns x D
        float* ml = reinterpret_cast<float*>(&sV[0][0]);
        const int cb = wave % WC;
        if (group == 1) {
#pragma unroll
            for (int i = 0; i < kDb; ++i)
#pragma unroll
                for (int r = 0; r < 16; ++r) hand[(cb * kDb * 16 + 16 * i + r) * 64 + lane] = acc[i][r];
            ml[(2 * cb) * 64 + lane] = m_run;
            ml[(2 * cb + 1) * 64 + lane] = l_run;
        }
        __syncthreads();
        if (group == 1) return;
        const float m2 = ml[(2 * cb) * 64 + lane], l2 = ml[(2 * cb + 1) * 64 + lane];
        const float M = fmaxf(m_run, m2);
        const float f1 = split_weight(m_run, M), f2 = split_weight(m2, M);
        l_run = l_run * f1 + l2 * f2;
        m_run = M;
#pragma unroll
        for (int i = 0; i < kDb; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][r] = acc[i][r] * f1 + hand[(cb * kDb * 16 + 16 * i + r) * 64 + lane] * f2;
    }
    if (!has) return;
    if (p.splits == 1) {
        const float inv = 1.0f / l_run;  // nothing visible: 0 * inf
        uint16_t* o = static_cast<uint16_t*>(p.out) + column_offset(p, u.b, row, head);
#pragma unroll
        for (int i = 0; i < kDb; ++i)
#pragma unroll
            for (int cc = 0; cc < 4; ++cc)
                *reinterpret_cast<uint2*>(o + 32 * i + 8 * cc + 4 * hl) =
                    make_uint2(cvt_pk_bf16(acc[i][4 * cc] * inv, acc[i][4 * cc + 1] * inv),
                               cvt_pk_bf16(acc[i][4 * cc + 2] * inv, acc[i][4 * cc + 3] * inv));
        return;
    }
    const int64_t part = (u.id * u.cols + col) * p.splits + split;
#pragma unroll
    for (int i = 0; i < kDb; ++i)
#pragma unroll
        for (int cc = 0; cc < 4; ++cc)
            *reinterpret_cast<float4*>(p.part_acc + part * kD + 32 * i + 8 * cc + 4 * hl) =
                make_float4(acc[i][4 * cc], acc[i][4 * cc + 1], acc[i][4 * cc + 2], acc[i][4 * cc + 3]);
    if (hl == 0) {
        p.part_ml[2 * part] = m_run;
        p.part_ml[2 * part + 1] = l_run;
    }
}

}  // namespace

TreeTiles tree_tiles(int64_t cols) {
    TreeTiles t{};
    t.waves = 4;
    t.col_waves = cols <= 64 ? 2 : 4;
    t.chunks = (cols + 32 * t.col_waves - 1) / (32 * t.col_waves);
    return t;
}

void launch_tree_tiles(const ChosenArgs& p, const TreeTiles& t, int64_t units, hipStream_t stream) {
    const unsigned grid = static_cast<unsigned>(units * t.chunks * p.splits);
    const int chunks = static_cast<int>(t.chunks), xcds = device_xcds(stream);
    if (p.head_dim == 128) {
        if (t.col_waves == 4) tree_tile_kernel<128, 4><<<grid, 256, 0, stream>>>(p, chunks, xcds);
        else tree_tile_kernel<128, 2><<<grid, 256, 0, stream>>>(p, chunks, xcds);
    } else {
        if (t.col_waves == 4) tree_tile_kernel<64, 4><<<grid, 256, 0, stream>>>(p, chunks, xcds);
        else tree_tile_kernel<64, 2><<<grid, 256, 0, stream>>>(p, chunks, xcds);
    }
}

}  // namespace sfg
