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

Kv8Plan plan_attn_kv8(const sfg_kv8_attn_args& a) { return Kv8Plan{1, 0}; }

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
    const dim3 grid(static_cast<unsigned>(a.tokens), static_cast<unsigned>(a.q_heads));
    if (s.pool_dtype == SFG_FP8) attn_kv8_rows_kernel<true><<<grid, 64, 0, stream>>>(a);
    else attn_kv8_rows_kernel<false><<<grid, 64, 0, stream>>>(a);
}

}  // namespace sfg
