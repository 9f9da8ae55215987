// sfg_kv8_append.hip -- keys and values stored in 8 bits at their slots, one scale for
// each page, kv head and pool.
#include <algorithm>

#include "sfg_kernels.hpp"
#include "sfg_kv8.hpp"

namespace sfg {
namespace {

struct AppendArgs {
    const void* keys; const void* values; int64_t key_stride, value_stride;
    uint8_t* k_pool; uint8_t* v_pool; float* scales; const int64_t* slots;
    int tokens, heads, dim, pt, pages;
    int shift;  // log2 of the page's tokens, -1 if they are no power of two
};

// The run of rows that row t begins: its page, the first slot there and how many rows; none
// if t goes on with a run or has no slot.
__device__ __forceinline__ int run_of(const AppendArgs& a, int t, int& page, int& off) {
    const int64_t slot = a.slots[t];
    if (slot < 0 || slot >= static_cast<int64_t>(a.pages) * a.pt) return 0;
    page = static_cast<int>(slot / a.pt);
    off = static_cast<int>(slot - static_cast<int64_t>(page) * a.pt);
    if (t > 0 && off > 0 && a.slots[t - 1] == slot - 1) return 0;
    int n = 1;
    while (off + n < a.pt && t + n < a.tokens && a.slots[t + n] == slot + n) ++n;
    return n;
}

template <typename T>
__device__ __forceinline__ float append_load(const T* p) {
    if constexpr (sizeof(T) == 4) return *p;
    else return bf16_to_f32(*p);
}

// Largest value of the wave (as wave_max, on integers: NaN above infinity).
__device__ __forceinline__ uint32_t wave_umax(uint32_t v) {
    const auto a = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    v = max(static_cast<uint32_t>(a[0]), static_cast<uint32_t>(a[1]));
    const auto b = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = max(static_cast<uint32_t>(b[0]), static_cast<uint32_t>(b[1]));
    auto lane = [](float x) { return __float_as_uint(x); };
    v = max(v, lane(lane_xor8(__uint_as_float(v))));
    v = max(v, lane(lane_xor4(__uint_as_float(v))));
    v = max(v, lane(lane_xor2(__uint_as_float(v))));
    return max(v, lane(lane_xor1(__uint_as_float(v))));
}

}  // namespace

// Any head dim and page size: a wave a run and (kv head, pool), its rows read twice.  token_step
// and dim_step: where a page's codes lie (K by tokens, V by dims).
template <typename T, bool FP8>
__global__ __launch_bounds__(64) void kv8_append_kernel(AppendArgs a) {
    const int t = blockIdx.x, h = blockIdx.y, which = blockIdx.z, lane = threadIdx.x;
    int page, off;
    const int n = run_of(a, t, page, off);
    if (n == 0) return;
    const int64_t stride = which ? a.value_stride : a.key_stride;
    const T* src = static_cast<const T*>(which ? a.values : a.keys) + static_cast<int64_t>(t) * stride + static_cast<int64_t>(h) * a.dim;
    const int64_t unit = static_cast<int64_t>(page) * a.heads + h;
    uint8_t* dst = (which ? a.v_pool : a.k_pool) + unit * a.pt * a.dim;
    const int token_step = which ? 1 : a.dim, dim_step = which ? a.pt : 1;
    uint32_t top = 0;
    for (int i = 0; i < n; ++i)
        for (int d = lane; d < a.dim; d += 64) top = max(top, __float_as_uint(append_load(src + i * stride + d)) & 0x7FFFFFFFu);
    float* at = a.scales + 2 * unit + which;
    const float old = off == 0 ? 0.0f : *at;
    const float scale = kv8_larger(old, kv8_scale<FP8>(wave_umax(top)));
    if (off > 0 && scale > old)
        for (int i = 0; i < off; ++i)
            for (int d = lane; d < a.dim; d += 64) {
                uint8_t* c = dst + i * token_step + d * dim_step;
                *c = kv8_code<FP8>(kv8_value<FP8>(*c) * old, scale);
            }
    for (int i = 0; i < n; ++i)
        for (int d = lane; d < a.dim; d += 64)
            dst[(off + i) * token_step + d * dim_step] = kv8_code<FP8>(append_load(src + i * stride + d), scale);
    if (lane == 0) *at = scale;
}

// ===========================================================================
// Head dim 64 and 128, pages of whole 16 tokens.  The workgroups of a window of 64 rows find the
// runs that begin there (in a prompt few rows begin one) and share them, a wave a run, kv head and
// pool.  K: lanes of 8 values along a row, the rows side by side in the page.  V: a lane owns D / 64
// dims, collects a dim's 16 tokens in registers and stores them as the 16 bytes that the page
// holds of them; a single token's bytes go one by one.  Rows stay in registers between the maximum and
// the codes (pages of 16 tokens).  Where the scale grew, the page's earlier codes are read, coded
// anew and written 16 bytes at a time, all of a lane's in flight.
// Bound by HBM for prompts (values read once, codes written once) and by latency for single
// tokens.  8100 rows of 8 kv heads of 128, bf16 to e4m3, four prompts: 16 us (3 TB/s; 20 with
// the compiler's division, 35 with a wave's registers holding fp32, 112 with a wave a row and both passes from
// memory); 64 rows of as many sequences: 3.6.
// ===========================================================================
namespace {

constexpr int kWindow = 64;

// N consecutive elements as they are in memory: fp32, or pairs of bf16.
typedef uint16_t uint16x2 __attribute__((ext_vector_type(2)));
template <typename T, int N>
struct Raw {
    static constexpr int kWords = sizeof(T) == 4 ? N : (N + 1) / 2;
    uint32_t w[kWords];
    __device__ __forceinline__ void load(const T* p, bool vec) {  // (vec: on a border of N elements, or of 16 bytes)
        if (vec && kWords % 4 == 0) {
#pragma unroll
            for (int i = 0; i < kWords; i += 4) {
                const uint4 v = reinterpret_cast<const uint4*>(p)[i / 4];
                w[i] = v.x; w[i + 1] = v.y; w[i + 2] = v.z; w[i + 3] = v.w;
            }
        } else if (vec && N == 2) {
            if constexpr (kWords == 2) {
                const uint2 v = *reinterpret_cast<const uint2*>(p);
                w[0] = v.x; w[1] = v.y;
            } else {
                w[0] = *reinterpret_cast<const uint32_t*>(p);
            }
        } else if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < N; ++i) w[i] = reinterpret_cast<const uint32_t*>(p)[i];
        } else {
#pragma unroll
            for (int i = 0; i < N; i += 2) w[i / 2] = static_cast<uint32_t>(p[i]) | (i + 1 < N ? static_cast<uint32_t>(p[i + 1]) << 16 : 0u);
        }
    }
    __device__ __forceinline__ float value(int i) const {
        if constexpr (sizeof(T) == 4) return __uint_as_float(w[i]);
        else return __uint_as_float(i & 1 ? w[i / 2] & 0xFFFF0000u : w[i / 2] << 16);
    }
    // the largest magnitude: of fp32 as its bits, of bf16 in both halves of a word
    __device__ __forceinline__ void top(uint32_t& t) const {
#pragma unroll
        for (int i = 0; i < kWords; ++i) {
            if constexpr (sizeof(T) == 4) t = max(t, w[i] & 0x7FFFFFFFu);
            else t = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(uint16x2, t), __builtin_bit_cast(uint16x2, w[i] & 0x7FFF7FFFu)));
        }
    }
};
template <typename T>
__device__ __forceinline__ uint32_t top_bits(uint32_t t) {
    if constexpr (sizeof(T) == 4) return wave_umax(t);
    else return wave_umax(max(t & 0xFFFFu, t >> 16)) << 16;
}

// A scale to divide many values by: mantissa, its correctly rounded reciprocal and exponent; no
// codes but 0 unless it is positive.
struct Divisor {
    float mant, inv;
    int exp;
    uint32_t mask;
    __device__ __forceinline__ explicit Divisor(float scale) {
        const bool live = scale > 0.0f;
        mant = live ? __builtin_amdgcn_frexp_mantf(scale) : 1.0f;
        exp = live ? -__builtin_amdgcn_frexp_expf(scale) : 0;
        inv = __fdiv_rn(1.0f, mant);
        mask = live ? ~0u : 0u;
    }
};
// Four codes (kv8_code's).  The quotient is the IEEE one in six operations instead of the
// division's ten and more: both sides times a power of two, so that nothing overflows or is
// subnormal where the code is not 0; x times the reciprocal is within 1.5 units of the quotient,
// one correction by the remainder, exact in an FMA, brings it within one, and the second one
// rounds it correctly since the reciprocal is (Markstein's theorem).  The remainder's zero
// would make +0 of a -0, whose code in e4m3 is another.
template <bool FP8>
__device__ __forceinline__ uint32_t codes4(const float (&v)[4], const Divisor& by) {
    constexpr float most = FP8 ? kMostFp8 : kMostI8;
    float y[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float x = __builtin_ldexpf(v[i], by.exp);
        float q = x * by.inv;
        q = fmaf(fmaf(-by.mant, q, x), by.inv, q);
        q = fmaf(fmaf(-by.mant, q, x), by.inv, q);
        q = __builtin_amdgcn_fmed3f(q, -most, most);
        y[i] = FP8 ? __builtin_copysignf(q, x) : q;
    }
    uint32_t r;
    if constexpr (FP8) {
        r = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
        r = __builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], r, true);
    } else {
        // (rounded to the nearest even whole number by the sum with 1.5 * 2^23, whose low byte it is)
        uint32_t u[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) u[i] = __float_as_uint(y[i] + 12582912.0f);
        r = __builtin_amdgcn_perm(__builtin_amdgcn_perm(u[3], u[2], 0x0C0C0400u), __builtin_amdgcn_perm(u[1], u[0], 0x0C0C0400u), 0x05040100u);
    }
    return r & by.mask;
}

// Four codes under a larger scale, the first `count` of them.
template <bool FP8>
__device__ __forceinline__ uint32_t recode4(uint32_t w, int count, float old, const Divisor& by) {
    float v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = kv8_value<FP8>(static_cast<uint8_t>(w >> (8 * i))) * old;
    const uint32_t r = codes4<FP8>(v, by);
    const uint32_t keep = count >= 4 ? 0 : count <= 0 ? ~0u : ~0u << (8 * count);
    return (w & keep) | (r & ~keep);
}
template <bool FP8>
__device__ __forceinline__ uint4 recode16(const uint4& w, int count, float old, const Divisor& by) {
    return make_uint4(recode4<FP8>(w.x, count, old, by), recode4<FP8>(w.y, count - 4, old, by), recode4<FP8>(w.z, count - 8, old, by),
                      recode4<FP8>(w.w, count - 12, old, by));
}

}  // namespace

template <typename T, bool FP8, int D>
__global__ __launch_bounds__(256) void kv8_append_runs_kernel(AppendArgs a, int vec_k, int vec_v) {
    constexpr int kL = D / 8, kRows = kWave / kL, kPass = kPageTok / kRows;  // K: lanes of a row, rows at a time
    constexpr int kV = D / kWave;                                            // V: dims of a lane
    const int lane = threadIdx.x & 63, base = blockIdx.x * kWindow;
    // the rows of the window that begin a run
    bool begins = false, goes = false;
    int64_t slot = -1;
    if (base + lane < a.tokens) {
        slot = a.slots[base + lane];
        const int64_t before = base + lane > 0 ? a.slots[base + lane - 1] : -2;
        const bool live = slot >= 0 && slot < static_cast<int64_t>(a.pages) * a.pt;
        begins = live && (before != slot - 1 || (a.shift >= 0 ? (slot & (a.pt - 1)) : slot % a.pt) == 0);
        goes = live && !begins;
    }
    const uint64_t runs = __ballot(begins), goes_on = __ballot(goes);
    const int count = __builtin_popcountll(runs) * a.heads * 2;
    for (int item = blockIdx.y * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); item < count; item += gridDim.y * 4) {
        const int which = item & 1, run = (item >> 1) / a.heads, h = (item >> 1) - run * a.heads;
        // the run-th row that begins one
        const int at = __builtin_ctzll(__ballot(begins && __builtin_popcountll(runs & ((uint64_t{1} << lane) - 1)) == run)), t = base + at;
        const int64_t s0 = static_cast<int64_t>(static_cast<uint64_t>(static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(slot >> 32), at))) << 32 |
                                                static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(slot), at)));
        const int page = static_cast<int>(a.shift >= 0 ? s0 >> a.shift : s0 / a.pt), off = static_cast<int>(s0 - static_cast<int64_t>(page) * a.pt);
        // rows of the run: to the next row of the window that does not go on with it, or beyond
        const uint64_t others = ~goes_on >> at >> 1;
        int n = others ? __builtin_ctzll(others) + 1 : kWindow - at;
        if (!others)
            for (int step = n;; step += kWave) {
                const int j = step + lane;
                const uint64_t stop = ~__ballot(off + j < a.pt && t + j < a.tokens && a.slots[t + j] == s0 + j);
                n = step + (stop ? __builtin_ctzll(stop) : kWave);
                if (stop) break;
            }
        const int64_t unit = static_cast<int64_t>(page) * a.heads + h;
        float* scale_at = a.scales + 2 * unit + which;
        const float old = off == 0 ? 0.0f : *scale_at;
        uint32_t top = 0;
        if (which == 0) {
            const T* src = static_cast<const T*>(a.keys) + static_cast<int64_t>(t) * a.key_stride + static_cast<int64_t>(h) * D + lane % kL * 8;
            uint8_t* dst = a.k_pool + unit * a.pt * D;
            Raw<T, 8> x[kPass];
            const int mine = lane / kL;  // the lane's row of those at a time
            auto load = [&](int from) {
#pragma unroll
                for (int i = 0; i < kPass; ++i)
                    x[i].load(src + static_cast<int64_t>(min(from + i * kRows + mine, n - 1)) * a.key_stride, vec_k);
            };
            for (int from = 0; from < n; from += kPageTok) {
                load(from);
#pragma unroll
                for (int i = 0; i < kPass; ++i) x[i].top(top);
            }
            const float scale = kv8_larger(old, kv8_scale<FP8>(top_bits<T>(top)));
            const Divisor by(scale);
            if (off > 0 && scale > old) {
                uint4* w = reinterpret_cast<uint4*>(dst);
                const int vectors = off * (D / 16);
                for (int i = lane; i < vectors; i += 2 * kWave) {  // (two in flight)
                    const bool two = i + kWave < vectors;
                    const uint4 p = w[i], q = two ? w[i + kWave] : p;
                    w[i] = recode16<FP8>(p, 16, old, by);
                    if (two) w[i + kWave] = recode16<FP8>(q, 16, old, by);
                }
            }
            for (int from = 0; from < n; from += kPageTok) {
                if (n > kPageTok) load(from);
#pragma unroll
                for (int i = 0; i < kPass; ++i) {
                    const int r = from + i * kRows + mine;
                    if (r >= n) continue;
                    float v[2][4];
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[e / 4][e % 4] = x[i].value(e);
                    *reinterpret_cast<uint2*>(dst + (off + r) * D + lane % kL * 8) = make_uint2(codes4<FP8>(v[0], by), codes4<FP8>(v[1], by));
                }
            }
            if (lane == 0) *scale_at = scale;
        } else {
            const T* src = static_cast<const T*>(a.values) + static_cast<int64_t>(t) * a.value_stride + static_cast<int64_t>(h) * D + lane * kV;
            uint8_t* dst = a.v_pool + unit * a.pt * D + static_cast<int64_t>(lane) * kV * a.pt;
            Raw<T, kV> x[kPageTok];
            // the run's tokens among the 16 of the page from `from`: [lo, hi)
            auto load = [&](int from, int& lo, int& hi) {
                lo = max(off - from, 0);
                hi = min(off + n - from, kPageTok);
#pragma unroll
                for (int i = 0; i < kPageTok; ++i) {
                    if (i >= lo && i < hi) x[i].load(src + static_cast<int64_t>(from + i - off) * a.value_stride, vec_v);
                }
            };
            const int first = off & ~(kPageTok - 1);
            int lo, hi;
            for (int from = first; from < off + n; from += kPageTok) {
                load(from, lo, hi);
#pragma unroll
                for (int i = 0; i < kPageTok; ++i)
                    if (i >= lo && i < hi) x[i].top(top);
            }
            const float scale = kv8_larger(old, kv8_scale<FP8>(top_bits<T>(top)));
            const Divisor by(scale);
            const bool anew = off > 0 && scale > old;
            if (anew)  // the runs of 16 before the one that the new tokens begin in
                for (int from = 0; from < first; from += kPageTok)
#pragma unroll
                    for (int e = 0; e < kV; ++e) {
                        uint4* w = reinterpret_cast<uint4*>(dst + e * a.pt + from);
                        *w = recode16<FP8>(*w, 16, old, by);
                    }
            for (int from = first; from < off + n; from += kPageTok) {
                if (off + n - first > kPageTok) load(from, lo, hi);
                const bool one = hi - lo == 1 && !anew;  // its bytes alone, with nothing read
                uint4 w[kV];
#pragma unroll
                for (int e = 0; e < kV; ++e)
                    w[e] = !one && (lo > 0 || hi < kPageTok) ? *reinterpret_cast<const uint4*>(dst + e * a.pt + from) : make_uint4(0, 0, 0, 0);
#pragma unroll
                for (int e = 0; e < kV; ++e) {
                    if (anew && lo > 0) w[e] = recode16<FP8>(w[e], lo, old, by);
                    uint32_t u[4] = {w[e].x, w[e].y, w[e].z, w[e].w};
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        if (4 * j + 4 <= lo || 4 * j >= hi) continue;
                        float v[4];
#pragma unroll
                        for (int i = 0; i < 4; ++i) v[i] = 4 * j + i >= lo && 4 * j + i < hi ? x[4 * j + i].value(e) : 0.0f;
                        const uint32_t c = codes4<FP8>(v, by);
                        // the bytes of [lo, hi)
                        const uint32_t from_lo = lo > 4 * j ? ~0u << (8 * (lo - 4 * j)) : ~0u;
                        const uint32_t to_hi = hi < 4 * j + 4 ? (1u << (8 * (hi - 4 * j))) - 1u : ~0u;
                        u[j] = (u[j] & ~(from_lo & to_hi)) | (c & from_lo & to_hi);
                        if (one) dst[e * a.pt + from + lo] = static_cast<uint8_t>(c >> (8 * (lo & 3)));
                    }
                    if (!one) *reinterpret_cast<uint4*>(dst + e * a.pt + from) = make_uint4(u[0], u[1], u[2], u[3]);
                }
            }
            if (lane == 0) *scale_at = scale;
        }
    }
}

// Workgroups among which the runs of all windows are shared, if there are as many (in a prompt
// a window begins four runs, so 2 heads workgroups have one each wave).
constexpr int kAppendGroups = 2048;

void launch_kv8_append(const sfg_kv8_append_args& s, hipStream_t stream) {
    AppendArgs a{};
    a.keys = s.keys; a.values = s.values; a.key_stride = s.key_stride; a.value_stride = s.value_stride;
    a.k_pool = static_cast<uint8_t*>(s.k_pool); a.v_pool = static_cast<uint8_t*>(s.v_pool);
    a.scales = s.scales; a.slots = s.slots;
    a.tokens = static_cast<int>(s.tokens); a.heads = static_cast<int>(s.kv_heads); a.dim = static_cast<int>(s.head_dim);
    a.pt = static_cast<int>(s.page_tokens); a.pages = static_cast<int>(s.num_pages);
    const bool fp8 = s.pool_dtype == SFG_FP8;
    const bool aligned = ((reinterpret_cast<uintptr_t>(s.k_pool) | reinterpret_cast<uintptr_t>(s.v_pool)) & 15) == 0;
    if ((a.dim == 64 || a.dim == 128) && a.pt % kPageTok == 0 && aligned) {
        const int bytes = s.dtype == SFG_F32 ? 4 : 2;
        const int vec_k = (reinterpret_cast<uintptr_t>(s.keys) & 15) == 0 && s.key_stride * bytes % 16 == 0;
        const int vec_v = reinterpret_cast<uintptr_t>(s.values) % (2 * bytes) == 0 && s.value_stride % 2 == 0;  // (two dims a lane)
        a.shift = (a.pt & (a.pt - 1)) == 0 ? __builtin_ctz(a.pt) : -1;
        const int windows = (a.tokens + kWindow - 1) / kWindow, most = 2 * a.heads * kWindow / 4;
        const int ways = std::min(std::max(kAppendGroups / windows, 2 * a.heads), most);
        const dim3 grid(static_cast<unsigned>(windows), static_cast<unsigned>(std::min(ways, 65535)));
        if (s.dtype == SFG_F32) {
            if (a.dim == 128) fp8 ? kv8_append_runs_kernel<float, true, 128><<<grid, 256, 0, stream>>>(a, vec_k, vec_v) : kv8_append_runs_kernel<float, false, 128><<<grid, 256, 0, stream>>>(a, vec_k, vec_v);
            else fp8 ? kv8_append_runs_kernel<float, true, 64><<<grid, 256, 0, stream>>>(a, vec_k, vec_v) : kv8_append_runs_kernel<float, false, 64><<<grid, 256, 0, stream>>>(a, vec_k, vec_v);
        } else {
            if (a.dim == 128) fp8 ? kv8_append_runs_kernel<uint16_t, true, 128><<<grid, 256, 0, stream>>>(a, vec_k, vec_v) : kv8_append_runs_kernel<uint16_t, false, 128><<<grid, 256, 0, stream>>>(a, vec_k, vec_v);
            else fp8 ? kv8_append_runs_kernel<uint16_t, true, 64><<<grid, 256, 0, stream>>>(a, vec_k, vec_v) : kv8_append_runs_kernel<uint16_t, false, 64><<<grid, 256, 0, stream>>>(a, vec_k, vec_v);
        }
        return;
    }
    const dim3 grid(static_cast<unsigned>(a.tokens), static_cast<unsigned>(a.heads), 2);
    if (s.dtype == SFG_F32) {
        if (fp8) kv8_append_kernel<float, true><<<grid, 64, 0, stream>>>(a);
        else kv8_append_kernel<float, false><<<grid, 64, 0, stream>>>(a);
    } else {
        if (fp8) kv8_append_kernel<uint16_t, true><<<grid, 64, 0, stream>>>(a);
        else kv8_append_kernel<uint16_t, false><<<grid, 64, 0, stream>>>(a);
    }
}

}  // namespace sfg
