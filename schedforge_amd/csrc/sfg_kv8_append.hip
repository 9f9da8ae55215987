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

__device__ __forceinline__ uint32_t wave_umax(uint32_t v) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) v = max(v, static_cast<uint32_t>(__shfl_xor(v, off, kWave)));
    return v;
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

void launch_kv8_append(const sfg_kv8_append_args& s, hipStream_t stream) {
    AppendArgs a{};
    a.keys = s.keys; a.values = s.values; a.key_stride = s.key_stride; a.value_stride = s.value_stride;
    a.k_pool = static_cast<uint8_t*>(s.k_pool); a.v_pool = static_cast<uint8_t*>(s.v_pool);
    a.scales = s.scales; a.slots = s.slots;
    a.tokens = static_cast<int>(s.tokens); a.heads = static_cast<int>(s.kv_heads); a.dim = static_cast<int>(s.head_dim);
    a.pt = static_cast<int>(s.page_tokens); a.pages = static_cast<int>(s.num_pages);
    const dim3 grid(static_cast<unsigned>(a.tokens), static_cast<unsigned>(a.heads), 2);
    const bool fp8 = s.pool_dtype == SFG_FP8;
    if (s.dtype == SFG_F32) {
        if (fp8) kv8_append_kernel<float, true><<<grid, 64, 0, stream>>>(a);
        else kv8_append_kernel<float, false><<<grid, 64, 0, stream>>>(a);
    } else {
        if (fp8) kv8_append_kernel<uint16_t, true><<<grid, 64, 0, stream>>>(a);
        else kv8_append_kernel<uint16_t, false><<<grid, 64, 0, stream>>>(a);
    }
}

}  // namespace sfg
