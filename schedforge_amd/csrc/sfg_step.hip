// sfg_step.hip -- what a serving step does before its cache is touched: pages and slots
// from the sequences' lengths (kv_plan), rotary positions (rope).
#include <algorithm>

#include "sfg_kernels.hpp"
#include "sfg_kv8.hpp"

namespace sfg {

// ===========================================================================
// Pages given back and taken, slots of the new tokens.
// ===========================================================================
namespace {

constexpr int kPlanThreads = 1024;

struct PlanArgs {
    const int32_t* keep; const int32_t* counts; int32_t* seq_lens; int32_t* page_table;
    int32_t* free_pages; int32_t* free_count; int32_t* starts; int32_t* positions; int64_t* slots;
    int batch, per, pages, pt, max_tokens;
    __device__ int pages_of(int tokens) const { return (tokens + pt - 1) / pt; }
};

// Sums of the lanes' values up to each thread of the workgroup (each sum cut to `most`,
// which the values do not exceed) and over all of it.
__device__ int block_inclusive(int v, uint32_t most, int* sums, int& total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint32_t x = static_cast<uint32_t>(v);
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const uint32_t y = __shfl_up(x, off, kWave);
        if (lane >= off) x = min(x + y, most);
    }
    __syncthreads();
    if (lane == 63) sums[wave] = static_cast<int>(x);
    __syncthreads();
    uint32_t before = 0, all = 0;
    for (int w = 0; w < kPlanThreads / 64; ++w) {
        if (w == wave) before = all;
        all = min(all + static_cast<uint32_t>(sums[w]), most);
    }
    total = static_cast<int>(all);
    return static_cast<int>(min(x + before, most));
}

// The last entry of at[0, kPlanThreads) that is not above i.
__device__ __forceinline__ int owner(const int* at, int i) {
    int lo = 0;
#pragma unroll
    for (int step = kPlanThreads / 2; step > 0; step >>= 1)
        if (at[lo + step] <= i) lo += step;
    return lo;
}

__device__ __forceinline__ void place(const PlanArgs& a, int t, int b, int pos) {
    const int id = a.page_table[static_cast<int64_t>(b) * a.per + pos / a.pt];
    a.positions[t] = pos;
    a.slots[t] = id < 0 || id >= a.pages ? -1 : static_cast<int64_t>(id) * a.pt + pos % a.pt;
}

}  // namespace

// One workgroup, a thread a sequence (1024 of them at a time): prefix sums give each
// sequence its place on the free list and among the rows, and the pages and rows
// themselves are dealt over all threads, which find their sequence by bisection.
__global__ __launch_bounds__(kPlanThreads) void kv_plan_kernel(PlanArgs a, int tokens_too) {
    __shared__ int sums[kPlanThreads / 64];
    __shared__ int at[kPlanThreads], from[kPlanThreads];
    const int tid = threadIdx.x;
    const int capacity = a.per * a.pt;
    constexpr uint32_t kAny = 0x7FFFFFFFu;
    const int had = min(max(a.free_count[0], 0), a.pages);
    // (the tables' entries are fewer than 2^31: so are the pages given back)
    int given = 0;
    if (a.keep) {
        for (int base = 0; base < a.batch; base += kPlanThreads) {
            const int b = base + tid;
            int last = 0, gone = 0;
            if (b < a.batch) {
                const int len = min(max(a.seq_lens[b], 0), capacity);
                last = a.pages_of(len);
                gone = last - a.pages_of(min(max(a.keep[b], 0), len));
            }
            int total;
            const int upto = block_inclusive(gone, kAny, sums, total);
            at[tid] = upto - gone;
            from[tid] = last - 1;
            __syncthreads();
            for (int i = tid; i < total; i += kPlanThreads) {
                const int q = owner(at, i);
                int32_t* entry = a.page_table + static_cast<int64_t>(base + q) * a.per + (from[q] - (i - at[q]));
                const int64_t to = static_cast<int64_t>(had) + given + i;
                if (to < a.pages) a.free_pages[to] = *entry;
                *entry = -1;
            }
            given += total;
            __syncthreads();
        }
    }
    const int have = static_cast<int>(min(static_cast<int64_t>(had) + given, static_cast<int64_t>(a.pages)));
    const uint32_t most = static_cast<uint32_t>(a.max_tokens) + 1;
    int asked = 0, rows_asked = 0, taken = 0, rows = 0;
    for (int base = 0; base < a.batch; base += kPlanThreads) {
        const int b = base + tid;
        int kept = 0, want = 0, need = 0, first = 0;
        if (b < a.batch) {
            const int len = min(max(a.seq_lens[b], 0), capacity);
            kept = a.keep ? min(max(a.keep[b], 0), len) : len;
            want = max(a.counts[b], 0);
            if (want > capacity - kept) want = 0;
            first = a.pages_of(kept);
            need = a.pages_of(kept + want) - first;
        }
        int total;
        const int need_upto = asked + block_inclusive(need, kAny, sums, total);
        asked += total;
        const uint32_t cut = min(static_cast<uint32_t>(want), most);
        const uint32_t want_upto = min(static_cast<uint32_t>(block_inclusive(static_cast<int>(cut), most, sums, total)) + rows_asked, most);
        rows_asked = static_cast<int>(min(static_cast<uint32_t>(rows_asked) + total, most));
        if ((need > 0 && need_upto > have) || want_upto >= most) want = need = 0;
        // pages
        int upto = block_inclusive(need, kAny, sums, total);
        at[tid] = upto - need;
        from[tid] = first;
        __syncthreads();
        for (int i = tid; i < total; i += kPlanThreads) {
            const int q = owner(at, i);
            a.page_table[static_cast<int64_t>(base + q) * a.per + from[q] + (i - at[q])] = a.free_pages[have - 1 - taken - i];
        }
        taken += total;
        // rows
        upto = block_inclusive(want, kAny, sums, total);  // (its barriers are behind the pages' last reads)
        at[tid] = upto - want;
        from[tid] = kept;
        if (b < a.batch) {
            a.seq_lens[b] = kept + want;
            a.starts[b] = rows + upto - want;
        }
        __syncthreads();
        if (tokens_too)
            for (int i = tid; i < total; i += kPlanThreads) {
                const int q = owner(at, i);
                place(a, rows + i, base + q, from[q] + (i - at[q]));
            }
        rows += total;
        __syncthreads();
    }
    if (tid == 0) {
        a.starts[a.batch] = rows;
        a.free_count[0] = have - taken;
    }
    if (tokens_too)
        for (int t = rows + tid; t < a.max_tokens; t += kPlanThreads) {
            a.positions[t] = -1;
            a.slots[t] = -1;
        }
}

// The rows of a step of many tokens: a thread a row, its sequence by bisection.
__global__ __launch_bounds__(256) void kv_plan_rows_kernel(PlanArgs a) {
    const int t = blockIdx.x * 256 + threadIdx.x;
    if (t >= a.max_tokens) return;
    if (t >= a.starts[a.batch]) {
        a.positions[t] = -1;
        a.slots[t] = -1;
        return;
    }
    int lo = 0, hi = a.batch;  // starts[lo] <= t < starts[hi]
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (a.starts[mid] <= t) lo = mid;
        else hi = mid;
    }
    place(a, t, lo, a.seq_lens[lo] - (a.starts[lo + 1] - a.starts[lo]) + (t - a.starts[lo]));
}

void launch_kv_plan(const sfg_kv_plan_args& s, hipStream_t stream) {
    PlanArgs a{};
    a.keep = s.keep; a.counts = s.counts; a.seq_lens = s.seq_lens; a.page_table = s.page_table;
    a.free_pages = s.free_pages; a.free_count = s.free_count; a.starts = s.starts;
    a.positions = s.positions; a.slots = s.slots;
    a.batch = static_cast<int>(s.batch); a.per = static_cast<int>(s.pages_per_seq);
    a.pages = static_cast<int>(s.num_pages); a.pt = static_cast<int>(s.page_tokens);
    a.max_tokens = static_cast<int>(s.max_tokens);
    const bool one = a.max_tokens <= 4 * kPlanThreads;
    kv_plan_kernel<<<1, kPlanThreads, 0, stream>>>(a, one);
    if (!one) kv_plan_rows_kernel<<<dim3(static_cast<unsigned>((a.max_tokens + 255) / 256)), 256, 0, stream>>>(a);
}

// ===========================================================================
// Rotary positions.
// ===========================================================================
namespace {

struct RopeArgs {
    const void* in[2]; void* out[2]; int64_t in_stride[2], out_stride[2]; int heads[2];
    const int32_t* positions; const uint64_t* turns; float magnitude;
    int tokens, dim, pairs, interleaved;
};

// Cosine and sine of a position's angle.  position * turns wraps modulo 2^64 as whole turns
// do; its upper half is the angle in turns to 2^-33, in [-1/2, 1/2) as a signed number.
__device__ __forceinline__ float2 rope_angle(int position, uint64_t turns, float magnitude) {
    const uint64_t phase = static_cast<uint64_t>(position) * turns;
    float s, c;
    sincospif(static_cast<float>(static_cast<int32_t>(phase >> 32)) * 0x1p-31f, &s, &c);
    return make_float2(c * magnitude, s * magnitude);
}

template <typename T>
__device__ __forceinline__ float rope_load(const T* p) {
    if constexpr (sizeof(T) == 4) return *p;
    else return bf16_to_f32(*p);
}
template <typename T>
__device__ __forceinline__ T rope_store(float v) {
    if constexpr (sizeof(T) == 4) return v;
    else return static_cast<uint16_t>(cvt_pk_bf16(v, v));  // (a NaN stays one)
}

}  // namespace

// A thread a pair (or a value behind the rotary part) of a row, for all heads.
template <typename T>
__global__ __launch_bounds__(256) void rope_kernel(RopeArgs a) {
    const int units = a.dim - a.pairs;  // pairs, then the values behind them
    const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    const int64_t t = i / units;
    const int u = static_cast<int>(i % units);
    if (t >= a.tokens) return;
    const int pos = a.positions[t];
    if (pos < 0) return;
    const bool turned = u < a.pairs;
    const int d0 = turned ? (a.interleaved ? 2 * u : u) : u + a.pairs;
    const int d1 = turned ? (a.interleaved ? 2 * u + 1 : u + a.pairs) : d0;
    const float2 cs = turned ? rope_angle(pos, a.turns[u], a.magnitude) : make_float2(1.f, 0.f);
    for (int w = 0; w < 2; ++w) {
        const T* x = static_cast<const T*>(a.in[w]) + t * a.in_stride[w];
        T* y = static_cast<T*>(a.out[w]) + t * a.out_stride[w];
        for (int h = 0; h < a.heads[w]; ++h, x += a.dim, y += a.dim) {
            if (!turned) {
                y[d0] = x[d0];
                continue;
            }
            const float p = rope_load(x + d0), q = rope_load(x + d1);
            y[d0] = rope_store<T>(p * cs.x - q * cs.y);
            y[d1] = rope_store<T>(q * cs.x + p * cs.y);
        }
    }
}

void launch_rope(const sfg_rope_args& s, hipStream_t stream) {
    RopeArgs a{};
    a.in[0] = s.q; a.in[1] = s.k; a.out[0] = s.q_out; a.out[1] = s.k_out;
    a.in_stride[0] = s.q_stride; a.in_stride[1] = s.k_stride;
    a.out_stride[0] = s.q_out_stride; a.out_stride[1] = s.k_out_stride;
    a.heads[0] = static_cast<int>(s.q_heads); a.heads[1] = static_cast<int>(s.kv_heads);
    a.positions = s.positions; a.turns = s.turns; a.magnitude = s.magnitude;
    a.tokens = static_cast<int>(s.tokens); a.dim = static_cast<int>(s.head_dim);
    a.pairs = static_cast<int>(s.rotary_dim / 2); a.interleaved = s.layout == SFG_ROPE_INTERLEAVED;
    const int64_t units = static_cast<int64_t>(a.tokens) * (a.dim - a.pairs);
    const dim3 grid(static_cast<unsigned>((units + 255) / 256));
    if (s.dtype == SFG_F32) rope_kernel<float><<<grid, 256, 0, stream>>>(a);
    else rope_kernel<uint16_t><<<grid, 256, 0, stream>>>(a);
}

}  // namespace sfg
