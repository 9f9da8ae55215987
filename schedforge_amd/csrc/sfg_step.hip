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

struct PlanArgs {
    const int32_t* keep; const int32_t* counts; int32_t* seq_lens; int32_t* page_table;
    int32_t* free_pages; int32_t* free_count; int32_t* starts; int32_t* positions; int64_t* slots;
    int batch, per, pages, pt, max_tokens;
    int shift;  // log2 of the page's tokens, -1 if they are no power of two
    __device__ __forceinline__ int page_of(int pos) const { return shift >= 0 ? pos >> shift : pos / pt; }
    __device__ __forceinline__ int pages_of(int tokens) const { return page_of(tokens + pt - 1); }
};

// A sequence's tokens, the kept ones, and the ones it asks for (none past the capacity).
struct PlanSeq {
    int len, kept, want;
};
__device__ __forceinline__ PlanSeq plan_seq(const PlanArgs& a, int b) {
    PlanSeq s{0, 0, 0};
    if (b >= a.batch) return s;
    const int capacity = a.per * a.pt;
    const int len = a.seq_lens[b], keep = a.keep ? a.keep[b] : 0x7FFFFFFF, want = a.counts[b];
    s.len = min(max(len, 0), capacity);
    s.kept = min(max(keep, 0), s.len);
    s.want = max(want, 0) > capacity - s.kept ? 0 : max(want, 0);
    return s;
}

// Sums of two values up to each thread of the workgroup and over all of it.  The second one's
// sums are cut to `most`, which its values do not exceed (64 of them fit 32 bits).
template <int THREADS>
__device__ __forceinline__ int2 block_inclusive(int2 v, int most, int2* sums, int2& total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int2 x = make_int2(wave_inclusive(v.x), wave_inclusive(v.y));
    if (lane == 63) sums[wave] = x;
    __syncthreads();
    int2 before = make_int2(0, 0), all = make_int2(0, 0);
#pragma unroll
    for (int w = 0; w < THREADS / 64; ++w) {
        if (w == wave) before = all;
        const int2 y = sums[w];
        all = make_int2(all.x + y.x, min(all.y + y.y, most));
    }
    total = all;
    return make_int2(x.x + before.x, min(x.y + before.y, most));
}

// The last entry of at[0, THREADS) that is not above i.
template <int THREADS>
__device__ __forceinline__ int owner(const int* at, int i) {
    int lo = 0;
#pragma unroll
    for (int step = THREADS / 2; step > 0; step >>= 1)
        if (at[lo + step] <= i) lo += step;
    return lo;
}

__device__ __forceinline__ void place(const PlanArgs& a, int t, int b, int pos) {
    const int page = a.page_of(pos), id = a.page_table[static_cast<int64_t>(b) * a.per + page];
    a.positions[t] = pos;
    a.slots[t] = id < 0 || id >= a.pages ? -1 : static_cast<int64_t>(id) * a.pt + (pos - page * a.pt);
}

}  // namespace

// One workgroup, a thread a sequence (THREADS of them at a time): prefix sums give each
// sequence its place on the free list and among the rows, and the pages and rows
// themselves are dealt over all threads, which find their sequence by bisection.  Bound by latency: a
// chain of loads, three sums and the list's and table's round trips.  64 sequences of one row 3.6 us
// (7.9 with the lengths read again for each sum, sums by shuffles and divisions by the page).
template <int THREADS>
__global__ __launch_bounds__(THREADS) void kv_plan_kernel(PlanArgs a, int rows_too) {
    __shared__ int2 sums[3][THREADS / 64];
    __shared__ int page_at[THREADS], page_from[THREADS], row_at[THREADS], row_from[THREADS];
    const int tid = threadIdx.x;
    constexpr int kAny = 0x7FFFFFFF;
    const int had = min(max(a.free_count[0], 0), a.pages);
    PlanSeq s = plan_seq(a, tid);
    // (the tables' entries are fewer than 2^31: so are the pages given back)
    int given = 0;
    if (a.keep) {
        for (int base = 0;;) {
            const int last = a.pages_of(s.len), gone = last - a.pages_of(s.kept);
            int2 total;
            const int upto = block_inclusive<THREADS>(make_int2(gone, 0), kAny, sums[0], total).x;
            if (total.x) {
                page_at[tid] = upto - gone;
                page_from[tid] = last - 1;
                __syncthreads();
                for (int i = tid; i < total.x; i += THREADS) {
                    const int q = owner<THREADS>(page_at, i);
                    int32_t* entry = a.page_table + static_cast<int64_t>(base + q) * a.per + (page_from[q] - (i - page_at[q]));
                    const int64_t to = static_cast<int64_t>(had) + given + i;
                    if (to < a.pages) a.free_pages[to] = *entry;
                    *entry = -1;
                }
                given += total.x;
                __syncthreads();
            }
            if ((base += THREADS) >= a.batch) break;
            __syncthreads();
            s = plan_seq(a, base + tid);
        }
        if (a.batch > THREADS) s = plan_seq(a, tid);
    }
    const int have = static_cast<int>(min(static_cast<int64_t>(had) + given, static_cast<int64_t>(a.pages)));
    const int most = a.max_tokens + 1;
    int asked = 0, rows_asked = 0, taken = 0, rows = 0;
    for (int base = 0;;) {
        const int b = base + tid, first = a.pages_of(s.kept);
        int want = s.want, need = a.pages_of(s.kept + want) - first;
        int2 total;
        int2 upto = block_inclusive<THREADS>(make_int2(need, min(want, most)), most, sums[1], total);
        if ((need > 0 && asked + upto.x > have) || rows_asked + upto.y >= most) want = need = 0;
        asked += total.x;
        rows_asked = min(rows_asked + total.y, most);
        upto = block_inclusive<THREADS>(make_int2(need, want), kAny, sums[2], total);
        page_at[tid] = upto.x - need;
        page_from[tid] = first;
        row_at[tid] = upto.y - want;
        row_from[tid] = s.kept;
        if (b < a.batch) {
            a.seq_lens[b] = s.kept + want;
            a.starts[b] = rows + upto.y - want;
        }
        __syncthreads();
        for (int i = tid; i < total.x; i += THREADS) {
            const int q = owner<THREADS>(page_at, i);
            a.page_table[static_cast<int64_t>(base + q) * a.per + page_from[q] + (i - page_at[q])] = a.free_pages[have - 1 - taken - i];
        }
        if (rows_too) {
            if (total.x) __syncthreads();
            for (int i = tid; i < total.y; i += THREADS) {
                const int q = owner<THREADS>(row_at, i);
                place(a, rows + i, base + q, row_from[q] + (i - row_at[q]));
            }
        }
        taken += total.x;
        rows += total.y;
        if ((base += THREADS) >= a.batch) break;
        s = plan_seq(a, base + tid);
        __syncthreads();
    }
    if (tid == 0) {
        a.starts[a.batch] = rows;
        a.free_count[0] = have - taken;
    }
    if (rows_too)
        for (int t = rows + tid; t < a.max_tokens; t += THREADS) {
            a.positions[t] = -1;
            a.slots[t] = -1;
        }
}

// The rows of a step of many: a thread a row, its sequence by bisection of the starts (in LDS
// where they fit).
constexpr int kPlanStarts = 2048;
__global__ __launch_bounds__(256) void kv_plan_rows_kernel(PlanArgs a) {
    __shared__ int begins[kPlanStarts];
    const bool fit = a.batch < kPlanStarts;
    if (fit) {
        for (int i = threadIdx.x; i <= a.batch; i += 256) begins[i] = a.starts[i];
        __syncthreads();
    }
    const int* starts = fit ? begins : a.starts;
    const int t = blockIdx.x * 256 + threadIdx.x;
    if (t >= a.max_tokens) return;
    if (t >= starts[a.batch]) {
        a.positions[t] = -1;
        a.slots[t] = -1;
        return;
    }
    int lo = 0, hi = a.batch;  // starts[lo] <= t < starts[hi]
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (starts[mid] <= t) lo = mid;
        else hi = mid;
    }
    place(a, t, lo, a.seq_lens[lo] - (starts[lo + 1] - starts[lo]) + (t - starts[lo]));
}

// Rows that the workgroup places itself: 8 x 250 in 7.3 us a call, 9.8 with a second launch; 8 x 500
// 7.6 and 9.8; 16 x 500 9.8 and 9.5.
constexpr int kPlanRows = 4096;

void launch_kv_plan(const sfg_kv_plan_args& s, hipStream_t stream) {
    PlanArgs a{};
    a.keep = s.keep; a.counts = s.counts; a.seq_lens = s.seq_lens; a.page_table = s.page_table;
    a.free_pages = s.free_pages; a.free_count = s.free_count; a.starts = s.starts;
    a.positions = s.positions; a.slots = s.slots;
    a.batch = static_cast<int>(s.batch); a.per = static_cast<int>(s.pages_per_seq);
    a.pages = static_cast<int>(s.num_pages); a.pt = static_cast<int>(s.page_tokens);
    a.max_tokens = static_cast<int>(s.max_tokens);
    a.shift = (a.pt & (a.pt - 1)) == 0 ? __builtin_ctz(a.pt) : -1;
    const bool one = a.max_tokens <= kPlanRows;
    if (a.batch <= 256 && a.max_tokens <= 1024) kv_plan_kernel<256><<<1, 256, 0, stream>>>(a, 1);
    else kv_plan_kernel<1024><<<1, 1024, 0, stream>>>(a, one);
    if (!one) kv_plan_rows_kernel<<<dim3(static_cast<unsigned>((a.max_tokens + 255) / 256)), 256, 0, stream>>>(a);
}

// ===========================================================================
// Rotary positions.
// ===========================================================================
namespace {

constexpr int kRopeThreads = 256;
constexpr int kRopeItems = 2;              // of a thread at a time
// Bytes written from which stores pass the caches by (2048 rows of 40 heads of 128, 21 MB: 8.9 us,
// 10.1 through them; what is smaller is left to the L2s, 32 MB together, for the next operator).
constexpr int64_t kRopeStream = 16 << 20;

struct RopeArgs {
    const void* in[2]; void* out[2]; int64_t in_stride[2], out_stride[2]; int heads[2];
    const int32_t* positions; const uint64_t* turns; float magnitude;
    int tokens, dim, pairs, interleaved;
    // a workgroup's rows and heads; units of a head and how to divide by them and by a row's (reciprocal: 0 for one)
    int rows, chunk, units;
    uint32_t by_units, by_row;
};

// Cosine and sine of a position's angle.  position * turns wraps modulo 2^64 as whole turns
// do; its upper half is the angle in turns to 2^-33, in [-1/2, 1/2) as a signed number.  Rounded to
// fp32 (2^-25 near half a turn), which is what the fp32 sine and cosine take: outputs in fp32 are 2.9e-8
// off, 2.1e-8 with angles in 64 bits.
__device__ __forceinline__ float2 rope_angle(int position, uint64_t turns, float magnitude) {
    const uint64_t phase = static_cast<uint64_t>(position) * turns;
    float s, c;
    sincospif(static_cast<float>(static_cast<int32_t>(phase >> 32)) * 0x1p-31f, &s, &c);
    return make_float2(c * magnitude, s * magnitude);
}

// A vector of N values (16 bytes, or one value) as fp32 and back.
template <typename T, int N>
__device__ __forceinline__ void rope_load(const T* p, float (&v)[N]) {
    if constexpr (N == 1) {
        v[0] = sizeof(T) == 4 ? *reinterpret_cast<const float*>(p) : bf16_to_f32(*reinterpret_cast<const uint16_t*>(p));
    } else if constexpr (sizeof(T) == 4) {
        const float4 w = *reinterpret_cast<const float4*>(p);
        v[0] = w.x; v[1] = w.y; v[2] = w.z; v[3] = w.w;
    } else {
        const uint4 w = *reinterpret_cast<const uint4*>(p);
        const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[2 * i] = __uint_as_float(u[i] << 16);
            v[2 * i + 1] = __uint_as_float(u[i] & 0xFFFF0000u);
        }
    }
}
template <bool STREAM>
__device__ __forceinline__ void rope_store16(void* p, const uint4& v) {
    typedef uint32_t uint32x4 __attribute__((ext_vector_type(4)));
    if constexpr (STREAM) __builtin_nontemporal_store(__builtin_bit_cast(uint32x4, v), static_cast<uint32x4*>(p));
    else *static_cast<uint4*>(p) = v;
}
template <typename T, int N, bool STREAM>
__device__ __forceinline__ void rope_store(T* p, const float (&v)[N]) {
    if constexpr (N == 1) {
        if constexpr (sizeof(T) == 4) *p = v[0];
        else *p = static_cast<uint16_t>(cvt_pk_bf16(v[0], v[0]));  // (a NaN stays one)
    } else if constexpr (sizeof(T) == 4) {
        rope_store16<STREAM>(p, make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])));
    } else {
        rope_store16<STREAM>(p, make_uint4(cvt_pk_bf16(v[0], v[1]), cvt_pk_bf16(v[2], v[3]), cvt_pk_bf16(v[4], v[5]), cvt_pk_bf16(v[6], v[7])));
    }
}

}  // namespace

// A workgroup turns `chunk` heads of `rows` rows.  Its threads first make the rows' cosines and
// sines, one each, into LDS: every head of a row uses the same ones.  A unit is then N
// values and the N they are paired with (half layout), N values that are pairs (interleaved; of
// single values the pair), or N that are copied.  Bound by HBM, each value read and written once:
// the vectors of kRopeItems units are in flight per thread, the first ones while the angles are
// made.  8192 rows of 32 + 8 heads of 128, bf16: 30.1 us (5.6 TB/s; 38.2 with stores that stay in the
// caches, 67 with a thread a pair for all heads); 512 rows 6.0 us either way.
template <typename T, int N, bool STREAM>
__global__ __launch_bounds__(kRopeThreads) void rope_kernel(RopeArgs a) {
    extern __shared__ float2 angles[];  // [rows][pairs]
    const int tid = threadIdx.x;
    const int first_row = blockIdx.x * a.rows, first_head = blockIdx.y * a.chunk;
    const int rows = min(a.rows, a.tokens - first_row), heads = min(a.chunk, a.heads[0] + a.heads[1] - first_head);
    // units of a head: paired vectors, then copied ones
    const int paired = a.interleaved ? (N == 1 ? a.pairs : 2 * a.pairs / N) : a.pairs / N;
    const bool partner = !a.interleaved || N == 1;  // the second value of a pair lies elsewhere
    const int items = rows * a.chunk * a.units;

    struct Item {
        T* out;
        int at, second;  // its angles (-1: copied), and how far its partner lies
        int position;
    };
    Item item[kRopeItems];
    float x[kRopeItems][N], y[kRopeItems][N];
    auto load = [&](int i, int e) {
        Item& it = item[i];
        it.position = -1;
        if (e >= items) return;
        const int row = a.by_row ? __umulhi(e, a.by_row) : e;
        const int in_row = e - row * a.chunk * a.units;
        const int h = a.by_units ? __umulhi(in_row, a.by_units) : in_row, u = in_row - h * a.units;
        if (h >= heads) return;
        it.position = a.positions[first_row + row];  // (looked at behind the loads)
        int head = first_head + h;
        const int which = head >= a.heads[0];
        head -= which ? a.heads[0] : 0;
        const bool turned = u < paired;
        const int d = !turned ? 2 * a.pairs + (u - paired) * N : a.interleaved && N == 1 ? 2 * u : u * N;
        it.at = turned ? row * a.pairs + (a.interleaved && N > 1 ? d / 2 : a.interleaved ? u : d) : -1;
        it.second = turned && partner ? (a.interleaved ? 1 : a.pairs) : 0;
        const int64_t t = first_row + row, o = static_cast<int64_t>(head) * a.dim + d;
        const T* in = static_cast<const T*>(a.in[which]) + t * a.in_stride[which] + o;
        it.out = static_cast<T*>(a.out[which]) + t * a.out_stride[which] + o;
        rope_load<T, N>(in, x[i]);
        if (it.second) rope_load<T, N>(in + it.second, y[i]);
    };
#pragma unroll
    for (int i = 0; i < kRopeItems; ++i) load(i, tid + i * kRopeThreads);
    for (int e = tid; e < rows * a.pairs; e += kRopeThreads) {
        const int row = e / a.pairs;
        angles[e] = rope_angle(a.positions[first_row + row], a.turns[e - row * a.pairs], a.magnitude);
    }
    __syncthreads();
    for (int base = tid;; base += kRopeItems * kRopeThreads) {
#pragma unroll
        for (int i = 0; i < kRopeItems; ++i) {
            const Item& it = item[i];
            if (it.position < 0) continue;
            if (it.at < 0) {
                rope_store<T, N, STREAM>(it.out, x[i]);
            } else if (it.second) {
                float p[N], q[N];
#pragma unroll
                for (int j = 0; j < N; ++j) {
                    const float2 cs = angles[it.at + j];
                    p[j] = x[i][j] * cs.x - y[i][j] * cs.y;
                    q[j] = y[i][j] * cs.x + x[i][j] * cs.y;
                }
                rope_store<T, N, STREAM>(it.out, p);
                rope_store<T, N, STREAM>(it.out + it.second, q);
            } else if constexpr (N > 1) {
                float p[N];
#pragma unroll
                for (int j = 0; j < N; j += 2) {
                    const float2 cs = angles[it.at + j / 2];
                    p[j] = x[i][j] * cs.x - x[i][j + 1] * cs.y;
                    p[j + 1] = x[i][j + 1] * cs.x + x[i][j] * cs.y;
                }
                rope_store<T, N, STREAM>(it.out, p);
            }
        }
        if (base - tid + kRopeItems * kRopeThreads >= items) return;
#pragma unroll
        for (int i = 0; i < kRopeItems; ++i) load(i, base + (kRopeItems + i) * kRopeThreads);
    }
}

namespace {

// ceil(2^32 / d): its high product with x is x / d while x * d < 2^32 (0 stands for d = 1).
uint32_t reciprocal(uint32_t d) { return d == 1 ? 0 : static_cast<uint32_t>(((uint64_t{1} << 32) + d - 1) / d); }

template <typename T, int N>
void launch_rope_n(RopeArgs a, hipStream_t stream) {
    a.units = (a.interleaved ? (N == 1 ? a.pairs : 2 * a.pairs / N) : a.pairs / N) + (a.dim - 2 * a.pairs) / N;
    const int heads = a.heads[0] + a.heads[1];
    constexpr int kMost = 2 * kRopeItems * kRopeThreads;
    a.chunk = std::max(1, std::min(heads, (kMost + a.units - 1) / a.units));
    a.rows = std::max(1, std::min({a.tokens, kMost / (a.chunk * a.units), kMost / a.pairs}));
    a.by_units = reciprocal(a.units);
    a.by_row = reciprocal(a.chunk * a.units);
    const dim3 grid(static_cast<unsigned>((a.tokens + a.rows - 1) / a.rows), static_cast<unsigned>((heads + a.chunk - 1) / a.chunk));
    const size_t lds = a.rows * a.pairs * sizeof(float2);
    const bool streams = N > 1 && static_cast<int64_t>(a.tokens) * heads * a.dim * static_cast<int64_t>(sizeof(T)) >= kRopeStream;
    if (streams) rope_kernel<T, N, true><<<grid, kRopeThreads, lds, stream>>>(a);
    else rope_kernel<T, N, false><<<grid, kRopeThreads, lds, stream>>>(a);
}

}  // namespace

void launch_rope(const sfg_rope_args& s, hipStream_t stream) {
    RopeArgs a{};
    a.in[0] = s.q; a.in[1] = s.k; a.out[0] = s.q_out; a.out[1] = s.k_out;
    a.in_stride[0] = s.q_stride; a.in_stride[1] = s.k_stride;
    a.out_stride[0] = s.q_out_stride; a.out_stride[1] = s.k_out_stride;
    a.heads[0] = static_cast<int>(s.q_heads); a.heads[1] = static_cast<int>(s.kv_heads);
    a.positions = s.positions; a.turns = s.turns; a.magnitude = s.magnitude;
    a.tokens = static_cast<int>(s.tokens); a.dim = static_cast<int>(s.head_dim);
    a.pairs = static_cast<int>(s.rotary_dim / 2); a.interleaved = s.layout == SFG_ROPE_INTERLEAVED;
    // vectors of 16 bytes where heads, halves and rows begin on their borders
    const int64_t per = s.dtype == SFG_F32 ? 4 : 8;
    const bool vec = ((reinterpret_cast<uintptr_t>(s.q) | reinterpret_cast<uintptr_t>(s.k) | reinterpret_cast<uintptr_t>(s.q_out) |
                       reinterpret_cast<uintptr_t>(s.k_out)) & 15) == 0 &&
                     (a.in_stride[0] | a.in_stride[1] | a.out_stride[0] | a.out_stride[1] | a.dim) % per == 0 &&
                     (a.interleaved ? 2 * a.pairs : a.pairs) % per == 0;
    if (s.dtype == SFG_F32) vec ? launch_rope_n<float, 4>(a, stream) : launch_rope_n<float, 1>(a, stream);
    else vec ? launch_rope_n<uint16_t, 8>(a, stream) : launch_rope_n<uint16_t, 1>(a, stream);
}

}  // namespace sfg
