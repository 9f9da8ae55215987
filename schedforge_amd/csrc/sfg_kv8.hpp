// sfg_kv8.hpp -- what the kernels of a step over an 8-bit paged cache share: codes and
// values, and the launchers that sfg_api_kv8.hip calls with checked arguments.
#pragma once

#include "../../include/sfg_hip.h"
#include "sfg_paged.hpp"

namespace sfg {

constexpr float kMostI8 = 127.0f, kMostFp8 = 448.0f;  // the largest codes

// The value of byte b: int8, or e4m3 (hardware conversion, exact).
template <bool FP8>
__device__ __forceinline__ float kv8_value(uint8_t b) {
    if constexpr (FP8) return __builtin_amdgcn_cvt_f32_fp8(b, 0);
    else return static_cast<float>(static_cast<int8_t>(b));
}

// The code of v under `scale`: the IEEE quotient in fp32, rounded to the nearest code, ties
// to even (v_rndne_f32; v_cvt_pk_fp8_f32), cut to the largest one; 0 unless scale > 0.
template <bool FP8>
__device__ __forceinline__ uint8_t kv8_code(float v, float scale) {
    if (!(scale > 0.0f)) return 0;
    constexpr float most = FP8 ? kMostFp8 : kMostI8;
    const float y = fminf(fmaxf(__fdiv_rn(v, scale), -most), most);
    if constexpr (FP8) return static_cast<uint8_t>(__builtin_amdgcn_cvt_pk_fp8_f32(y, y, 0, false));
    else return static_cast<uint8_t>(static_cast<int>(rintf(y)));
}

// The scale that holds values up to the one whose magnitude has these bits; NaN for an
// infinity or a NaN.
template <bool FP8>
__device__ __forceinline__ float kv8_scale(uint32_t top) {
    if (top >= 0x7F800000u) return __uint_as_float(0x7FC00000u);
    return __fdiv_rn(__uint_as_float(top), FP8 ? kMostFp8 : kMostI8);
}

// The larger of two scales, NaN if one is.
__device__ __forceinline__ float kv8_larger(float a, float b) { return a >= b || a != a ? a : b; }

void launch_kv_plan(const sfg_kv_plan_args& a, hipStream_t stream);
void launch_rope(const sfg_rope_args& a, hipStream_t stream);
void launch_kv8_append(const sfg_kv8_append_args& a, hipStream_t stream);
// How an attention runs.  A unit is a block of at most `width` columns of a sequence over the
// tiles it sees.  share: the workgroups a kv head that all tiles are dealt to if there are more than
// `few` for each; with fewer, units are split into pieces of `least` tiles or more, at most
// share and the units together.  quads (0: never): with so many tiles of all heads, a workgroup
// takes four heads, and there are four times as many shares.  fixed: pieces a unit, instead of
// all that.  row_shift: a block has 2^row_shift whole rows (-1: it has not).  slots: partial
// results a kv head, at most; groups: workgroups.  bytes: 0 if no unit is split.  Units run whole (fixed
// 1, share 0) where the bounds' partial results pass 128 MiB or their costs the 32-bit sums: two sequences of
// 131072 tokens take 70 us under a bound of one row, 1377 under one of 8192.
struct Kv8Plan {
    bool mfma;
    int nt, waves, width, slots, groups, share, quads, fixed, least, few, row_shift;
    size_t bytes;
};
Kv8Plan plan_attn_kv8(const sfg_kv8_attn_args& a);
size_t workspace_attn_kv8(const sfg_kv8_attn_args& a);  // for these and all shorter bounds: plans' bytes or more
void launch_attn_kv8(const sfg_kv8_attn_args& a, const Kv8Plan& plan, void* workspace, hipStream_t stream);

}  // namespace sfg
