// sfg_paged.hpp -- what the kernels over the paged KV pools share
// (K [page][Hkv][page_tokens][D], V [page][Hkv][D][page_tokens]).
#pragma once

#include "sfg_device.hpp"

namespace sfg {

constexpr int kRowMaxD = 256;  // head_dim of the row-per-wave kernels
constexpr int kPageTok = 16;   // page size of the matrix-core kernels

typedef short short4v __attribute__((ext_vector_type(4)));

__device__ __forceinline__ short4v as_short4(const uint2& v) { return __builtin_bit_cast(short4v, v); }

// An fp32 operand of the bf16 matrix instructions as three bf16 terms (24 bits).
struct Bf16x3 {
    bf16x8 t[3];
};
// (truncated terms: a rounded leading one could overflow to infinity)
__device__ __forceinline__ void split3(float v, uint16_t& hi, uint16_t& mid, uint16_t& lo) {
    hi = static_cast<uint16_t>(__float_as_uint(v) >> 16);
    const float r = v - bf16_to_f32(hi);
    mid = static_cast<uint16_t>(__float_as_uint(r) >> 16);
    lo = static_cast<uint16_t>(__float_as_uint(r - bf16_to_f32(mid)) >> 16);
}
// Two softmax weights as two bf16 terms each, packed: the leading one truncated, the second
// what is left of p (1 + 2^-23), rounded (2^-15 of p at most, and the 2^-23).  Both terms are
// positive wherever p is, so that an infinity times them keeps its sign and is not 0 * inf.
__device__ __forceinline__ void split2_weights(float p0, float p1, uint32_t& hi, uint32_t& lo) {
    const uint32_t u0 = __float_as_uint(p0), u1 = __float_as_uint(p1);
    hi = __builtin_amdgcn_perm(u1, u0, 0x07060302u);
    lo = cvt_pk_bf16(fmaf(p0, 1.0f + 0x1p-23f, -__uint_as_float(u0 & 0xFFFF0000u)),
                     fmaf(p1, 1.0f + 0x1p-23f, -__uint_as_float(u1 & 0xFFFF0000u)));
}
// two bf16 values, the infinite and NaN ones replaced by zero
__device__ __forceinline__ uint32_t finite_bf16x2(uint32_t w) {
    const uint32_t bad = ((w & 0x7F807F80u) + 0x00800080u) & 0x80008000u;  // exponent all ones
    return w & ~((bad >> 15) * 0xFFFFu);
}

// Sum of the lanes up to this one, by DPP: row shifts, then the rows' totals broadcast.
__device__ __forceinline__ int wave_inclusive(int x) {
    x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xF, 0xF, false);  // row_shr:1
    x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xF, 0xF, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xF, 0xF, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xF, 0xF, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xA, 0xF, false);  // row_bcast:15 to rows 1, 3
    x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xC, 0xF, false);  // row_bcast:31 to rows 2, 3
    return x;
}
template <typename KvT>
__device__ __forceinline__ float kv_f32(const KvT* p, int64_t i) {
    if constexpr (sizeof(KvT) == 4) return p[i];
    else return bf16_to_f32(p[i]);
}

}  // namespace sfg
