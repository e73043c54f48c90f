// Matrix products with codes of 4-bit caches: 16 x 16 x 32 products, the codes as 16-bit
// numbers, and sums over the four quarters of a wave that such a product's columns lie in.
#pragma once

#include "fta_common.h"
#include "fta_tile.h"

template <int DT>
__device__ __forceinline__ f32x4 fta_mma16(fta_frag a, fta_frag b, f32x4 c) {
    if constexpr (DT == FTA_DTYPE_BF16)
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(fta_bf16x8, a), __builtin_bit_cast(fta_bf16x8, b), c,
                                                       0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(fta_f16x8, a), __builtin_bit_cast(fta_f16x8, b), c, 0,
                                                      0, 0);
}

// Eight codes as 16-bit numbers 16 + n: the code is the upper half of the mantissa of a number whose
// exponent says 16.  Two codes take a shift and an and-or.  Pairs (0, 4), (1, 5), (2, 6), (3, 7).
template <int DT>
constexpr uint32_t kFtaSixteen = DT == FTA_DTYPE_BF16 ? 0x41804180u : 0x4c004c00u;
// A constant held in a vector register: an and-or takes one scalar operand, and has the mask for it.
__device__ __forceinline__ uint32_t fta_in_vgpr(uint32_t x) {
    asm volatile("" : "+v"(x));
    return x;
}
template <int DT>
__device__ __forceinline__ fta_frag fta_codes16(uint32_t w, uint32_t sixteen) {
    constexpr uint32_t mask = DT == FTA_DTYPE_BF16 ? 0x00780078u : 0x03c003c0u;
    constexpr int up = DT == FTA_DTYPE_BF16 ? 3 : 6;
    fta_frag f;
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = ((up >= 4 * i ? w << (up - 4 * i) : w >> (4 * i - up)) & mask) | sixteen;
    return f;
}
// Eight 16-bit values in that order of pairs.
__device__ __forceinline__ fta_frag fta_paired(fta_frag x) {
    return fta_frag{(x[0] & 0xffffu) | x[2] << 16, x[0] >> 16 | (x[2] & 0xffff0000u), (x[1] & 0xffffu) | x[3] << 16,
                    x[1] >> 16 | (x[3] & 0xffff0000u)};
}

// Lanes 16 .. 31 of a with 0 .. 15 of b, 48 .. 63 with 32 .. 47 (v_permlane16_swap on two
// registers; through asm with its waits, as fta_swap32).
__device__ __forceinline__ void fta_swap16(float& a, float& b) {
    asm volatile("s_nop 1\n\tv_permlane16_swap_b32 %0, %1\n\ts_nop 1" : "+v"(a), "+v"(b));
}
// Sum and maximum over lanes l, l ^ 16, l ^ 32, l ^ 48.
__device__ __forceinline__ float fta_sum_quarters(float x) {
    float y = x;
    fta_swap16(x, y);
    x += y;
    y = x;
    fta_swap32(x, y);
    return x + y;
}
__device__ __forceinline__ float fta_max_quarters(float x) {
    float y = x;
    fta_swap16(x, y);
    x = fmaxf(x, y);
    y = x;
    fta_swap32(x, y);
    return fmaxf(x, y);
}
