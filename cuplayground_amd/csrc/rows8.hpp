// Rows in e4m3 with one fp32 scale for 128 values of a row (the format of moe_quant_rows128), for kernels that make them of sums in fp32:
// scale = amax / 448 -- not below 2^-126, 1 where all are zero -- and code = e4m3(v / scale), to the nearest, halves to even.  A piece with an
// infinity in it has an infinite scale, so all of it reads as NaN; a NaN is a NaN's code and leaves the others alone.
#pragma once

#include "moe_internal.hpp"

namespace moe355 {
namespace {

constexpr int kRows8Piece = 128;      // values that share a scale

// Lanes of a row of 16, turned by N places: a DPP move, which the operation that takes it does on its way.
template <int N>
__device__ __forceinline__ float row_turned(float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x120 + N, 0xF, 0xF, true));
}
// The maximum over 16 or 32 neighbouring lanes, in all of them.  (fmaxf passes over a NaN.)
template <int LANES>
__device__ __forceinline__ float rows8_max(float v) {
    static_assert(LANES == 16 || LANES == 32, "rows of lanes");
    v = fmaxf(v, row_turned<8>(v));
    v = fmaxf(v, row_turned<4>(v));
    v = fmaxf(v, row_turned<2>(v));
    v = fmaxf(v, row_turned<1>(v));
    if constexpr (LANES == 32) v = fmaxf(v, __shfl_xor(v, 16, kWave));
    return v;
}
__device__ __forceinline__ float rows8_scale(float amax) { return amax > 0.0f ? fmaxf(amax / 448.0f, 0x1p-126f) : 1.0f; }

// Four values -> four codes.  The quotient is the product with the scale's reciprocal, corrected once by its remainder: two fused operations
// where the IEEE division has ten, and the same number but for the last place now and then, which an e4m3 rounding sees as seldom.  No quotient
// is above 448 by more than that, so the conversion, which would make a NaN of 480, has nothing to clamp.  An infinite scale's reciprocal is 0 and the
// remainder of anything a NaN.
__device__ __forceinline__ uint32_t rows8_codes(float a, float b, float c, float d, float scale, float inverse) {
    auto quotient = [&](float v) {
        const float q = v * inverse;
        return __builtin_fmaf(__builtin_fmaf(-q, scale, v), inverse, q);
    };
    int r = __builtin_amdgcn_cvt_pk_fp8_f32(quotient(a), quotient(b), 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(quotient(c), quotient(d), r, true);
}

}  // namespace
}  // namespace moe355
