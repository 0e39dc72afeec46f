// MXFP4 (OCP Microscaling Formats 1.0): values of four bits (e2m1: sign, two exponent bits, one of the mantissa -- 0, 0.5, 1, 1.5, 2, 3, 4,
// 6), 32 consecutive ones of a row with one power of two (e8m0: the byte s stands for 2^(s - 127), 255 for NaN).  A row of K values (a
// multiple of 32) is K / 2 bytes of codes, the value of the even index in the low half, and K / 32 bytes of scales, both row-major.
#pragma once

#include "moe_internal.hpp"

namespace moe355 {
namespace {

constexpr int kMxBlock = 32;               // values that share a scale
constexpr uint32_t kMxScaleNan = 255;      // its e8m0 code
constexpr uint32_t kMxScaleOne = 127;

typedef __bf16 mx_bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 mx_bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 mx_f16x2 __attribute__((ext_vector_type(2)));
typedef float mx_f32x2 __attribute__((ext_vector_type(2)));
typedef float mx_f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t mx_u32x4 __attribute__((ext_vector_type(4)));
typedef int mx_i32x8 __attribute__((ext_vector_type(8)));

// The scale as the conversions of gfx950 take it, a float of which they read the exponent field alone: field 0 is 2^-127 to them and 255
// NaN, as in e8m0, so every byte is the field as it is.
__device__ __forceinline__ float mx_scale(uint32_t e8m0) { return __uint_as_float(e8m0 << 23); }

// Eight codes -> eight bf16, exact (two significant bits; the smallest value, 2^-128, is a subnormal bf16).  With a scale from 253 on the
// largest overflow to infinity, as they do in fp32.
__device__ __forceinline__ mx_bf16x8 mx_widen8(uint32_t codes, float scale) {
    union {
        mx_bf16x8 v;
        mx_bf16x2 p[4];
    } r;
    r.p[0] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 0);
    r.p[1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 1);
    r.p[2] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 2);
    r.p[3] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 3);
    return r.v;
}

}  // namespace
}  // namespace moe355
