// Rows and weights to MXFP4 and back (mxfp4.hpp has the format).
//
// The scale of 32 values with the largest magnitude amax is 2^(floor(log2 amax) - 2) -- 2 is the exponent of e2m1's largest binade --, not
// below 2^-127; a value is x / scale rounded to the nearest even code, and to +-6 beyond it (amax / scale lies in [4, 8)).  The exponent
// of amax is its fp32 exponent field E, so the scale's byte is max(E - 2, 0): no logarithm, and the division is exact.  A block of zeros
// has scale 1.  The format has no infinity and no NaN among its codes: a block that holds either gets the scale NaN, so that it shows.
//
// Blocks follow each other in memory as rows do, so the pass knows no rows: a flat array of 32-value blocks.  Bound by memory: four lanes
// share a block, 16 bytes of 16-bit values each, so that loads and stores are whole lines; a wavefront takes four times 512 values
// at once to have that many loads in flight, and its lanes keep one scale each of the 64 for a single store of a whole piece.
// 114688 x 4096 bf16 values: 215 to 235 us to codes (5.3 TB/s read and written), 185 back (6.4); 64 x 7168, 2.8 and 2.6, a launch.
#include "mxfp4.hpp"

namespace moe355 {
namespace {

constexpr int kUnroll = 4;                           // pieces of 512 values a wavefront has in flight
constexpr int kWaveValues = 512 * kUnroll;

struct f32_s { float v; };

// Eight values of a lane as they lie in memory.
template <class T> struct Eight { mx_u32x4 w; };
template <> struct Eight<f32_s> { mx_u32x4 w, w1; };

template <class T>
__device__ __forceinline__ Eight<T> load8(const void* p, int64_t i) {
    Eight<T> r;
    if constexpr (std::is_same<T, f32_s>::value) {
        r.w = reinterpret_cast<const mx_u32x4*>(p)[2 * i];
        r.w1 = reinterpret_cast<const mx_u32x4*>(p)[2 * i + 1];
    } else {
        r.w = reinterpret_cast<const mx_u32x4*>(p)[i];
    }
    return r;
}

// The exponent field of the largest magnitude of the four lanes' values, as of fp32 (255: an infinity or a NaN), and whether all are zero.
// Magnitudes order as their bit patterns do, NaN above infinity.
template <class T>
__device__ __forceinline__ uint32_t block_scale(const Eight<T>& x) {
    uint32_t m = 0;
    if constexpr (std::is_same<T, f32_s>::value) {
#pragma unroll
        for (int i = 0; i < 4; ++i) m = max(m, max(x.w[i] & 0x7FFFFFFFu, x.w1[i] & 0x7FFFFFFFu));
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) m = max(m, max(x.w[i] & 0x7FFFu, (x.w[i] >> 16) & 0x7FFFu));
    }
    m = max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0xB1, 0xF, 0xF, false));     // quad_perm [1,0,3,2]
    m = max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0x4E, 0xF, 0xF, false));     // quad_perm [2,3,0,1]
    if (m == 0) return kMxScaleOne;
    uint32_t e;
    if constexpr (std::is_same<T, f32_s>::value) e = m >> 23;
    else if constexpr (std::is_same<T, bf16_s>::value) e = m >> 7;
    else e = __float_as_uint((float)__builtin_bit_cast(_Float16, (uint16_t)m)) >> 23;         // subnormal halves are normal floats
    if (e == 255) return kMxScaleNan;
    return e > 2 ? e - 2 : 0;
}

// Values 2 I and 2 I + 1 into byte I of the codes.
template <int I, class T>
__device__ __forceinline__ uint32_t narrow2(uint32_t c, const Eight<T>& x, float scale) {
    if constexpr (std::is_same<T, f32_s>::value) {
        const mx_u32x4& h = I < 2 ? x.w : x.w1;
        return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, __uint_as_float(h[2 * (I & 1)]), __uint_as_float(h[2 * (I & 1) + 1]), scale, I);
    } else {
        const uint32_t pair = x.w[I];
        if constexpr (std::is_same<T, bf16_s>::value) return __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(mx_bf16x2, pair), scale, I);
        else return __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(c, __builtin_bit_cast(mx_f16x2, pair), scale, I);
    }
}
template <class T>
__device__ __forceinline__ uint32_t narrow8(const Eight<T>& x, float scale) {
    return narrow2<3, T>(narrow2<2, T>(narrow2<1, T>(narrow2<0, T>(0u, x, scale), x, scale), x, scale), x, scale);
}

// blocks: 32-value blocks of the whole array.
template <class T>
__global__ __launch_bounds__(256) void quant_mxfp4_kernel(const void* __restrict__ x, uint32_t* __restrict__ codes, uint8_t* __restrict__ scales, int64_t blocks) {
    const int lane = threadIdx.x & 63;
    const int64_t wave = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int64_t block0 = wave * (kWaveValues / kMxBlock);
    if (block0 >= blocks) return;
    const int64_t eights = blocks * 4, first = block0 * 4 + lane;
    Eight<T> v[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) v[u] = load8<T>(x, min(first + 64 * u, eights - 1));      // behind the end: the last again, not stored
    uint32_t mine = 0;
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
        const uint32_t s = block_scale<T>(v[u]);
        const uint32_t c = s == kMxScaleNan ? 0u : narrow8<T>(v[u], mx_scale(s));
        if (first + 64 * u < eights) codes[first + 64 * u] = c;
        if ((lane & 3) == u) mine = s;
    }
    // lane 4 b + u holds the scale of block b of piece u
    const int64_t b = block0 + 16 * (lane & 3) + (lane >> 2);
    if (b < blocks) scales[b] = (uint8_t)mine;
}

template <class T>
__device__ __forceinline__ void widen_store8(void* out, int64_t i, uint32_t c, float s) {
    if constexpr (std::is_same<T, f32_s>::value) {
        mx_f32x2 p[4] = {__builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, s, 0), __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, s, 1),
                         __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, s, 2), __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, s, 3)};
        reinterpret_cast<mx_f32x4*>(out)[2 * i] = mx_f32x4{p[0][0], p[0][1], p[1][0], p[1][1]};
        reinterpret_cast<mx_f32x4*>(out)[2 * i + 1] = mx_f32x4{p[2][0], p[2][1], p[3][0], p[3][1]};
    } else if constexpr (std::is_same<T, bf16_s>::value) {
        reinterpret_cast<mx_u32x4*>(out)[i] = __builtin_bit_cast(mx_u32x4, mx_widen8(c, s));
    } else {
        mx_f16x2 p[4] = {__builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c, s, 0), __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c, s, 1),
                         __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c, s, 2), __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c, s, 3)};
        mx_u32x4 w;
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = __builtin_bit_cast(uint32_t, p[j]);
        reinterpret_cast<mx_u32x4*>(out)[i] = w;
    }
}

template <class T>
__global__ __launch_bounds__(256) void dequant_mxfp4_kernel(const uint32_t* __restrict__ codes, const uint8_t* __restrict__ scales, void* __restrict__ out, int64_t blocks) {
    const int lane = threadIdx.x & 63;
    const int64_t wave = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int64_t first = wave * (kWaveValues / 8) + lane, eights = blocks * 4;
    uint32_t c[kUnroll], s[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
        const int64_t i = min(first + 64 * u, eights - 1);
        c[u] = codes[i];
        s[u] = scales[i >> 2];
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
        if (first + 64 * u < eights) widen_store8<T>(out, first + 64 * u, c[u], mx_scale(s[u]));
}

}  // namespace

hipError_t launch_quant_mxfp4(const void* x, int dtype, int64_t values, void* codes, uint8_t* scales, hipStream_t st) {
    if (values <= 0) return hipSuccess;
    const unsigned grid = (unsigned)((values + 4 * kWaveValues - 1) / (4 * kWaveValues));
    const int64_t blocks = values / kMxBlock;
    if (dtype == MOE_DTYPE_F32) quant_mxfp4_kernel<f32_s><<<grid, 256, 0, st>>>(x, (uint32_t*)codes, scales, blocks);
    else if (dtype == MOE_DTYPE_BF16) quant_mxfp4_kernel<bf16_s><<<grid, 256, 0, st>>>(x, (uint32_t*)codes, scales, blocks);
    else quant_mxfp4_kernel<f16_s><<<grid, 256, 0, st>>>(x, (uint32_t*)codes, scales, blocks);
    return hipGetLastError();
}

hipError_t launch_dequant_mxfp4(const void* codes, const uint8_t* scales, int64_t values, int dtype, void* out, hipStream_t st) {
    if (values <= 0) return hipSuccess;
    const unsigned grid = (unsigned)((values + 4 * kWaveValues - 1) / (4 * kWaveValues));
    const int64_t blocks = values / kMxBlock;
    if (dtype == MOE_DTYPE_F32) dequant_mxfp4_kernel<f32_s><<<grid, 256, 0, st>>>((const uint32_t*)codes, scales, out, blocks);
    else if (dtype == MOE_DTYPE_BF16) dequant_mxfp4_kernel<bf16_s><<<grid, 256, 0, st>>>((const uint32_t*)codes, scales, out, blocks);
    else dequant_mxfp4_kernel<f16_s><<<grid, 256, 0, st>>>((const uint32_t*)codes, scales, out, blocks);
    return hipGetLastError();
}

}  // namespace moe355

using namespace moe355;

namespace {
// rows of K values that the flat passes take, in `at` (aligned to `align` bytes) and the codes
bool mx_array_ok(const void* at, const void* codes, const void* scales, int64_t rows, int64_t K) {
    if (rows < 0 || K < kMxBlock || K % kMxBlock || rows > INT64_MAX / K) return false;
    if (rows * K > (int64_t)0xFFFFFF * 4 * kWaveValues) return false;         // threads of a launch
    if (rows == 0) return true;
    return at && codes && scales && (uintptr_t)at % 16 == 0 && (uintptr_t)codes % 4 == 0;
}
bool mx_float(int32_t dtype) { return dtype == MOE_DTYPE_F32 || dtype == MOE_DTYPE_BF16 || dtype == MOE_DTYPE_FP16; }
}  // namespace

extern "C" int moe_quant_mxfp4(const void* x, int32_t src_dtype, int64_t rows, int64_t K, void* codes, uint8_t* scales, void* stream) {
    if (!mx_array_ok(x, codes, scales, rows, K)) return MOE_ERR_BAD_ARGUMENT;
    if (!mx_float(src_dtype)) return MOE_ERR_UNSUPPORTED;
    return launch_quant_mxfp4(x, src_dtype, rows * K, codes, scales, (hipStream_t)stream) == hipSuccess ? MOE_OK : MOE_ERR_HIP;
}

extern "C" int moe_dequant_mxfp4(const void* codes, const uint8_t* scales, int64_t rows, int64_t K, int32_t dst_dtype, void* out, void* stream) {
    if (!mx_array_ok(out, codes, scales, rows, K)) return MOE_ERR_BAD_ARGUMENT;
    if (!mx_float(dst_dtype)) return MOE_ERR_UNSUPPORTED;
    return launch_dequant_mxfp4(codes, scales, rows * K, dst_dtype, out, (hipStream_t)stream) == hipSuccess ? MOE_OK : MOE_ERR_HIP;
}
