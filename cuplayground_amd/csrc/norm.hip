// The root-mean-square norm of a residual stream, and what else makes rows in e4m3 for the products with block scales.
//
//   h = round(x + residual)         (without a residual: x; the stream keeps h in its own type, and what it keeps is what is normalised)
//   y = h r w,  r = 1 / sqrt(mean(h^2) + eps)
//   dx = r (dy w - n mean(dy w n)) + dsum,  n = h r;   dw = sum over rows of dy n
//
// Memory bounds all of it: every array passes once.  A row stays in the registers of the threads that fetched it, 16 bytes of every operand a
// thread and step, from the sum of its squares to its results.  8192 rows of 4096 in bf16 with a residual, kernel times on three inputs in turn, least to
// median: the norm 45 to 48 us (5.6 to 5.9 TB/s; a copy of 1 GiB reaches 5.15 here, one of 128 MiB 7.2), in e4m3 and bf16 55 to 59, the gradients 51 to 54
// (with one of the sum; 44 to 46 without) and 4 for the weight's.
#include "ffn_common.hpp"
#include "mxfp4.hpp"
#include "rows8.hpp"

namespace moe355 {
namespace {

// ---- elements ----
struct f32_e { typedef float raw; };
struct bf16_e { typedef uint16_t raw; };
struct f16_e { typedef uint16_t raw; };
template <class T> __device__ __forceinline__ float widen(typename T::raw v);
template <> __device__ __forceinline__ float widen<f32_e>(float v) { return v; }
template <> __device__ __forceinline__ float widen<bf16_e>(uint16_t v) { return bf16_bits_to_f32(v); }
template <> __device__ __forceinline__ float widen<f16_e>(uint16_t v) { return (float)__builtin_bit_cast(_Float16, v); }
template <class T> __device__ __forceinline__ typename T::raw narrow(float v);
template <> __device__ __forceinline__ float narrow<f32_e>(float v) { return v; }
template <> __device__ __forceinline__ uint16_t narrow<bf16_e>(float v) { return __builtin_bit_cast(uint16_t, (__bf16)v); }
template <> __device__ __forceinline__ uint16_t narrow<f16_e>(float v) { return __builtin_bit_cast(uint16_t, (_Float16)v); }

// 16 bytes of neighbouring elements, fetched and stored as one.  WHOLE: rows begin on 16 bytes and end with a piece; else a piece lies anywhere that an
// element can (memory takes 16 bytes from any address), and the last of a row may have fewer elements: those behind the row's end are zeros,
// and are not stored.
template <class T> constexpr int kNormVec = 16 / (int)sizeof(typename T::raw);
template <class RAW>
struct alignas(16) Piece { RAW e[16 / sizeof(RAW)]; };
template <class T, bool WHOLE>
__device__ __forceinline__ Piece<typename T::raw> load(const void* p, int64_t element, int left) {
    typedef typename T::raw RAW;
    const RAW* at = static_cast<const RAW*>(p) + element;
    if constexpr (WHOLE) {
        return *reinterpret_cast<const Piece<RAW>*>(at);
    } else {
        Piece<RAW> v = {};
        if (left >= kNormVec<T>) {
            __builtin_memcpy(&v, at, 16);
        } else {
#pragma unroll
            for (int k = 0; k < kNormVec<T>; ++k)
                if (k < left) v.e[k] = at[k];
        }
        return v;
    }
}
template <class T, bool WHOLE>
__device__ __forceinline__ void store(void* p, int64_t element, int left, const Piece<typename T::raw>& v) {
    typedef typename T::raw RAW;
    RAW* at = static_cast<RAW*>(p) + element;
    if constexpr (WHOLE) {
        *reinterpret_cast<Piece<RAW>*>(at) = v;
    } else if (left >= kNormVec<T>) {
        __builtin_memcpy(at, &v, 16);
    } else {
#pragma unroll
        for (int k = 0; k < kNormVec<T>; ++k)
            if (k < left) at[k] = v.e[k];
    }
}
// Of the norm's weights, in the rows' type or in fp32.
template <class T, bool WHOLE>
__device__ __forceinline__ void load_weights(float (&w)[kNormVec<T>], const void* p, bool f32, int c, int left) {
    constexpr int VEC = kNormVec<T>;
    if (f32) {
#pragma unroll
        for (int i = 0; i < VEC; i += 4) {
            const auto v = load<f32_e, WHOLE>(p, c + i, left - i);
#pragma unroll
            for (int k = 0; k < 4; ++k) w[i + k] = v.e[k];
        }
    } else {
        const auto v = load<T, WHOLE>(p, c, left);
#pragma unroll
        for (int i = 0; i < VEC; ++i) w[i] = widen<T>(v.e[i]);
    }
}

// ---- sums over the threads of a row, in a fixed order, in all of them ----
__device__ __forceinline__ float wave_sum(float v) {
    v += row_turned<8>(v);
    v += row_turned<4>(v);
    v += row_turned<2>(v);
    v += row_turned<1>(v);
    // of both rows of either half, then of both halves: what a swap leaves in its two results
    const uint32_t r = __float_as_uint(v);
    const auto rows = __builtin_amdgcn_permlane16_swap(r, r, false, false);
    const uint32_t h = __float_as_uint(__uint_as_float(rows[0]) + __uint_as_float(rows[1]));
    const auto halves = __builtin_amdgcn_permlane32_swap(h, h, false, false);
    return __uint_as_float(halves[0]) + __uint_as_float(halves[1]);
}
// N sums at once; part: [N][waves of the row], of this row alone.
template <int THREADS, int N>
__device__ __forceinline__ void row_sums(float (&v)[N], float* part) {
#pragma unroll
    for (int n = 0; n < N; ++n) v[n] = wave_sum(v[n]);
    if constexpr (THREADS > kWave) {
        constexpr int W = THREADS / kWave;
        if ((threadIdx.x & 63) == 0) {
#pragma unroll
            for (int n = 0; n < N; ++n) part[n * W + (threadIdx.x >> 6)] = v[n];
        }
        __syncthreads();
#pragma unroll
        for (int n = 0; n < N; ++n) {
            float s = part[n * W];
#pragma unroll
            for (int i = 1; i < W; ++i) s += part[n * W + i];
            v[n] = s;
        }
    }
}

// The squares' sum of a row may pass fp32 where their mean does not, and a value may be larger than any whose square fp32 holds.  Such a row is summed
// again from its values times this: no sum is above 2^126 then, the product is exact but for values below 2^-54 (whose n is below 2^-111 in such a
// row), and r takes the factor back (21 bits of it at least where r is below fp32's normal numbers).  fp16 has no such rows.
constexpr float kFarRow = 0x1p-72f;
template <class T> constexpr bool kHasFarRows = true;
template <> constexpr bool kHasFarRows<f16_e> = false;

// THREADS threads to a row, NV pieces each; of rows that a wavefront holds, four share a workgroup.
template <int THREADS> constexpr int kNormBlock = THREADS == kWave ? 4 * kWave : THREADS;

template <class T, int NV, int THREADS, bool WHOLE, bool Q8>
__global__ __launch_bounds__(kNormBlock<THREADS>) void norm_rows_kernel(NormArgs a) {
    constexpr int ROWS = kNormBlock<THREADS> / THREADS, VEC = kNormVec<T>;
    typedef Piece<typename T::raw> P;
    __shared__ float part[THREADS / kWave];
    const int64_t row = (int64_t)blockIdx.x * ROWS + threadIdx.x / THREADS;
    const int t = threadIdx.x % THREADS;
    if (ROWS > 1 && row >= a.rows) return;        // (whole wavefronts, which meet nobody)
    const int64_t at = row * a.H;
    P x[NV], res[NV];
    float w[NV][VEC], h[NV][VEC];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (t + THREADS * i) * VEC;
        if (c < a.H) x[i] = load<T, WHOLE>(a.x, at + c, a.H - c);
    }
    if (a.residual) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (t + THREADS * i) * VEC;
            if (c < a.H) res[i] = load<T, WHOLE>(a.residual, at + c, a.H - c);
        }
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (t + THREADS * i) * VEC;
        if (c < a.H) load_weights<T, WHOLE>(w[i], a.weight, a.weight_f32, c, a.H - c);
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (t + THREADS * i) * VEC;
        if (c >= a.H) continue;
        if (a.residual) {
#pragma unroll
            for (int k = 0; k < VEC; ++k) x[i].e[k] = narrow<T>(widen<T>(x[i].e[k]) + widen<T>(res[i].e[k]));
            store<T, WHOLE>(a.sum, at + c, a.H - c, x[i]);
        }
#pragma unroll
        for (int k = 0; k < VEC; ++k) h[i][k] = widen<T>(x[i].e[k]);
    }
    float sum[1], mean, far = 1.0f;
    for (;;) {
        sum[0] = 0.0f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            if ((t + THREADS * i) * VEC >= a.H) continue;
#pragma unroll
            for (int k = 0; k < VEC; ++k) sum[0] = __builtin_fmaf(h[i][k] * far, h[i][k] * far, sum[0]);
        }
        row_sums<THREADS, 1>(sum, part);
        mean = sum[0] / (float)a.H + a.eps * far * far;
        if (!kHasFarRows<T> || mean < INFINITY || far != 1.0f) break;      // (the same in all threads of the row)
        far = kFarRow;
        if (THREADS > kWave) __syncthreads();     // (everybody has read the sums)
    }
    const float r = 1.0f / sqrtf(mean) * far;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (t + THREADS * i) * VEC;
        if (c >= a.H) continue;                   // (Q8: H is whole pieces of 128, so the lanes of a piece agree)
        float y[VEC];
#pragma unroll
        for (int k = 0; k < VEC; ++k) y[k] = h[i][k] * r * w[i][k];
        if (a.out) {
            P o;
#pragma unroll
            for (int k = 0; k < VEC; ++k) o.e[k] = narrow<T>(y[k]);
            store<T, WHOLE>(a.out, at + c, a.H - c, o);
        }
        if constexpr (Q8) {
            constexpr int LANES = kRows8Piece / VEC;
            struct alignas(VEC) Codes { uint32_t e[VEC / 4]; } q;
            float amax = 0.0f;
#pragma unroll
            for (int k = 0; k < VEC; ++k) amax = fmaxf(amax, fabsf(y[k]));
            const float s = rows8_scale(rows8_max<LANES>(amax)), inverse = 1.0f / s;
            if (t % LANES == 0) a.scales[row * (a.H / kRows8Piece) + c / kRows8Piece] = s;
#pragma unroll
            for (int k = 0; k < VEC; k += 4) q.e[k / 4] = rows8_codes(y[k], y[k + 1], y[k + 2], y[k + 3], s, inverse);
            *reinterpret_cast<Codes*>(a.q + at + c) = q;
        }
    }
}

// The gradients.  A workgroup takes every gridDim.x-th row (ROWS of them at a time) and keeps its threads' columns of dw in registers; what it has of dw
// at the end is a row of `part`, and norm_weight_grad_kernel adds those up in their order: no atomics, the same bits every time.  The next
// row's operands are on their way while a row's sums are made, where a thread's share of a row is small.  (Of fp32 rows above 8192 values 36 bytes a
// lane spill to scratch memory, 44 where rows begin on no 16 bytes: 2048 x 16384 with a gradient of the sum 124 us, 4.3 TB/s.)
template <class T, int NV, int THREADS, bool WHOLE>
__global__ __launch_bounds__(kNormBlock<THREADS>) void norm_backward_kernel(NormBackwardArgs a) {
    constexpr int ROWS = kNormBlock<THREADS> / THREADS, VEC = kNormVec<T>;
    typedef Piece<typename T::raw> P;
    __shared__ float part[2][2 * (THREADS / kWave)];
    const int t = threadIdx.x % THREADS;
    const int64_t step = (int64_t)gridDim.x * ROWS;
    float w[NV][VEC], dw[NV][VEC];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (t + THREADS * i) * VEC;
#pragma unroll
        for (int k = 0; k < VEC; ++k) w[i][k] = dw[i][k] = 0.0f;
        if (c < a.H) load_weights<T, WHOLE>(w[i], a.weight, a.weight_f32, c, a.H - c);
    }
    struct Operands { P h[NV], dy[NV], ds[NV]; };
    auto fetch = [&](int64_t row, Operands& o) {
        if (row >= a.rows) return;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (t + THREADS * i) * VEC;
            if (c >= a.H) continue;
            o.h[i] = load<T, WHOLE>(a.h, row * a.H + c, a.H - c);
            o.dy[i] = load<T, WHOLE>(a.dy, row * a.H + c, a.H - c);
            if (a.dsum) o.ds[i] = load<T, WHOLE>(a.dsum, row * a.H + c, a.H - c);
        }
    };
    auto times_far = [&](Operands& o) {
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if ((t + THREADS * i) * VEC < a.H)
#pragma unroll
                for (int k = 0; k < VEC; ++k) o.h[i].e[k] = narrow<T>(widen<T>(o.h[i].e[k]) * kFarRow);
    };
    constexpr bool AHEAD = NV == 1;               // (wider rows: the registers do not hold two rows' operands)
    int64_t row = (int64_t)blockIdx.x * ROWS + threadIdx.x / THREADS;
    Operands next;
    if (AHEAD) fetch(row, next);
    float far = 1.0f;
    for (int turn = 0; row < a.rows; turn ^= 1) {
        const int64_t at = row * a.H;
        float sums[2] = {0.0f, 0.0f};
        Operands now;
        if (!AHEAD) {
            fetch(row, now);
            if (kHasFarRows<T> && far != 1.0f) times_far(now);
        }
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            if ((t + THREADS * i) * VEC >= a.H) continue;
            if (AHEAD) now.h[i] = next.h[i], now.dy[i] = next.dy[i], now.ds[i] = next.ds[i];
#pragma unroll
            for (int k = 0; k < VEC; ++k) {
                const float hv = widen<T>(now.h[i].e[k]);
                sums[0] = __builtin_fmaf(hv, hv, sums[0]);
                sums[1] = __builtin_fmaf(widen<T>(now.dy[i].e[k]) * w[i][k], hv, sums[1]);
            }
        }
        if (AHEAD) fetch(row + step, next);
        row_sums<THREADS, 2>(sums, part[turn]);
        const float mean = sums[0] / (float)a.H + a.eps * far * far;
        if (kHasFarRows<T> && far == 1.0f && __builtin_amdgcn_readfirstlane(!(mean < INFINITY))) {      // another turn for this row (a wavefront's are one row's)
            far = kFarRow;
            if (AHEAD) fetch(row, next), times_far(next);
            continue;
        }
        const float r = 1.0f / sqrtf(mean), along = sums[1] * r / (float)a.H, r_dx = r * far;      // (n = h r: h has the factor)
        far = 1.0f;
        row += step;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (t + THREADS * i) * VEC;
            if (c >= a.H) continue;
            if (!AHEAD) {                         // as fetched, and not widened since: of several pieces the registers do not hold both
                asm volatile("" : "+v"(*reinterpret_cast<mx_u32x4*>(&now.h[i])));
                asm volatile("" : "+v"(*reinterpret_cast<mx_u32x4*>(&now.dy[i])));
            }
            P o;
#pragma unroll
            for (int k = 0; k < VEC; ++k) {
                const float n = widen<T>(now.h[i].e[k]) * r, d = widen<T>(now.dy[i].e[k]);
                dw[i][k] = __builtin_fmaf(d, n, dw[i][k]);
                float v = r_dx * (d * w[i][k] - n * along);
                if (a.dsum) v += widen<T>(now.ds[i].e[k]);
                o.e[k] = narrow<T>(v);
            }
            store<T, WHOLE>(a.dx, at + c, a.H - c, o);
        }
    }
    if constexpr (ROWS > 1) {                      // the rows of a workgroup share a row of partial sums
        __shared__ float shared[ROWS][THREADS * NV * VEC];
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (t + THREADS * i) * VEC;
#pragma unroll
            for (int k = 0; k < VEC; ++k) shared[threadIdx.x / THREADS][c + k] = dw[i][k];
        }
        __syncthreads();
        for (int c = threadIdx.x; c < a.H; c += kNormBlock<THREADS>) {
            float s = shared[0][c];
#pragma unroll
            for (int g = 1; g < ROWS; ++g) s += shared[g][c];
            a.part[(int64_t)blockIdx.x * a.H + c] = s;
        }
    } else {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (t + THREADS * i) * VEC;
#pragma unroll
            for (int k = 0; k < VEC; ++k)
                if (c + k < a.H) a.part[(int64_t)blockIdx.x * a.H + c + k] = dw[i][k];
        }
    }
}

// dw[c] = the sum of column c of `parts` rows: 32 columns a workgroup, 32 threads a column.
template <class T>
__global__ __launch_bounds__(1024) void norm_weight_grad_kernel(const float* __restrict__ part, int parts, int H, bool f32, void* __restrict__ dw) {
    __shared__ float s[32][33];
    const int x = threadIdx.x & 31, y = threadIdx.x >> 5, c = blockIdx.x * 32 + x;
    float sum = 0.0f;
    if (c < H) {
#pragma unroll 8
        for (int p = y; p < parts; p += 32) sum += part[(int64_t)p * H + c];
    }
    s[y][x] = sum;
    __syncthreads();
    if (y == 0 && c < H) {
        float v = s[0][x];
#pragma unroll
        for (int i = 1; i < 32; ++i) v += s[i][x];
        if (f32) static_cast<float*>(dw)[c] = v;
        else static_cast<typename T::raw*>(dw)[c] = narrow<T>(v);
    }
}

// ---- the experts' activation ----
//
// silu(g) u, gelu(u) or relu(u) of bf16 rows, to e4m3.  Hardware exp2 and reciprocal, 1 ulp each.  The exponential's argument is rounded once, so for
// negative g the result is off by |g| 2^-24 and the constant's half of that, 1.45 |g| 2^-24 in all: 2^-17 at g = -88, which three bits behind the
// first one see seldom.  What it saves is time: the vector ALU, not memory, bounded the kernel with an exponential of an argument in two parts, a
// Newton step and clamps: 16384 x 14336 SwiGLU 234 us.
// The quotient is made of quarters, 4 / (1 + e^-g): the hardware's reciprocal is 0 below fp32's normal numbers, and so is as wide as e^-g is one of
// fp32, g > -88.72.  Behind that e^-g / 4 or the sum is too large or infinite and the result 0 (exact: below 2.6e-37); NaN for -infinity.
__device__ __forceinline__ float silu_to8(float g) {
    return 0.25f * g * __builtin_amdgcn_rcpf(0.25f + __builtin_amdgcn_exp2f(__builtin_fmaf(g, -1.4426950408889634f, -2.0f)));
}

// COLD: more rows than the memory-side cache holds, read past it (16384 x 14336 SwiGLU 196 -> 175 to 186 us; 6000 x 1408, which the products in front have
// left there, 9.0 -> 9.8).  181 to 194 us are 6.1 to 6.5 TB/s.
template <int ACT, bool COLD>
__global__ __launch_bounds__(256) void act_rows128_kernel(const uint16_t* __restrict__ u, const uint16_t* __restrict__ g, const int32_t* __restrict__ count,
                                                          const int32_t* __restrict__ offset, int E, int64_t rows, int I, uint8_t* __restrict__ q,
                                                          float* __restrict__ scales) {
    const int64_t kept = count ? min((int64_t)offset[E - 1] + count[E - 1], rows) : rows;
    const int64_t chunk = (int64_t)blockIdx.x * 256 + threadIdx.x;      // 8 values; 16 lanes share a piece
    if (chunk >= kept * (I / 8)) return;
    auto fetch = [&](const uint16_t* p) {
        if constexpr (COLD) return __builtin_bit_cast(Piece<uint16_t>, __builtin_nontemporal_load(reinterpret_cast<const mx_u32x4*>(p + chunk * 8)));
        else return load<bf16_e, true>(p, chunk * 8, 8);
    };
    const auto uu = fetch(u);
    float v[8], amax = 0.0f;
    if constexpr (ACT == MOE_ACT_SWIGLU) {
        const auto gg = fetch(g);
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = silu_to8(widen<bf16_e>(gg.e[k])) * widen<bf16_e>(uu.e[k]);
    } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = act_apply(widen<bf16_e>(uu.e[k]), ACT);
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) amax = fmaxf(amax, fabsf(v[k]));
    const float s = rows8_scale(rows8_max<16>(amax)), inverse = 1.0f / s;
    if ((chunk & 15) == 0) scales[chunk >> 4] = s;
    *reinterpret_cast<uint2*>(q + chunk * 8) = uint2{rows8_codes(v[0], v[1], v[2], v[3], s, inverse), rows8_codes(v[4], v[5], v[6], v[7], s, inverse)};
}

// ---- launches ----

// f(threads, pieces a thread), as types: one piece a thread, and as few wavefronts as that takes, up to 16; then two or four.  8192 rows in bf16, us a call in a row, 256
// threads of several pieces / this: norm of 4096 values 49 / 44, of 7168 97 / 88, to e4m3 56 / 51, gradients without one of the sum 64 / 47; 64 rows of
// 7168 5.0 / 3.6.
// (BACKWARD: for wide rows eight wavefronts, which have twice the registers each that sixteen have.)
template <class T, bool BACKWARD, class F>
hipError_t with_norm_shape(int H, F f) {
    const int pieces = (H + kNormVec<T> - 1) / kNormVec<T>;
    auto go = [&](auto threads, auto nv) { return f(threads, nv); };
    typedef std::integral_constant<int, 1> One;
    if (pieces <= 64) return go(std::integral_constant<int, 64>{}, One{});
    if (pieces <= 128) return go(std::integral_constant<int, 128>{}, One{});
    if (pieces <= 256) return go(std::integral_constant<int, 256>{}, One{});
    if (pieces <= 512) return go(std::integral_constant<int, 512>{}, One{});
    if (pieces <= 1024) return go(std::integral_constant<int, 1024>{}, One{});
    constexpr int WIDE = BACKWARD ? 512 : 1024;
    if constexpr (sizeof(typename T::raw) == 4) {
        if (pieces > 2048) return go(std::integral_constant<int, 1024>{}, std::integral_constant<int, 4>{});
    }
    return go(std::integral_constant<int, WIDE>{}, std::integral_constant<int, 2048 / WIDE>{});
}

template <class T>
hipError_t launch_norm_type(const NormArgs& a, hipStream_t st) {
    auto off = [](const void* p) { return (uintptr_t)p % 16 != 0; };
    const bool whole = a.H % kNormVec<T> == 0 && !off(a.x) && !off(a.residual) && !off(a.weight) && !off(a.sum) && !off(a.out);
    return with_norm_shape<T, false>(a.H, [&](auto threads, auto nv) {
        constexpr int TH = decltype(threads)::value, NV = decltype(nv)::value, ROWS = kNormBlock<TH> / TH;
        const dim3 grid((unsigned)((a.rows + ROWS - 1) / ROWS));
        if (a.q) norm_rows_kernel<T, NV, TH, true, true><<<grid, kNormBlock<TH>, 0, st>>>(a);
        else if (whole) norm_rows_kernel<T, NV, TH, true, false><<<grid, kNormBlock<TH>, 0, st>>>(a);
        else norm_rows_kernel<T, NV, TH, false, false><<<grid, kNormBlock<TH>, 0, st>>>(a);
        return hipGetLastError();
    });
}

// Rows of partial sums of dw, one a workgroup: at most 1024 of up to 256 threads, fewer of more, so that 4096 wavefronts are on their way (16 a compute unit: 8192
// rows of 4096 without a gradient of the sum 47 us, 52 with twice as many, 62 with half; rows of 128 threads make 2048); no more than a quarter of the rows beyond one for each
// compute unit; and none that has no row (of rows that a wavefront holds, a workgroup takes four).  threads = 0: the most of any.
int64_t norm_parts(int64_t rows, int threads) {
    const int64_t filled = threads == kWave ? (rows + 3) / 4 : rows;
    return std::min<int64_t>(filled, std::min<int64_t>(4096 * 64 / std::max(threads, 256), std::max<int64_t>(256, rows / 4)));
}

template <class T>
hipError_t launch_norm_backward_type(const NormBackwardArgs& a, hipStream_t st) {
    auto off = [](const void* p) { return (uintptr_t)p % 16 != 0; };
    const bool whole = a.H % kNormVec<T> == 0 && !off(a.h) && !off(a.dy) && !off(a.dsum) && !off(a.weight) && !off(a.dx);
    int64_t parts = 0;
    if (a.rows > 0) {
        const hipError_t e = with_norm_shape<T, true>(a.H, [&](auto threads, auto nv) {
            constexpr int TH = decltype(threads)::value, NV = decltype(nv)::value;
            parts = norm_parts(a.rows, TH);
            if (whole) norm_backward_kernel<T, NV, TH, true><<<(unsigned)parts, kNormBlock<TH>, 0, st>>>(a);
            else norm_backward_kernel<T, NV, TH, false><<<(unsigned)parts, kNormBlock<TH>, 0, st>>>(a);
            return hipGetLastError();
        });
        if (e != hipSuccess) return e;
    }
    norm_weight_grad_kernel<T><<<(unsigned)((a.H + 31) / 32), 1024, 0, st>>>(a.part, (int)parts, a.H, a.weight_f32, a.dw);
    return hipGetLastError();
}

bool norm_dtype(int dtype) { return dtype == MOE_DTYPE_F32 || dtype == MOE_DTYPE_BF16 || dtype == MOE_DTYPE_FP16; }
int norm_refusal(int64_t rows, int32_t H, float eps, int32_t dtype, int32_t weight_dtype) {
    if (rows < 0 || H < 1 || !(eps >= 0.0f) || eps > 3.0e38f) return MOE_ERR_BAD_ARGUMENT;
    if (!norm_dtype(dtype) || (weight_dtype != dtype && weight_dtype != MOE_DTYPE_F32)) return MOE_ERR_UNSUPPORTED;
    return H > kNormMost || rows > kNormRows ? MOE_ERR_UNSUPPORTED : MOE_OK;
}
// Addresses of whole elements.
bool norm_element(const void* p, int dtype) { return (uintptr_t)p % (dtype == MOE_DTYPE_F32 ? 4 : 2) == 0; }

}  // namespace
}  // namespace moe355

using namespace moe355;

extern "C" int moe_rms_norm(const void* x, const void* residual, const void* weight, int64_t rows, int32_t H, float eps, int32_t dtype, int32_t weight_dtype,
                            void* sum, void* out, void* q, float* scales, void* stream) {
    const int rc = norm_refusal(rows, H, eps, dtype, weight_dtype);
    if (rc) return rc;
    if (rows == 0) return MOE_OK;                 // (tensors without elements have no address)
    if (!x || !weight || (residual != nullptr) != (sum != nullptr) || (q != nullptr) != (scales != nullptr) || (!out && !q)) return MOE_ERR_BAD_ARGUMENT;
    if (q && H % kRows8Piece) return MOE_ERR_BAD_ARGUMENT;
    for (const void* p : {x, residual, (const void*)sum, (const void*)out})
        if (!norm_element(p, dtype) || (q && (uintptr_t)p % 16)) return MOE_ERR_BAD_ARGUMENT;
    if (!norm_element(weight, weight_dtype) || (q && (uintptr_t)weight % 16) || (uintptr_t)q % 8 || (uintptr_t)scales % 4) return MOE_ERR_BAD_ARGUMENT;
    const NormArgs a{x, residual, weight, sum, out, (uint8_t*)q, scales, rows, H, eps, weight_dtype == MOE_DTYPE_F32};
    hipStream_t st = (hipStream_t)stream;
    const hipError_t e = dtype == MOE_DTYPE_F32 ? launch_norm_type<f32_e>(a, st) : dtype == MOE_DTYPE_BF16 ? launch_norm_type<bf16_e>(a, st) : launch_norm_type<f16_e>(a, st);
    return e == hipSuccess ? MOE_OK : MOE_ERR_HIP;
}

extern "C" int moe_rms_norm_scratch_bytes(int64_t rows, int32_t H, size_t* bytes) {
    if (rows < 0 || H < 1 || !bytes) return MOE_ERR_BAD_ARGUMENT;
    if (H > kNormMost || rows > kNormRows) return MOE_ERR_UNSUPPORTED;
    *bytes = (size_t)norm_parts(rows, 0) * H * sizeof(float);
    return MOE_OK;
}

extern "C" int moe_rms_norm_backward(const void* dout, const void* h, const void* weight, const void* dsum, int64_t rows, int32_t H, float eps, int32_t dtype,
                                     int32_t weight_dtype, void* dx, void* dweight, void* scratch, size_t scratch_bytes, void* stream) {
    const int rc = norm_refusal(rows, H, eps, dtype, weight_dtype);
    if (rc) return rc;
    if (!weight || !dweight || (rows > 0 && (!dout || !h || !dx))) return MOE_ERR_BAD_ARGUMENT;
    for (const void* p : {dout, h, dsum, (const void*)dx})
        if (!norm_element(p, dtype)) return MOE_ERR_BAD_ARGUMENT;
    if (!norm_element(weight, weight_dtype) || !norm_element(dweight, weight_dtype)) return MOE_ERR_BAD_ARGUMENT;
    if (rows > 0 && (!scratch || (uintptr_t)scratch % 4 || scratch_bytes < (size_t)norm_parts(rows, 0) * H * sizeof(float))) return MOE_ERR_WORKSPACE;
    const NormBackwardArgs a{dout, h, weight, dsum, dx, dweight, (float*)scratch, rows, H, eps, weight_dtype == MOE_DTYPE_F32};
    hipStream_t st = (hipStream_t)stream;
    const hipError_t e = dtype == MOE_DTYPE_F32 ? launch_norm_backward_type<f32_e>(a, st) : dtype == MOE_DTYPE_BF16 ? launch_norm_backward_type<bf16_e>(a, st) : launch_norm_backward_type<f16_e>(a, st);
    return e == hipSuccess ? MOE_OK : MOE_ERR_HIP;
}

extern "C" int moe_act_rows128(const void* u, const void* g, int64_t rows, int32_t I, int32_t act, const int32_t* expert_count, const int32_t* expert_offset,
                               int32_t E, void* q, float* scales, void* stream) {
    if (rows < 0 || I < kRows8Piece || I % kRows8Piece || (expert_count != nullptr) != (expert_offset != nullptr) || (expert_count && E < 1)) return MOE_ERR_BAD_ARGUMENT;
    if (act != MOE_ACT_SWIGLU && act != MOE_ACT_GELU && act != MOE_ACT_RELU) return MOE_ERR_BAD_ARGUMENT;
    if (rows == 0) return MOE_OK;
    if ((act == MOE_ACT_SWIGLU) != (g != nullptr)) return MOE_ERR_BAD_ARGUMENT;
    if ((uintptr_t)u % 16 || (uintptr_t)g % 16 || (uintptr_t)q % 8 || (uintptr_t)scales % 4) return MOE_ERR_BAD_ARGUMENT;
    if (!u || !q || !scales) return MOE_ERR_BAD_ARGUMENT;
    const int64_t blocks = (rows > INT32_MAX ? INT64_MAX : rows * (I / 8) + 255) / 256;
    if (blocks > (1 << 24) - 1) return MOE_ERR_UNSUPPORTED;      // (of 256 threads: a launch has less than 2^32)
    const dim3 grid((unsigned)blocks);
    hipStream_t st = (hipStream_t)stream;
    auto launch = [&](auto kernel) {
        kernel<<<grid, 256, 0, st>>>((const uint16_t*)u, (const uint16_t*)g, expert_count, expert_offset, E, rows, I, (uint8_t*)q, scales);
        return hipGetLastError() == hipSuccess ? MOE_OK : MOE_ERR_HIP;
    };
    const bool cold = rows * I * (g ? 4 : 2) > ((int64_t)256 << 20);
    auto of = [&](auto a) { return cold ? launch(act_rows128_kernel<decltype(a)::value, true>) : launch(act_rows128_kernel<decltype(a)::value, false>); };
    if (act == MOE_ACT_SWIGLU) return of(std::integral_constant<int, MOE_ACT_SWIGLU>{});
    if (act == MOE_ACT_GELU) return of(std::integral_constant<int, MOE_ACT_GELU>{});
    return of(std::integral_constant<int, MOE_ACT_RELU>{});
}
