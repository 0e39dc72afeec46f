// The root-mean-square norm of a residual stream, and what else makes rows in e4m3 for the products with block scales.
//
//   h = round(x + residual)         (without a residual: x; the stream keeps h in its own type, and what it keeps is what is normalised)
//   y = h r w,  r = 1 / sqrt(mean(h^2) + eps)
//   dx = r (dy w - n mean(dy w n)) + dsum,  n = h r;   dw = sum over rows of dy n
//
// Memory bounds all of it: every array passes once.  A row stays in the registers of the threads that fetched it, 16 bytes of every operand a
// thread and step, from the sum of its squares to its results.
#include "ffn_common.hpp"
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

// VEC neighbouring elements, fetched and stored as one.
template <class RAW, int VEC>
struct alignas(sizeof(RAW) * VEC) Piece { RAW e[VEC]; };
template <class T, int VEC>
__device__ __forceinline__ Piece<typename T::raw, VEC> load(const void* p, int64_t element) {
    return *reinterpret_cast<const Piece<typename T::raw, VEC>*>(static_cast<const typename T::raw*>(p) + element);
}
template <class T, int VEC>
__device__ __forceinline__ void store(void* p, int64_t element, const Piece<typename T::raw, VEC>& v) {
    *reinterpret_cast<Piece<typename T::raw, VEC>*>(static_cast<typename T::raw*>(p) + element) = v;
}
// Of the norm's weights, in the rows' type or in fp32.
template <class T, int VEC>
__device__ __forceinline__ void load_weights(float (&w)[VEC], const void* p, bool f32, int c) {
    if (f32) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) w[i] = static_cast<const float*>(p)[c + i];
    } else {
        const auto v = load<T, VEC>(p, c);
#pragma unroll
        for (int i = 0; i < VEC; ++i) w[i] = widen<T>(v.e[i]);
    }
}

// ---- sums over the threads of a row, in a fixed order, in all of them ----
__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
    for (int off = 1; off < kWave; off <<= 1) v += __shfl_xor(v, off, kWave);
    return v;
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

// THREADS threads to a row, NV pieces of VEC columns each; narrow rows share a workgroup of 256.
template <int THREADS> constexpr int kNormBlock = THREADS < 256 ? 256 : THREADS;

template <class T, int VEC, int NV, int THREADS, bool Q8>
__global__ __launch_bounds__(kNormBlock<THREADS>) void norm_rows_kernel(NormArgs a) {
    constexpr int ROWS = kNormBlock<THREADS> / THREADS;
    typedef Piece<typename T::raw, VEC> P;
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
        if (c < a.H) x[i] = load<T, VEC>(a.x, at + c);
    }
    if (a.residual) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (t + THREADS * i) * VEC;
            if (c < a.H) res[i] = load<T, VEC>(a.residual, at + c);
        }
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (t + THREADS * i) * VEC;
        if (c < a.H) load_weights<T, VEC>(w[i], a.weight, a.weight_f32, c);
    }
    float sum[1] = {0.0f};
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (t + THREADS * i) * VEC;
        if (c >= a.H) continue;
        if (a.residual) {
#pragma unroll
            for (int k = 0; k < VEC; ++k) x[i].e[k] = narrow<T>(widen<T>(x[i].e[k]) + widen<T>(res[i].e[k]));
            store<T, VEC>(a.sum, at + c, x[i]);
        }
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
            h[i][k] = widen<T>(x[i].e[k]);
            sum[0] = __builtin_fmaf(h[i][k], h[i][k], sum[0]);
        }
    }
    row_sums<THREADS, 1>(sum, part);
    const float r = 1.0f / sqrtf(sum[0] / (float)a.H + a.eps);
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
            store<T, VEC>(a.out, at + c, o);
        }
        if constexpr (Q8) {
            constexpr int LANES = kRows8Piece / VEC;
            float amax = 0.0f;
#pragma unroll
            for (int k = 0; k < VEC; ++k) amax = fmaxf(amax, fabsf(y[k]));
            const float s = rows8_scale(rows8_max<LANES>(amax)), inverse = 1.0f / s;
            if (t % LANES == 0) a.scales[row * (a.H / kRows8Piece) + c / kRows8Piece] = s;
            Piece<uint32_t, VEC / 4> q;
#pragma unroll
            for (int k = 0; k < VEC; k += 4) q.e[k / 4] = rows8_codes(y[k], y[k + 1], y[k + 2], y[k + 3], s, inverse);
            *reinterpret_cast<Piece<uint32_t, VEC / 4>*>(a.q + at + c) = q;
        }
    }
}

// The gradients.  A workgroup takes every gridDim.x-th row (ROWS of them at a time) and keeps its threads' columns of dw in registers; what it has of dw
// at the end is a row of `part`, and norm_weight_grad_kernel adds those up in their order: no atomics, the same bits every time.  The next
// row's operands are on their way while a row's sums are made.
template <class T, int VEC, int NV, int THREADS>
__global__ __launch_bounds__(kNormBlock<THREADS>) void norm_backward_kernel(NormBackwardArgs a) {
    constexpr int ROWS = kNormBlock<THREADS> / THREADS;
    typedef Piece<typename T::raw, VEC> P;
    __shared__ float part[2][2 * (THREADS / kWave)];
    const int t = threadIdx.x % THREADS;
    const int64_t step = (int64_t)gridDim.x * ROWS;
    float w[NV][VEC], dw[NV][VEC];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (t + THREADS * i) * VEC;
#pragma unroll
        for (int k = 0; k < VEC; ++k) w[i][k] = dw[i][k] = 0.0f;
        if (c < a.H) load_weights<T, VEC>(w[i], a.weight, a.weight_f32, c);
    }
    P h[NV], dy[NV], ds[NV];
    auto fetch = [&](int64_t row) {
        if (row >= a.rows) return;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (t + THREADS * i) * VEC;
            if (c >= a.H) continue;
            h[i] = load<T, VEC>(a.h, row * a.H + c);
            dy[i] = load<T, VEC>(a.dy, row * a.H + c);
            if (a.dsum) ds[i] = load<T, VEC>(a.dsum, row * a.H + c);
        }
    };
    int64_t row = (int64_t)blockIdx.x * ROWS + threadIdx.x / THREADS;
    fetch(row);
    for (int turn = 0; row < a.rows; row += step, turn ^= 1) {
        const int64_t at = row * a.H;
        float hv[NV][VEC], dn[NV][VEC], sums[2] = {0.0f, 0.0f};
        P ds_now[NV];
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            if ((t + THREADS * i) * VEC >= a.H) continue;
            ds_now[i] = ds[i];
#pragma unroll
            for (int k = 0; k < VEC; ++k) {
                hv[i][k] = widen<T>(h[i].e[k]);
                dn[i][k] = widen<T>(dy[i].e[k]);
                sums[0] = __builtin_fmaf(hv[i][k], hv[i][k], sums[0]);
                sums[1] = __builtin_fmaf(dn[i][k] * w[i][k], hv[i][k], sums[1]);
            }
        }
        fetch(row + step);
        row_sums<THREADS, 2>(sums, part[turn]);
        const float r = 1.0f / sqrtf(sums[0] / (float)a.H + a.eps), along = sums[1] * r / (float)a.H;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (t + THREADS * i) * VEC;
            if (c >= a.H) continue;
            P o;
#pragma unroll
            for (int k = 0; k < VEC; ++k) {
                const float n = hv[i][k] * r;
                dw[i][k] = __builtin_fmaf(dn[i][k], n, dw[i][k]);
                float d = r * (dn[i][k] * w[i][k] - n * along);
                if (a.dsum) d += widen<T>(ds_now[i].e[k]);
                o.e[k] = narrow<T>(d);
            }
            store<T, VEC>(a.dx, at + c, o);
        }
    }
    if constexpr (ROWS > 1) {                      // the rows of a workgroup share a row of partial sums
        extern __shared__ float shared[];          // [ROWS][H]
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (t + THREADS * i) * VEC;
            if (c >= a.H) continue;
#pragma unroll
            for (int k = 0; k < VEC; ++k) shared[(threadIdx.x / THREADS) * a.H + c + k] = dw[i][k];
        }
        __syncthreads();
        for (int c = threadIdx.x; c < a.H; c += kNormBlock<THREADS>) {
            float s = shared[c];
#pragma unroll
            for (int g = 1; g < ROWS; ++g) s += shared[g * a.H + c];
            a.part[(int64_t)blockIdx.x * a.H + c] = s;
        }
    } else {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (t + THREADS * i) * VEC;
            if (c >= a.H) continue;
#pragma unroll
            for (int k = 0; k < VEC; ++k) a.part[(int64_t)blockIdx.x * a.H + c + k] = dw[i][k];
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
// silu(g) u, gelu(u) or relu(u) of bf16 rows, to e4m3.  The exponential of an argument in two parts and a reciprocal with one Newton step: what
// is rounded to four bits next is then as good as with the library's expf and a division, and its code as seldom the neighbour of the exact one's.
__device__ __forceinline__ float silu_to8(float g) {
    constexpr float kLog2e = 1.44269504088896340736f, kLog2eRest = 1.92596299e-8f;      // log2(e) = the sum
    const float hi = fminf(fmaxf(g * -kLog2e, -200.0f), 126.0f);
    const float lo = fmaxf(__builtin_fmaf(g, -kLog2e, -hi) - g * kLog2eRest, -1.0f);      // (2^-16 at most, but where hi was cut)
    const float e = __builtin_amdgcn_exp2f(hi);
    const float d = 1.0f + __builtin_fmaf(e, lo * 0.693147180559945309417f, e);
    const float r = __builtin_amdgcn_rcpf(d);
    return g * (hi < 126.0f ? __builtin_fmaf(__builtin_fmaf(-d, r, 1.0f), r, r) : 0.0f);      // further out the result is below 2^-119: 0 (of -infinity: NaN)
}

template <int ACT>
__global__ __launch_bounds__(256) void act_rows128_kernel(const uint16_t* __restrict__ u, const uint16_t* __restrict__ g, const int32_t* __restrict__ count,
                                                          const int32_t* __restrict__ offset, int E, int64_t rows, int I, uint8_t* __restrict__ q,
                                                          float* __restrict__ scales) {
    const int64_t kept = count ? min((int64_t)offset[E - 1] + count[E - 1], rows) : rows;
    const int64_t chunk = (int64_t)blockIdx.x * 256 + threadIdx.x;      // 8 values; 16 lanes share a piece
    if (chunk >= kept * (I / 8)) return;
    const auto uu = load<bf16_e, 8>(u, chunk * 8);
    float v[8], amax = 0.0f;
    if constexpr (ACT == MOE_ACT_SWIGLU) {
        const auto gg = load<bf16_e, 8>(g, chunk * 8);
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

template <class T> constexpr int kNormVec = 16 / (int)sizeof(typename T::raw);

// f(threads, pieces a thread, columns a piece), as types: the fewest threads that hold a row in four pieces each, or, where the rows are few and
// nothing but latency counts, in one.  Columns one by one where rows do not begin on 16 bytes.
template <class T, bool BACKWARD, class F>
hipError_t with_norm_shape(int H, int64_t rows, bool whole, F f) {
    constexpr int V = kNormVec<T>;
    auto go = [&](auto threads, auto nv, auto vec) { return f(threads, nv, vec); };
#define NORM_SHAPE(TH, NV, VEC) go(std::integral_constant<int, TH>{}, std::integral_constant<int, NV>{}, std::integral_constant<int, VEC>{})
    if (!whole) {
        if (!BACKWARD && H <= 1024) return NORM_SHAPE(64, 16, 1);
        if (H <= 4096) return NORM_SHAPE(256, 16, 1);
        return NORM_SHAPE(1024, 16, 1);
    }
    const int pieces = (H + V - 1) / V;
    if (pieces <= 64) return NORM_SHAPE(64, 1, V);
    if (!BACKWARD && rows >= 4096 && pieces <= 128) return NORM_SHAPE(64, 2, V);
    if (pieces <= 256) return NORM_SHAPE(256, 1, V);
    if (pieces <= 512) return NORM_SHAPE(256, 2, V);
    if (pieces <= 1024) return NORM_SHAPE(256, 4, V);
    if (pieces <= 2048) return NORM_SHAPE(1024, 2, V);
    return NORM_SHAPE(1024, 4, V);
#undef NORM_SHAPE
}

template <class T, bool Q8>
hipError_t launch_norm_of(const NormArgs& a, bool whole, hipStream_t st) {
    return with_norm_shape<T, false>(a.H, a.rows, whole, [&](auto threads, auto nv, auto vec) {
        constexpr int TH = decltype(threads)::value, NV = decltype(nv)::value, V = decltype(vec)::value, ROWS = kNormBlock<TH> / TH;
        if constexpr (Q8 && V == 1) {
            return hipErrorInvalidValue;          // (rows of e4m3 are whole pieces of 128)
        } else {
            norm_rows_kernel<T, V, NV, TH, Q8><<<(unsigned)((a.rows + ROWS - 1) / ROWS), kNormBlock<TH>, 0, st>>>(a);
            return hipGetLastError();
        }
    });
}
template <class T>
hipError_t launch_norm_type(const NormArgs& a, hipStream_t st) {
    constexpr int V = kNormVec<T>;
    auto off = [](const void* p) { return (uintptr_t)p % 16 != 0; };
    const bool whole = a.H % V == 0 && !off(a.x) && !off(a.residual) && !off(a.weight) && !off(a.sum) && !off(a.out);
    return a.q ? launch_norm_of<T, true>(a, whole, st) : launch_norm_of<T, false>(a, whole, st);
}

// Rows of partial sums of dw: as many workgroups as keep four on a compute unit busy, and not more than a quarter of the rows beyond one each.
int64_t norm_parts(int64_t rows) { return std::min<int64_t>(rows, std::min<int64_t>(1024, std::max<int64_t>(256, rows / 4))); }

template <class T>
hipError_t launch_norm_backward_type(const NormBackwardArgs& a, hipStream_t st) {
    constexpr int V = kNormVec<T>;
    auto off = [](const void* p) { return (uintptr_t)p % 16 != 0; };
    const bool whole = a.H % V == 0 && !off(a.h) && !off(a.dy) && !off(a.dsum) && !off(a.weight) && !off(a.dx);
    const int64_t parts = norm_parts(a.rows);
    if (a.rows > 0) {
        const hipError_t e = with_norm_shape<T, true>(a.H, a.rows, whole, [&](auto threads, auto nv, auto vec) {
            constexpr int TH = decltype(threads)::value, NV = decltype(nv)::value, VE = decltype(vec)::value, ROWS = kNormBlock<TH> / TH;
            norm_backward_kernel<T, VE, NV, TH><<<(unsigned)parts, kNormBlock<TH>, ROWS > 1 ? ROWS * a.H * 4 : 0, st>>>(a);
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
    *bytes = (size_t)norm_parts(rows) * H * sizeof(float);
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
    if (rows > 0 && (!scratch || (uintptr_t)scratch % 4 || scratch_bytes < (size_t)norm_parts(rows) * H * sizeof(float))) return MOE_ERR_WORKSPACE;
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
    if (act == MOE_ACT_SWIGLU) return launch(act_rows128_kernel<MOE_ACT_SWIGLU>);
    if (act == MOE_ACT_GELU) return launch(act_rows128_kernel<MOE_ACT_GELU>);
    return launch(act_rows128_kernel<MOE_ACT_RELU>);
}
