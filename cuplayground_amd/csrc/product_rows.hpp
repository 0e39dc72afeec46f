// What the tiles of products over rows share, whatever their operands are held in: the meeting of a slab, the sums of wavefronts that split a
// contraction, and the way of results to memory.  PRODUCT has N and act, TASK the block's bias, out and rows.
#pragma once

#include "act_deriv.hpp"
#include "skinny.hpp"

namespace moe355 {
namespace {

typedef __attribute__((address_space(3))) void mx_lds_void;

__device__ __forceinline__ int64_t mx_uniform(int64_t v) {
    return (int64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)v) | (int64_t)__builtin_amdgcn_readfirstlane((int)(v >> 32)) << 32;
}

// The bias of CG groups of four neighbouring columns, COLS apart; of columns behind the last some bias.  All loads at once and without a
// question: one trip to memory -- and, where a kernel holds them as they come (fetch()) from its start on, one that nothing waits for.
template <int CG, int COLS>
struct MxBias {
    uint16_t raw[CG][4];
    bool any;
    template <class PRODUCT, class TASK>
    __device__ __forceinline__ void fetch(const PRODUCT& p, const TASK& t, int col0) {
        any = t.bias != nullptr;
        if (!any) return;
        if (p.N & 3) {
#pragma unroll
            for (int g = 0; g < CG; ++g) {
                const int col = col0 + COLS * g;
                if (col + 4 <= p.N) {
                    __builtin_memcpy(raw[g], t.bias + col, 8);
                } else {
#pragma unroll
                    for (int r = 0; r < 4; ++r) raw[g][r] = t.bias[min(col + r, p.N - 1)];
                }
            }
        } else {
#pragma unroll
            for (int g = 0; g < CG; ++g) __builtin_memcpy(raw[g], t.bias + min(col0 + COLS * g, p.N - 4), 8);
        }
    }
    __device__ __forceinline__ void widen(mx_f32x4 (&b)[CG]) const {
#pragma unroll
        for (int g = 0; g < CG; ++g) b[g] = mx_f32x4{0.f, 0.f, 0.f, 0.f};
        if (!any) return;
#pragma unroll
        for (int g = 0; g < CG; ++g)
#pragma unroll
            for (int r = 0; r < 4; ++r) b[g][r] = bf16_bits_to_f32(raw[g][r]);
    }
};
template <int CG, int COLS, class PRODUCT, class TASK>
__device__ __forceinline__ void mx_bias(const PRODUCT& p, const TASK& t, int col0, mx_f32x4 (&b)[CG]) {
    MxBias<CG, COLS> raw;
    raw.fetch(p, t, col0);
    raw.widen(b);
}
// Four neighbouring columns of a token row, as the matrix instructions leave them in a lane, in one store (memory takes 8 bytes at any address) but where
// the row ends.  whole: N is a multiple of 4.
template <int ACT, class TASK>
__device__ __forceinline__ void mx_store4(const TASK& t, int N, bool whole, int row, int col, const mx_f32x4& u) {
    float v[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) v[r] = ACT == MOE_ACT_GELU ? gelu16(u[r]) : ACT == MOE_ACT_RELU && u[r] < 0.0f ? 0.0f : u[r];      // a NaN stays a NaN
    const uint32_t lo = pack2_bf16(v[0], v[1]), hi = pack2_bf16(v[2], v[3]);
    uint16_t* o = t.out + (int64_t)row * N + col;
    if (whole || col + 4 <= N) {
        const uint2 both{lo, hi};
        __builtin_memcpy(o, &both, 8);
    } else {
        const uint32_t w[4] = {lo, lo >> 16, hi, hi >> 16};
#pragma unroll
        for (int r = 0; r < 4; ++r)
            if (col + r < N) o[r] = (uint16_t)w[r];
    }
}
// ... for NT x CG of them: rows row0 + ROWS i, columns col0 + COLS g.  One activation for all: a switch at every value costs more than the values.
template <int NT, int CG, int ROWS = 16, int COLS = 16, class PRODUCT, class TASK>
__device__ __forceinline__ void mx_store_tile(const PRODUCT& p, const TASK& t, int row0, int col0, const mx_f32x4 (&acc)[NT][CG], const MxBias<CG, COLS>* held = nullptr) {
    const int N = p.N;
    mx_f32x4 b[CG];
    if (held) held->widen(b);
    else mx_bias<CG, COLS>(p, t, col0, b);
    auto all = [&](auto act_c, auto whole_c) {
#pragma unroll
        for (int i = 0; i < NT; ++i) {
            if (row0 + ROWS * i >= t.rows) break;
#pragma unroll
            for (int g = 0; g < CG; ++g)
                if (col0 + COLS * g < N) mx_store4<decltype(act_c)::value>(t, N, decltype(whole_c)::value, row0 + ROWS * i, col0 + COLS * g, acc[i][g] + b[g]);
        }
    };
    typedef std::true_type Whole;
    if (N & 3) {
        if (p.act == MOE_ACT_GELU) all(std::integral_constant<int, MOE_ACT_GELU>{}, std::false_type{});
        else if (p.act == MOE_ACT_RELU) all(std::integral_constant<int, MOE_ACT_RELU>{}, std::false_type{});
        else all(std::integral_constant<int, MOE_ACT_NONE>{}, std::false_type{});
    } else if (p.act == MOE_ACT_GELU) all(std::integral_constant<int, MOE_ACT_GELU>{}, Whole{});
    else if (p.act == MOE_ACT_RELU) all(std::integral_constant<int, MOE_ACT_RELU>{}, Whole{});
    else all(std::integral_constant<int, MOE_ACT_NONE>{}, Whole{});
}

// mx_store_tile through LDS of the wavefront's own (mx_rows_lds bytes, where nothing else is read or written any more): as the instructions leave
// them, a store writes 16 or 32 bytes of 32 or 16 rows; this way it writes 64 to 256 bytes of a row, from any address.  Both rows in
// MXFP4, us, without / with: 8192 x 14336 x 4096 305 / 275, 1777 x 2752 x 1344 14.0 / 11.4; rows in bf16 672 / 657, 19.7 / 17.8.
template <int NT, int CG, int ROWS, int COLS>
__device__ __host__ constexpr int mx_rows_lds() { return ROWS * NT * (2 * COLS * CG + 16); }
template <int NT, int CG, int ROWS, int COLS, class PRODUCT, class TASK>
__device__ __forceinline__ void mx_store_rows(const PRODUCT& p, const TASK& t, unsigned char* own, int lane, int row, int col, int row0, int col0, const mx_f32x4 (&acc)[NT][CG], const MxBias<CG, COLS>* held = nullptr) {
    constexpr int PITCH = 2 * COLS * CG + 16, LANES = COLS * CG / 8;      // LANES of 16 bytes to a row
    mx_f32x4 b[CG];
    if (held) held->widen(b);
    else mx_bias<CG, COLS>(p, t, col0 + col, b);
    auto all = [&](auto act_c) {
        constexpr int ACT = decltype(act_c)::value;
#pragma unroll
        for (int g = 0; g < CG; ++g) {
#pragma unroll
            for (int i = 0; i < NT; ++i) {
                const mx_f32x4 u = acc[i][g] + b[g];
                float v[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) v[r] = ACT == MOE_ACT_GELU ? gelu16(u[r]) : ACT == MOE_ACT_RELU && u[r] < 0.0f ? 0.0f : u[r];      // a NaN stays a NaN
                *reinterpret_cast<uint2*>(own + (ROWS * i + row) * PITCH + 2 * (COLS * g + col)) = uint2{pack2_bf16(v[0], v[1]), pack2_bf16(v[2], v[3])};
            }
        }
    };
    if (p.act == MOE_ACT_GELU) all(std::integral_constant<int, MOE_ACT_GELU>{});
    else if (p.act == MOE_ACT_RELU) all(std::integral_constant<int, MOE_ACT_RELU>{});
    else all(std::integral_constant<int, MOE_ACT_NONE>{});
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    const int at = lane / LANES, piece = lane % LANES, c = col0 + 8 * piece;
    if (!(p.N & 7)) {                             // (a path of its own, without branches: 1777 x 2752 x 1408 15.2 / 14.4)
#pragma unroll
        for (int r = 0; r < ROWS * NT; r += 64 / LANES) {
            const mx_u32x4 v = *reinterpret_cast<const mx_u32x4*>(own + (r + at) * PITCH + 16 * piece);
            if (row0 + r + at < t.rows && c < p.N) *reinterpret_cast<mx_u32x4*>(t.out + (int64_t)(row0 + r + at) * p.N + c) = v;
        }
        return;
    }
#pragma unroll
    for (int r = 0; r < ROWS * NT; r += 64 / LANES) {
        const mx_u32x4 v = *reinterpret_cast<const mx_u32x4*>(own + (r + at) * PITCH + 16 * piece);
        if (row0 + r + at >= t.rows) continue;
        uint16_t* const o = t.out + (int64_t)(row0 + r + at) * p.N + c;
        if (c + 8 <= p.N) {
            __builtin_memcpy(o, &v, 16);
        } else {
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (c + k < p.N) o[k] = (uint16_t)(v[k / 2] >> (16 * (k & 1)));
        }
    }
}

// Every request of this wavefront for the slab has landed -- LATER ones that came behind may be on their way -- and its reads of the stage
// that is filled next are done, then so have everybody's.
template <int LATER = 0>
__device__ __forceinline__ void mx_meet() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(LATER) : "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}
// The sets' sums, in their order, through LDS: returns whether this wavefront holds them.
template <int KS, int SET, int NT, int CG>
__device__ __forceinline__ bool mx_join(mx_f32x4 (&acc)[NT][CG], int ks, int sw, unsigned char* smem, int lane) {
    if constexpr (KS > 1) {
        mx_meet();
        mx_f32x4* red = reinterpret_cast<mx_f32x4*>(smem) + sw * NT * CG * 64 + lane;
        if (ks > 0) {
#pragma unroll
            for (int i = 0; i < NT; ++i)
#pragma unroll
                for (int g = 0; g < CG; ++g) red[((ks - 1) * SET * NT * CG + i * CG + g) * 64] = acc[i][g];
        }
        __syncthreads();
        if (ks > 0) return false;
        for (int k = 0; k < KS - 1; ++k)
#pragma unroll
            for (int i = 0; i < NT; ++i)
#pragma unroll
                for (int g = 0; g < CG; ++g) acc[i][g] += red[(k * SET * NT * CG + i * CG + g) * 64];
    }
    return true;
}

}  // namespace
}  // namespace moe355
