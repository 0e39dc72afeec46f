// Products of a few token rows with weights that are read once: what a wavefront of a weight streamer does, for weights in 16 bits and in
// MXFP4 (mxfp4.hpp).
//
// A wavefront owns G groups of 16 weight rows (output columns) over its share of the contraction dimension: the weights are the "A" operand
// of the 16 x 16 matrix instructions, up to 16 token rows the "B" operand.  Weights come whole 128-byte lines of eight rows at a time
// (stream_lines.hpp); a lane then has, of each 64 bytes of row (lane & 15), piece (lane >> 4).  Which values of k an instruction multiplies
// does not matter as long as both operands agree: with 16-bit weights a piece is the eight values an instruction takes of a lane.  With
// MXFP4 a piece is 32 codes, a whole block with one scale: four instructions of bf16, eight of its codes each -- widened exactly, scale
// included, two an instruction -- or, against rows in MXFP4, the whole operand of one scaled instruction over 128 values.
#pragma once

#include "ffn_common.hpp"
#include "mxfp4.hpp"
#include "stream_lines.hpp"

namespace moe355 {
namespace {

typedef _Float16 sk_f16x8 __attribute__((ext_vector_type(8)));

// Weights in 16 bits (ET: bf16_s, f16_s).  A chunk is what a wavefront has in flight twice: 256 bytes of each of 16 rows.
template <class ET>
struct Weights16 {
    static constexpr bool MX = false;
    static constexpr bool F16 = std::is_same<ET, f16_s>::value;
    static constexpr int K = 128;            // values of k of a chunk
    static constexpr int LINES = 2;          // 128-byte lines of a row
    static constexpr int FRAGS = 4;          // 16-byte pieces of a token row that a lane multiplies
    static __host__ __device__ __forceinline__ int64_t row_bytes(int64_t k) { return 2 * k; }
};
struct WeightsMx {
    static constexpr bool MX = true;
    static constexpr bool F16 = false;
    static constexpr int K = 256;
    static constexpr int LINES = 1;
    static constexpr int FRAGS = 8;
    static __host__ __device__ __forceinline__ int64_t row_bytes(int64_t k) { return k >> 1; }
};

// Where 16 rows of a matrix lie for this lane.
struct SkinnyRows {
    const char* first;       // of the line instruction's lower eight rows
    const char* second;      // ... and of the upper eight
    const uint8_t* scale;    // of row (lane & 15)
};
// Rows n0 .. n0 + 15 of [N][K]; rows behind the last one read it again.
template <class W>
__device__ __forceinline__ SkinnyRows skinny_rows(const void* w, const uint8_t* s, int n0, int N, int K, int lane) {
    const int64_t rb = W::row_bytes(K);
    const char* base = static_cast<const char*>(w) + ((lane >> 4) + ((lane & 8) >> 1)) * 16;
    SkinnyRows r;
    r.first = base + min(n0 + (lane & 7), N - 1) * rb;
    r.second = base + min(n0 + 8 + (lane & 7), N - 1) * rb + ((lane & 8) ? -64 : 64);
    r.scale = W::MX ? s + (int64_t)min(n0 + (lane & 15), N - 1) * (K >> 5) : nullptr;
    return r;
}

template <class W, int G>
struct SkinnyChunk {
    mx_u32x4 v[G][2 * W::LINES];
    uint32_t s[W::MX ? G : 1][2];            // MXFP4: the scales of the row's eight blocks
};

template <class W, int G, bool COLD>
__device__ __forceinline__ void skinny_load(SkinnyChunk<W, G>& d, const SkinnyRows (&r)[G], int c) {
#pragma unroll
    for (int g = 0; g < G; ++g) {
#pragma unroll
        for (int l = 0; l < W::LINES; ++l) {
            const int64_t at = ((int64_t)c * W::LINES + l) * 128;
            d.v[g][2 * l] = load_piece<COLD>(r[g].first + at);
            d.v[g][2 * l + 1] = load_piece<COLD>(r[g].second + at);
        }
        if constexpr (W::MX) __builtin_memcpy(d.s[g], r[g].scale + 8 * (int64_t)c, 8);
    }
}

// A row's last chunk, cut off: pieces behind its end are read from the chunk's first (which is inside) and become zeros in skinny_settle_tail.
// left: bytes of the row that the chunk has.
template <class W, int G, bool COLD>
__device__ __forceinline__ void skinny_load_tail(SkinnyChunk<W, G>& d, const SkinnyRows (&r)[G], int c, int left, int lane) {
    const int piece = (lane >> 4) + ((lane & 8) >> 1);
#pragma unroll
    for (int g = 0; g < G; ++g) {
#pragma unroll
        for (int l = 0; l < W::LINES; ++l) {
            const int64_t at = ((int64_t)c * W::LINES + l) * 128;
            const int o1 = 128 * l + 16 * piece, o2 = 128 * l + 16 * (piece ^ 4);
            d.v[g][2 * l] = load_piece<COLD>(r[g].first + at - (o1 < left ? 0 : o1));
            d.v[g][2 * l + 1] = load_piece<COLD>(r[g].second + at - (o2 < left ? 0 : o2));
        }
        if constexpr (W::MX) {
            const int blocks = left >> 4;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                d.s[g][h] = 0;
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (4 * h + i < blocks) d.s[g][h] |= (uint32_t)r[g].scale[8 * (int64_t)c + 4 * h + i] << (8 * i);
            }
        }
    }
}
// Lines -> pieces: v[g][2 l] and v[g][2 l + 1] become this lane's piece of the lower and the upper 64 bytes of line l.
template <class W, int G>
__device__ __forceinline__ void skinny_settle(SkinnyChunk<W, G>& d) {
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
        for (int l = 0; l < W::LINES; ++l) line_pieces(d.v[g][2 * l], d.v[g][2 * l + 1], d.v[g][2 * l], d.v[g][2 * l + 1]);
}
template <class W, int G>
__device__ __forceinline__ void skinny_zero_tail(SkinnyChunk<W, G>& d, int left, int lane) {
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
        for (int p = 0; p < 2 * W::LINES; ++p)
            if (64 * p + 16 * (lane >> 4) >= left) d.v[g][p] = mx_u32x4{0u, 0u, 0u, 0u};
}

// The scale of piece p (0: the lower 64 bytes, 1: the upper) of this lane, in the low byte.
__device__ __forceinline__ uint32_t skinny_scale(const uint32_t (&s)[2], int p, int lane) { return s[p] >> (8 * (lane >> 4)); }

// Token rows of 16 bits: x points at the lane's row; the pieces of chunk c.  k of piece p, 16-bit weights: 32 p + 8 q; MXFP4: 128 (p / 4) +
// 32 q + 8 (p % 4), q = lane >> 4.
template <class W>
__device__ __forceinline__ int skinny_k(int p, int lane) {
    return W::MX ? 128 * (p >> 2) + 32 * (lane >> 4) + 8 * (p & 3) : 32 * p + 8 * (lane >> 4);
}
template <class W>
__device__ __forceinline__ void skinny_tokens(mx_u32x4 (&x)[W::FRAGS], const uint16_t* row, int c, int lane) {
#pragma unroll
    for (int p = 0; p < W::FRAGS; ++p) x[p] = *reinterpret_cast<const mx_u32x4*>(row + (int64_t)c * W::K + skinny_k<W>(p, lane));
}
// ... zeros behind the row's end (an infinity there would make a NaN of the weights' zeros).  left: values of the row that the chunk has.
template <class W>
__device__ __forceinline__ void skinny_tokens_tail(mx_u32x4 (&x)[W::FRAGS], const uint16_t* row, int c, int left, int lane) {
#pragma unroll
    for (int p = 0; p < W::FRAGS; ++p) {
        const int k = skinny_k<W>(p, lane);
        x[p] = mx_u32x4{0u, 0u, 0u, 0u};
        if (k < left) x[p] = *reinterpret_cast<const mx_u32x4*>(row + (int64_t)c * W::K + k);
    }
}

template <class W>
__device__ __forceinline__ mx_f32x4 skinny_mfma(mx_u32x4 a, mx_u32x4 b, mx_f32x4 c) {
    if constexpr (W::F16) return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(sk_f16x8, a), __builtin_bit_cast(sk_f16x8, b), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(mx_bf16x8, a), __builtin_bit_cast(mx_bf16x8, b), c, 0, 0, 0);
}
// acc[g] += the chunk's weights times 16 token rows of 16 bits; d has been settled.
template <class W, int G>
__device__ __forceinline__ void skinny_multiply(mx_f32x4 (&acc)[G], const SkinnyChunk<W, G>& d, const mx_u32x4 (&x)[W::FRAGS], int lane) {
#pragma unroll
    for (int p = 0; p < 2 * W::LINES; ++p) {
#pragma unroll
        for (int g = 0; g < G; ++g) {
            if constexpr (W::MX) {
                const float s = mx_scale(skinny_scale(d.s[g], p, lane) & 255u);
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    acc[g] = skinny_mfma<W>(__builtin_bit_cast(mx_u32x4, mx_widen8(d.v[g][p][j], s)), x[4 * p + j], acc[g]);
            } else {
                acc[g] = skinny_mfma<W>(d.v[g][p], x[p], acc[g]);
            }
        }
    }
}

// Both operands in MXFP4: the scaled instruction over 128 values; a scale is the low byte of its register.
__device__ __forceinline__ mx_f32x4 mx_mfma(mx_u32x4 a, uint32_t sa, mx_u32x4 b, uint32_t sb, mx_f32x4 c) {
    // (the upper half, which 4-bit operands do not have, is left open)
    const mx_i32x8 av = __builtin_bit_cast(mx_i32x8, __builtin_shufflevector(a, a, 0, 1, 2, 3, -1, -1, -1, -1));
    const mx_i32x8 bv = __builtin_bit_cast(mx_i32x8, __builtin_shufflevector(b, b, 0, 1, 2, 3, -1, -1, -1, -1));
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(av, bv, c, 4 /* e2m1 */, 4, 0, (int)sa, 0, (int)sb);
}

// Sums of KS wavefronts that shared a contraction, through LDS, in the order of the wavefronts: returns whether this one holds them.
// red: [KS - 1][G][64] of 16 bytes for each set of columns.  Every wavefront of the workgroup calls it.
template <int G>
__device__ __forceinline__ bool skinny_join(mx_f32x4 (&acc)[G], int ks, int KS, mx_f32x4* red, int lane) {
    if (KS == 1) return true;
    if (ks > 0) {
#pragma unroll
        for (int g = 0; g < G; ++g) red[((ks - 1) * G + g) * 64 + lane] = acc[g];
    }
    __syncthreads();
    if (ks > 0) return false;
    for (int k = 0; k < KS - 1; ++k)
#pragma unroll
        for (int g = 0; g < G; ++g) acc[g] += red[(k * G + g) * 64 + lane];
    return true;
}

}  // namespace
}  // namespace moe355
