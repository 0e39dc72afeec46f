// Products of a few token rows with weights that are read once: what a wavefront of a weight streamer does, for weights in 16 bits and in
// MXFP4 (mxfp4.hpp).
//
// A wavefront owns G groups of 16 weight rows (output columns) over its share of the contraction dimension: the weights are the "A" operand
// of the 16 x 16 matrix instructions, up to 16 token rows the "B" operand.  Weights come whole 128-byte lines of eight rows at a time
// (stream_lines.hpp); a lane then has, of each 64 bytes of row (lane & 15), piece (lane >> 4).  Which values of k an instruction multiplies
// does not matter as long as both operands agree: with 16-bit weights a piece is the eight values an instruction takes of a lane.  With
// MXFP4 a piece is 32 codes, a whole block with one scale: four instructions of bf16, eight of its codes each -- widened exactly, scale
// included, two an instruction -- or, against rows in MXFP4, the whole operand of one scaled instruction over 128 values.
//
// What bounds it is memory, and then the address unit, which takes as long over a request for 64 bytes as over one for a kilobyte.  So
// nothing but weights is fetched in the shape in which it is used: a chunk's token rows go, as they lie, into LDS of the wavefront's own
// (for one row an instruction a chunk instead of eight), and scales come for four chunks at a time, 32 bytes of 16 rows an instruction, and
// find their lanes by a permutation.  One row times 65536 x 4096 in MXFP4, us, everything fetched as it is used / scales left out / rows left out
// / both: 40.2 / 36.6 / 31.9 / 25.6; this way 29.6 (4.8 TB/s), and 84 for 65536 x 14336 (5.9 TB/s).  A launch in which wavefronts have less
// than four chunks each pays as for four.  All operands are read through buffers that end where they end: what lies behind is zeros, without a
// branch.
#pragma once

#include "ffn_common.hpp"
#include "mxfp4.hpp"
#include "stream_lines.hpp"

namespace moe355 {
namespace {

typedef _Float16 sk_f16x8 __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) void sk_lds_void;

constexpr uint32_t kBehind = 0xD0000000u;      // an offset behind the end of every buffer here, also with a tile's rows added to it (offsets
                                               // are whole in the vector register: the range check is against what a scalar offset leaves of the
                                               // buffer, and that may be less than nothing)
__device__ __forceinline__ __amdgpu_buffer_rsrc_t mx_buffer(const void* p, uint32_t bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, (int)bytes, 0x00020000);
}

// Weights in 16 bits (ET: bf16_s, f16_s).  A chunk: 256 bytes of each of 16 rows, 256 bytes of a token row.
template <class ET>
struct Weights16 {
    static constexpr bool MX = false;
    static constexpr bool F16 = std::is_same<ET, f16_s>::value;
    static constexpr int K = 128;            // values of k of a chunk
    static constexpr int LINES = 2;          // 128-byte lines of a weight row
    static constexpr int ROWB = 256;         // bytes of a token row
    static __host__ __device__ __forceinline__ int64_t row_bytes(int64_t k) { return 2 * k; }
    static __device__ __forceinline__ uint32_t token_bytes(uint32_t k) { return 2 * k; }
};
// Weights in MXFP4; token rows in bf16, or (ROWS4) in MXFP4 too.
template <bool ROWS4_>
struct WeightsMx {
    static constexpr bool MX = true;
    static constexpr bool ROWS4 = ROWS4_;
    static constexpr bool F16 = false;
    static constexpr int K = 256;
    static constexpr int LINES = 1;
    static constexpr int ROWB = ROWS4 ? 128 : 512;
    static __host__ __device__ __forceinline__ int64_t row_bytes(int64_t k) { return k >> 1; }
    static __device__ __forceinline__ uint32_t token_bytes(uint32_t k) { return ROWS4 ? k >> 1 : 2 * k; }
};
// Dynamic LDS of a launch; on every launch, for it holds for the current device.
template <class K>
hipError_t allow_lds(K kernel, int bytes) {
    return hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
}
constexpr int kUnit = 4;                       // chunks that share a fetch of scales
constexpr uint32_t kNoChunk = 1u << 22;        // a chunk behind every row's end
// LDS of a wavefront: two chunks of token rows, whole instructions of them.
template <class W>
__host__ __device__ constexpr int skinny_lds(int rows) {
    return 2 * ((rows * W::ROWB + 1023) / 1024) * 1024;
}

// Where the pieces (16 bytes) of a row's segments (64 bytes) lie in LDS.  A 16-byte read is served to lanes 0-3, 12-15 and 20-27 in a cycle, to
// 4-11, 16-19 and 28-31 in the next, and so on.  Lane (row, q) reads piece j of segment q: with segment q in place q ^ sk_turn(row), and
// piece j in place j ^ row of it, those of a cycle meet every bank once.  And the four lanes that fill a place read one segment: of pieces from
// four segments the address unit makes four requests.
__device__ __forceinline__ int sk_turn(int row) { return (4 - (row >> 2)) & 3; }

// One wavefront's stream.  aim_weights() and aim_tokens() say what the next unit is made of; scales(), fetch() and multiply() go through its
// chunks.
template <class W, int G, bool COLD>
struct Skinny {
    static constexpr bool rows4() { return W::MX && W::ROWB == 128; }
    static constexpr int PER = 1024 / W::ROWB;             // token rows an instruction brings
    static constexpr int MOST = 16 / PER;                  // ... and instructions for 16 rows
    static constexpr int LATER = 2 * W::LINES * G;         // requests for a chunk's weights, its last ones

    mx_u32x4 v[2][G][2 * W::LINES];
    uint64_t s_raw[G], sx_raw;
    uint32_t s_early[G], sx_early;                         // bytes that the fetch lies in front of what was wanted
    uint32_t s[G][2], sx[2];                               // this chunk's scales (MXFP4): blocks 0-3 and 4-7 of row (lane & 15)
    uint64_t s_held[G], sx_held;

    __amdgpu_buffer_rsrc_t w_buf[G], x_buf;
    const uint8_t* s_at[G];
    const uint8_t* sx_at;
    uint32_t s_last;                                       // the last eight bytes of the matrix's scales
    int64_t sx_base, sx_end;                               // the token rows' scales: where row 0 begins, the array's last eight bytes
    uint32_t w1, w2, w_add, s_row[G], sx_row, row, x_row;
    uint32_t x_of[(MOST + 3) / 4];                         // the lane's token rows' places in x_buf, a byte each
    int rows, chunk0, chunk_end;                           // token rows, chunks [chunk0, chunk_end) of the unit
    int lane;
    unsigned char* lds;
    int half;                                              // bytes of one of its two parts

    __device__ __forceinline__ void init(unsigned char* own, int rows_most, int K) {
        lane = threadIdx.x & 63;
        lds = own;
        half = skinny_lds<W>(rows_most) / 2;
        row = (uint32_t)W::row_bytes(K);
        x_row = W::token_bytes(K);
    }
    // Weight rows n0 .. n0 + 15 of [N][K], and of group g those 16 g further on (or the same ones of another matrix: w_buf, s_at).
    __device__ __forceinline__ void aim_weights(int n0, int N, int step) {
        w1 = (uint32_t)(n0 + (lane & 7)) * row;
        w2 = w1 + 8 * row;
        w_add = (uint32_t)step * row;
        if constexpr (W::MX) {
            const uint32_t sr = row >> 4;
            s_last = (uint32_t)N * sr - 8;
#pragma unroll
            for (int g = 0; g < G; ++g) s_row[g] = (uint32_t)min(n0 + step * g + (lane >> 2), N - 1) * sr;
        }
    }
    // Token rows: row r is row of(r) of x_buf.
    template <class OF>
    __device__ __forceinline__ void aim_tokens(int n, OF of) {
        rows = n;
#pragma unroll
        for (int p = 0; p < MOST; ++p) {
            if (p % 4 == 0) x_of[p / 4] = 0;
            if (PER * p < n) x_of[p / 4] |= (uint32_t)of(min(PER * p + lane / (64 / PER), n - 1)) << (8 * (p & 3));
        }
    }

    // Eight bytes of scales: inside the array, which has eight.
    __device__ __forceinline__ void eight(uint64_t& raw, uint32_t& early, const uint8_t* at, uint32_t want, uint32_t last) {
        const uint32_t o = min(want, last);
        early = want - o;
        __builtin_memcpy(&raw, at + o, 8);
    }
    // Lane 4 r + j: of row r the scales of chunk j of the unit.
    __device__ __forceinline__ void scales() {
        if constexpr (W::MX) {
            const uint32_t sr = row >> 4, c = min(8u * (uint32_t)(chunk0 + (lane & 3)), sr);      // behind the row's end: some bytes that are not used
#pragma unroll
            for (int g = 0; g < G; ++g) eight(s_raw[g], s_early[g], s_at[g], s_row[g] + c, s_last);
            if constexpr (rows4()) {
                const int64_t want = sx_base + sx_row + c, o = min(want, sx_end);
                sx_early = (uint32_t)(want - o);
                __builtin_memcpy(&sx_raw, sx_at + o, 8);
            }
        }
    }
    __device__ __forceinline__ void settle_scales() {
        if constexpr (W::MX) {
#pragma unroll
            for (int g = 0; g < G; ++g) s_held[g] = s_raw[g] >> (4 * s_early[g]) >> (4 * s_early[g]);
            if constexpr (rows4()) sx_held = sx_raw >> (4 * sx_early) >> (4 * sx_early);
        }
    }

    // Chunk j of the unit into part b.
    __device__ __forceinline__ void fetch(int b, int j) {
        const uint32_t c = chunk0 + j < chunk_end ? (uint32_t)(chunk0 + j) : kNoChunk;
        {
            const int slots = W::ROWB / 16, slot = lane % slots;
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");             // what lay there has been read
#pragma unroll
            for (int p = 0; p < MOST; ++p) {
                if (p > 0 && PER * p >= rows) break;                       // (the first one without a question: the waits below count on it)
                const int r = PER * p + lane / slots;
                uint32_t piece;                                            // which 16 bytes of the row slot `slot` holds (see fragment)
                if constexpr (!W::MX) piece = slot ^ (r & 15);
                else if constexpr (W::ROWB == 512) piece = (slot & 16) + 4 * (((slot >> 2) & 3) ^ sk_turn(r)) + ((slot ^ r) & 3);
                else piece = slot ^ ((r >> 1) & 7);
                const uint32_t at = c * W::ROWB + 16 * piece;
                __builtin_amdgcn_raw_ptr_buffer_load_lds(x_buf, (sk_lds_void*)(lds + b * half + p * 1024), 16, (int)(at < x_row ? (x_of[p / 4] >> (8 * (p & 3)) & 255u) * x_row + at : kBehind), 0, 0, 0);
            }
        }
        const uint32_t piece = (lane >> 4) + ((lane & 8) >> 1);
#pragma unroll
        for (int l = 0; l < W::LINES; ++l) {
            const uint32_t at = (c * W::LINES + l) * 128, o1 = at + 16 * piece, o2 = at + 16 * (piece ^ 4);
            const uint32_t v1 = o1 < row ? w1 + o1 : kBehind, v2 = o2 < row ? w2 + o2 : kBehind;
#pragma unroll
            for (int g = 0; g < G; ++g) {
                v[b][g][2 * l] = __builtin_bit_cast(mx_u32x4, __builtin_amdgcn_raw_buffer_load_b128(w_buf[g], (int)(v1 + g * w_add), 0, COLD ? 2 : 0));      // 2: not kept
                v[b][g][2 * l + 1] = __builtin_bit_cast(mx_u32x4, __builtin_amdgcn_raw_buffer_load_b128(w_buf[g], (int)(v2 + g * w_add), 0, COLD ? 2 : 0));
            }
        }
    }

    // Piece p of the lane's token row in part b.  Slots are permuted by the row (sk_turn).  Lanes behind the last row read row 0.
    __device__ __forceinline__ mx_u32x4 fragment(int b, int p, int rows_of_unit) const {
        const int q = lane >> 4, r = (lane & 15) < rows_of_unit ? lane & 15 : 0;
        int slot;
        if constexpr (!W::MX) slot = (4 * p + q) ^ r;
        else if constexpr (W::ROWB == 512) slot = 16 * (p >> 2) + 4 * (q ^ sk_turn(r)) + ((p ^ r) & 3);
        else slot = (4 * p + q) ^ ((r >> 1) & 7);
        return *reinterpret_cast<const mx_u32x4*>(lds + b * half + r * W::ROWB + 16 * slot);
    }
    static __device__ __forceinline__ mx_f32x4 mfma(mx_u32x4 a, mx_u32x4 x, mx_f32x4 c) {
        if constexpr (W::F16) return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(sk_f16x8, a), __builtin_bit_cast(sk_f16x8, x), c, 0, 0, 0);
        else return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(mx_bf16x8, a), __builtin_bit_cast(mx_bf16x8, x), c, 0, 0, 0);
    }
    // acc[g] += chunk j of the unit that began with chunk `first` and has so many rows, in part b.
    __device__ __forceinline__ void multiply(mx_f32x4 (&acc)[G], int b, int j, int first, int rows_of_unit) {
        // the other part's requests came later than all of this one's, those for its weights and one for a token row at least
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"(LATER + 1) : "memory");
        __builtin_amdgcn_sched_barrier(0);                                 // (nothing that waits for this part moves in front of the requests)
        if constexpr (W::MX) {
            const int from = 16 * (lane & 15) + 4 * j, q = lane >> 4;      // bytes: lane 4 (lane & 15) + j
            const uint32_t block = 8 * (uint32_t)(first + j) + q, blocks = row >> 4;
            auto turn = [&](uint32_t (&d)[2], uint64_t held) {             // this lane's bytes; behind the row's end: 0
                const uint32_t lo = (uint32_t)__builtin_amdgcn_ds_bpermute(from, (int)(uint32_t)held), hi = (uint32_t)__builtin_amdgcn_ds_bpermute(from, (int)(uint32_t)(held >> 32));
                d[0] = block < blocks ? lo >> (8 * q) & 255u : 0u;
                d[1] = block + 4 < blocks ? hi >> (8 * q) & 255u : 0u;
            };
#pragma unroll
            for (int g = 0; g < G; ++g) turn(s[g], s_held[g]);
            if constexpr (rows4()) turn(sx, sx_held);
        }
        mx_u32x4 x[W::MX && W::ROWB == 512 ? 8 : 4];
        constexpr int P = W::MX ? (W::ROWB == 512 ? 8 : 2) : 4;
#pragma unroll
        for (int p = 0; p < P; ++p) x[p] = fragment(b, p, rows_of_unit);
#pragma unroll
        for (int g = 0; g < G; ++g)
#pragma unroll
            for (int l = 0; l < W::LINES; ++l) line_pieces(v[b][g][2 * l], v[b][g][2 * l + 1], v[b][g][2 * l], v[b][g][2 * l + 1]);
#pragma unroll
        for (int p = 0; p < 2 * W::LINES; ++p) {
            if constexpr (!W::MX) {
#pragma unroll
                for (int g = 0; g < G; ++g) acc[g] = mfma(v[b][g][p], x[p], acc[g]);
            } else if constexpr (W::ROWB == 512) {
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int g = 0; g < G; ++g) {
                        const uint32_t codes = v[b][g][p][i];
                        acc[g] = mfma(__builtin_bit_cast(mx_u32x4, mx_widen8(codes, mx_scale(s[g][p]))), x[4 * p + i], acc[g]);
                    }
            } else {
#pragma unroll
                for (int g = 0; g < G; ++g) {
                    // (the upper half, which 4-bit operands do not have, is left open)
                    const mx_i32x8 av = __builtin_bit_cast(mx_i32x8, __builtin_shufflevector(v[b][g][p], v[b][g][p], 0, 1, 2, 3, -1, -1, -1, -1));
                    const mx_i32x8 bv = __builtin_bit_cast(mx_i32x8, __builtin_shufflevector(x[p], x[p], 0, 1, 2, 3, -1, -1, -1, -1));
                    acc[g] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(av, bv, acc[g], 4 /* e2m1 */, 4, 0, (int)s[g][p], 0, (int)sx[p]);
                }
            }
        }
    }
    // Units 0 .. n - 1: next(u) aims at unit u (u = n: nothing, chunk_end = 0), done(u) follows the last product of unit u.
    template <class NEXT, class DONE>
    __device__ __forceinline__ void run(int n, mx_f32x4 (&acc)[G], NEXT next, DONE done) {
        if (n == 0) return;
        next(0);
        scales();
        fetch(0, 0);
        fetch(1, 1);
        for (int u = 0; u < n; ++u) {
            const int first = chunk0, n_rows = rows;
            settle_scales();
            multiply(acc, 0, 0, first, n_rows);
            fetch(0, 2);
            multiply(acc, 1, 1, first, n_rows);
            fetch(1, 3);
            next(u + 1);
            scales();
            multiply(acc, 0, 2, first, n_rows);
            fetch(0, 0);
            multiply(acc, 1, 3, first, n_rows);
            fetch(1, 1);
            done(u);
        }
    }
};

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
