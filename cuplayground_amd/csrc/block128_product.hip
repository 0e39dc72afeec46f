// Products of rows in e4m3 (rows8.hpp: a scale for 128 values of a row) with weights in e4m3 that have a scale for each block of 128 x 128:
//
//   out[m, n] = act(sum over blocks b of K:  s_a[m, b] s_w[n / 128, b]  (sum over k in b of a[m, k] w[n, k])  + bias[n])
//
// One matrix, or a matrix per expert over packed rows, which may be fetched from the tokens' rows by their indices.  The inner sums are one 16 x 16 x
// 128 matrix instruction each, exact products in fp32; the vector ALU folds them into the accumulators with the product of the two scales, which is
// one number a lane where the token rows are the instruction's columns.  Sums in fp32, rounded once on store -- but for what the instruction itself does:
// it adds eight neighbouring products at a time, cut off below 2^-13 of the power of two that the largest begins with (measured).  Rounded
// to bf16, results lie 2.7e-4 (2-norm) from exact sums that are rounded to it, where that rounding itself is 1.7e-3.
//
// Two kinds of kernel: a weight streamer for up to 16 rows a block, and tiles.  block_form() takes the one whose fitted cost is least.
//
// Few rows: memory bounds it, weights once -- 1 x 4096 x 14336 11.4 us and 48 x 14336 x 4096 12.4, where a bare read of the 58.7 MB takes 9.4.  Many: the matrix
// instructions under the card's power -- 8192 x 14336 x 4096 427 us and x 14336 1367 (2.25 and 2.46 PFLOP/s; zeros 325 and 1157).  The instructions alone
// on random data reach 4.29 PFLOP/s, with the scales' multiplications 3.70.
#include "grouped_task.hpp"
#include "product_rows.hpp"

namespace moe355 {
namespace {

struct RowsTask {
    const uint8_t* a;         // the block's first row (rows fetched by index: row 0 of all)
    const float* a_scales;
    const uint8_t* w;         // the expert's matrix
    const float* s;
    const uint16_t* bias;     // of the expert, or null
    const int32_t* token;     // of the block's rows, or null
    uint16_t* out;            // at the block's first row
    int rows, n0;
    int kind;                 // a block of a tile's rows; with 256: kLeftRows at most; kPieceRows at most and half a tile's columns
};
enum { kBlockTask, kLeftTask, kPieceTask };
constexpr int kLeftRows = 128, kPieceRows = 64;

// The tiles of one matrix: blocks of BM rows; with 256 what is left of at most kLeftRows stands behind them, and the last round may be in smaller tiles, as of
// experts (grouped_task.hpp).
struct RowsDense {
    int blocks, lefts;
    int64_t share, halved, left_share;          // of an XCD
    bool pieces;
};
__host__ __device__ __forceinline__ RowsDense rows_dense(const RowsProduct& p, int BM, int BN) {
    const int ncol = (p.N + BN - 1) / BN;
    RowsDense d;
    d.blocks = (int)((p.M + BM - 1 - (BM == 256 ? kLeftRows : 0)) / BM);
    const int64_t left = p.M - (int64_t)d.blocks * BM;
    const int high = left <= 0 ? 0 : left <= kPieceRows ? 1 : 2;
    d.share = ((int64_t)d.blocks * ncol + 7) / 8;
    d.pieces = d.share % kXcdUnits == 0 && 2 * (int64_t)high * ncol <= kGroupedUnits;
    d.lefts = high == 0 ? 0 : d.pieces ? 2 * high * ncol : ncol;
    d.left_share = ((int64_t)d.lefts + 7) / 8;
    d.halved = BM == 256 ? halved_blocks(d.share, d.left_share) : 0;
    return d;
}
// Which block of BM rows and which BN columns a workgroup takes.
template <int BM>
__device__ __forceinline__ bool rows_task(const RowsProduct& p, int BN, RowsTask& t) {
    const int ncol = (p.N + BN - 1) / BN;
    constexpr bool LEFT = BM == 256;
    int expert = 0, ctile, rows, kind = kBlockTask;
    int64_t row0;
    if (p.count) {
        GroupedTask g;
        if (!grouped_task<BM, LEFT ? kPieceRows : 0>(p.count, p.offset, p.E, ncol, (int)blockIdx.x, g)) return false;
        expert = g.expert, ctile = g.ctile, row0 = g.row0, rows = g.rows;
        if (LEFT) kind = g.piece ? kPieceTask : rows <= kLeftRows ? kLeftTask : kBlockTask;
        if (row0 < 0 || row0 + rows > p.M) return false;          // tables that are not this layer's: nothing behind the buffers is touched
    } else {
        // an eighth of the tiles in a row for each XCD, kRowChunk row blocks at a time, then the same of the remainder, as for the experts
        const RowsDense d = rows_dense(p, BM, BN);
        int64_t id = blockIdx.x >> 3;
        const int xcd = blockIdx.x & 7;
        if (id < d.share + d.halved) {
            const int64_t behind = id - (d.share - d.halved);
            if (LEFT && behind >= 0) id -= (behind + 1) >> 1;
            id += xcd * d.share;
            if (id >= (int64_t)d.blocks * ncol) return false;
            int rb = (int)(id / ((int64_t)kRowChunk * ncol)) * kRowChunk;
            const int width = min(kRowChunk, d.blocks - rb), local = (int)(id - (int64_t)rb * ncol);
            ctile = local / width;
            rb += local - ctile * width;
            row0 = (int64_t)rb * BM;
            rows = (int)min((int64_t)BM, p.M - row0);
            if (LEFT && behind >= 0) {
                const int first = (int)(behind & 1) * kLeftRows;
                row0 += first, rows = min(rows - first, kLeftRows), kind = kLeftTask;
            }
        } else {
            id = id - d.share - d.halved + xcd * d.left_share;
            const int cols = d.pieces ? 2 * ncol : ncol;
            if (id >= d.lefts || id >= (xcd + 1) * d.left_share) return false;
            const int rb = (int)id / cols;
            ctile = (int)id - rb * cols;
            row0 = (int64_t)d.blocks * BM + rb * kPieceRows;
            rows = (int)(p.M - row0);
            if (d.pieces) rows = min(rows, kPieceRows);
            kind = d.pieces ? kPieceTask : kLeftTask;
        }
    }
    // the same in every lane, and said so
    row0 = mx_uniform(row0), expert = __builtin_amdgcn_readfirstlane(expert), ctile = __builtin_amdgcn_readfirstlane(ctile), rows = __builtin_amdgcn_readfirstlane(rows);
    kind = __builtin_amdgcn_readfirstlane(kind);
    const int KB = p.K >> 7;
    const int64_t first = p.token ? 0 : row0;
    t.a = p.a + first * p.K;
    t.a_scales = p.a_scales + first * KB;
    t.w = p.w + (int64_t)expert * p.N * p.K;
    t.s = p.s + (int64_t)expert * ((p.N + 127) >> 7) * KB;
    t.bias = p.bias ? p.bias + (int64_t)expert * p.N : nullptr;
    t.token = p.token ? p.token + row0 : nullptr;
    t.out = p.out + row0 * p.N;
    t.rows = rows;
    t.n0 = ctile * (kind == kPieceTask ? BN / 2 : BN);
    t.kind = kind;
    return t.n0 < p.N;        // (half tiles: the last one may have no column)
}
// Row r of the block as the buffers below count rows; kNoRow where there is none (an index that is no token's is none).
constexpr uint32_t kNoRow = 0xFFFFFFFFu;
__device__ __forceinline__ uint32_t rows_source(const RowsProduct& p, const RowsTask& t, int r) {
    if (r >= t.rows) return kNoRow;
    if (!t.token) return (uint32_t)r;
    const uint32_t i = (uint32_t)t.token[r];
    return i < (uint32_t)p.tokens ? i : kNoRow;
}
__device__ __forceinline__ mx_f32x4 rows_mfma(const mx_i32x8& w, const mx_i32x8& x) {
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w, x, mx_f32x4{0.f, 0.f, 0.f, 0.f}, 0 /* e4m3 */, 0, 0, 0, 0, 0);
}
__device__ __forceinline__ mx_i32x8 rows_operand(const mx_u32x4& lower, const mx_u32x4& upper) {
    return __builtin_bit_cast(mx_i32x8, __builtin_shufflevector(lower, upper, 0, 1, 2, 3, 4, 5, 6, 7));
}

// ---- up to 16 rows a block: a weight streamer ----
//
// A wavefront owns G groups of 16 columns over its share of the contraction; weights come whole 128-byte lines of eight rows at a time
// (stream_lines.hpp), which is a block of K, and stay in registers, kDepth blocks on their way.  Token rows come the same way (of up to eight rows,
// without MORE, one instruction), and the token rows' scales four blocks of 16 rows an instruction: the address unit takes as long over a
// request in pieces as over whole lines.
constexpr int kRowsWaves = 8, kDepth = 4;      // (four: the blocks of K that an instruction brings the scales of)

template <int G, bool MORE, bool COLD>
__global__ __launch_bounds__(64 * kRowsWaves) void rows_stream_kernel(RowsProduct p, int KS) {
    __shared__ mx_f32x4 red[(kRowsWaves - 1) * G * 64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int ks = wave % KS, set = wave / KS;
    RowsTask t;
    if (!rows_task<16>(p, 16 * G * (kRowsWaves / KS), t)) return;
    const int n0 = t.n0 + 16 * G * set, KB = p.K >> 7;
    const uint32_t K = (uint32_t)p.K;
    const int64_t rows_all = p.token ? p.tokens : t.rows;
    const __amdgpu_buffer_rsrc_t x_buf = mx_buffer(t.a, (uint32_t)(rows_all * K)), w_buf = mx_buffer(t.w, (uint32_t)p.N * K),
                                 s_buf = mx_buffer(t.a_scales, (uint32_t)(rows_all * KB * 4));
    const int q = lane >> 4;
    const uint32_t piece = q + ((lane & 8) >> 1);
    const uint32_t w1 = (uint32_t)(n0 + (lane & 7)) * K + 16 * piece, w2 = (uint32_t)(n0 + 8 + (lane & 7)) * K + 16 * (piece ^ 4);
    auto row_at = [&](int r, uint32_t bytes, uint32_t more) {
        const uint32_t src = rows_source(p, t, r);
        return src == kNoRow ? kBehind : src * bytes + more;
    };
    const uint32_t x1 = row_at(lane & 7, K, 16 * piece), x2 = row_at(8 + (lane & 7), K, 16 * (piece ^ 4));
    const uint32_t s_at = row_at(lane & 15, (uint32_t)KB * 4, 4 * q);
    const float* const ws = t.s + (int64_t)min(n0 >> 7, (p.N - 1) >> 7) * KB;

    const int share = (KB + KS - 1) / KS, begin = min(ks * share, KB), end = min(begin + share, KB);
    mx_u32x4 w[kDepth][G][2], x[kDepth][2];
    float raw;                                     // lane 16 q + r: the scale of row r in block q of a turn
    // What lies behind the share's end: zeros.
    auto fetch = [&](int slot, int c) {
        const bool in = c < end;
        const uint32_t at = 128u * (uint32_t)c;
        x[slot][0] = __builtin_bit_cast(mx_u32x4, __builtin_amdgcn_raw_buffer_load_b128(x_buf, (int)(in ? x1 + at : kBehind), 0, 0));
        if (MORE) x[slot][1] = __builtin_bit_cast(mx_u32x4, __builtin_amdgcn_raw_buffer_load_b128(x_buf, (int)(in ? x2 + at : kBehind), 0, 0));
#pragma unroll
        for (int g = 0; g < G; ++g) {
            w[slot][g][0] = __builtin_bit_cast(mx_u32x4, __builtin_amdgcn_raw_buffer_load_b128(w_buf, (int)(in ? w1 + at + g * 16 * K : kBehind), 0, COLD ? 2 : 0));      // 2: not kept
            w[slot][g][1] = __builtin_bit_cast(mx_u32x4, __builtin_amdgcn_raw_buffer_load_b128(w_buf, (int)(in ? w2 + at + g * 16 * K : kBehind), 0, COLD ? 2 : 0));
        }
    };
    auto fetch_scales = [&](int c) { raw = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(s_buf, (int)(c + q < end ? s_at + 4u * (uint32_t)c : kBehind), 0, 0)); };
    MxBias<G, 16> bias;
    bias.fetch(p, t, n0 + 4 * q);
    mx_f32x4 acc[1][G] = {};
    if (begin < end) {
        // The weights' scales: one a block of K, 64 of them in the lanes of a register.
        float held = begin + lane < end ? ws[begin + lane] : 0.0f;
        fetch_scales(begin);
#pragma unroll
        for (int d = 0; d < kDepth; ++d) fetch(d, begin + d);
        for (int c = begin; c < end; c += kDepth) {
            if (c > begin && ((c - begin) & 63) == 0) {
                held = c + lane < end ? ws[c + lane] : 0.0f;
                asm volatile("" : "+v"(held));    // (the wait for it is here, not in every turn)
            }
            const int sa = __builtin_bit_cast(int, raw);
            fetch_scales(c + kDepth);
#pragma unroll
            for (int d = 0; d < kDepth; ++d) {
                const float s = __builtin_bit_cast(float, __builtin_amdgcn_ds_bpermute(4 * ((lane & 15) + 16 * d), sa)) *
                                __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, held), (c - begin + d) & 63));
                mx_u32x4 lower, upper;
                if (MORE) {
                    line_pieces(x[d][0], x[d][1], lower, upper);
                } else {
                    lower = x[d][0];
#pragma unroll
                    for (int i = 0; i < 4; ++i) upper[i] = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x[d][0][i], 0x128, 0xF, 0xF, false);      // row_ror:8
                }
                const mx_i32x8 xv = rows_operand(lower, upper);
#pragma unroll
                for (int g = 0; g < G; ++g) {
                    line_pieces(w[d][g][0], w[d][g][1], lower, upper);
                    const mx_f32x4 part = rows_mfma(rows_operand(lower, upper), xv);
#pragma unroll
                    for (int r = 0; r < 4; ++r) acc[0][g][r] = __builtin_fmaf(part[r], s, acc[0][g][r]);
                }
                fetch(d, c + d + kDepth);
            }
        }
    }
    if (!skinny_join<G>(acc[0], ks, KS, red + set * (KS - 1) * G * 64, lane)) return;
    mx_store_tile<1, G>(p, t, lane & 15, n0 + 4 * q, acc, &bias);
}

// ---- more rows: tiles ----
//
// RH x CW wavefronts of 16 NT rows x 16 CG columns each, KS sets of them that share the contraction.  A slab is a block of K: 128 bytes of every row
// of either operand, straight into LDS AHEAD slabs ahead, and 4 bytes of every token row, its scale.  Everything is read through buffers that end
// where the operands do: rows behind the block's last one, columns behind the matrix's and what lies behind K are zeros without a branch.
template <int RH_, int NT_, int CW_, int CG_, int KS_, int AHEAD_>
struct RowsTile {
    static constexpr int RH = RH_, NT = NT_, CW = CW_, CG = CG_, KS = KS_, AHEAD = AHEAD_;
    static constexpr int STAGES = AHEAD + 1;
    static constexpr int BM = 16 * NT * RH, BN = 16 * CG * CW;
    static constexpr int SET = RH * CW;
    static constexpr int THREADS = 64 * SET * KS;
    static constexpr int LOADS_A = BM / 8 / SET, LOADS_W = BN / 8 / SET;      // an instruction of a wavefront brings 8 rows
    static constexpr int SCALERS = (BM + 63) / 64;                            // wavefronts of a set that bring scales
    static constexpr int STAGE = (BM + BN) * 128 + SCALERS * 256;
    static constexpr int SUMS = (KS - 1) * SET * NT * CG * 1024;
    static constexpr int OUT = KS == 1 ? SET * mx_rows_lds<NT, CG, 16, 16>() : 0;
    static constexpr int LDS = std::max(std::max(STAGES * KS * STAGE, SUMS), OUT);
    static constexpr int BLOCKS = std::min(160 * 1024 / LDS, NT * CG >= 32 ? 8 / (SET * KS) : 16 / (SET * KS));      // workgroups of a compute unit
    static constexpr int WAVES_PER_SIMD = std::max(1, BLOCKS * THREADS / 256);
    static_assert(BM % (8 * SET) == 0 && BN % (8 * SET) == 0 && SCALERS <= SET, "every wavefront of a set brings as many rows");
    static_assert(128 % (16 * CG) == 0, "a wavefront's columns have one scale");
    static_assert(LDS <= 160 * 1024, "LDS of a compute unit");
};

template <class T, bool COLD>
__device__ __forceinline__ void rows_tile(const RowsProduct& p, const RowsTask& t, unsigned char* smem) {
    constexpr int NT = T::NT, CG = T::CG, KS = T::KS, SET = T::SET, BM = T::BM, BN = T::BN, AHEAD = T::AHEAD;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int ks = wave / SET, sw = wave % SET;
    const int wm = sw / T::CW, wn = sw % T::CW;
    const int idx = lane & 15, q = lane >> 4;
    const int N = p.N, KB = p.K >> 7;
    const uint32_t K = (uint32_t)p.K;

    // Rows into LDS: an instruction writes 1 KB of LDS in the order of its lanes.  Piece c (16 bytes) of a row lies in slot c ^ (row / 2): the reads
    // below meet no bank twice in a cycle.
    const int lrow = lane >> 3;
    const uint32_t chunk = (lane & 7) ^ (((8 * sw + lrow) >> 1) & 7);         // (the rows of a wavefront's further instructions are a multiple of 16 on)
    static_assert(SET % 2 == 0, "rows of a wavefront's instructions lie a multiple of 16 apart");
    const int64_t rows_all = p.token ? p.tokens : t.rows;
    const __amdgpu_buffer_rsrc_t a_buf = mx_buffer(t.a, (uint32_t)(rows_all * K)), w_buf = mx_buffer(t.w, (uint32_t)N * K),
                                 s_buf = mx_buffer(t.a_scales, (uint32_t)(rows_all * KB * 4));
    uint32_t a_off[T::LOADS_A], s_off = kBehind;
    const uint32_t w_off = (uint32_t)(t.n0 + 8 * sw + lrow) * K + 16 * chunk;
    const bool scaler = sw < T::SCALERS;
    unsigned char* const stages = smem + ks * T::STAGES * T::STAGE;
    const int slabs = (KB + KS - 1) / KS, begin = ks * slabs, end = min(begin + slabs, KB);      // of the set; all run as many
    constexpr int LOADS = T::LOADS_A + T::LOADS_W;
    auto issue = [&](int s, unsigned char* st, int first, int last) {         // requests [first, last) of slab number s of this set
        const int k = begin + s;
        const bool in = k < end;
        const uint32_t at = 128u * (uint32_t)k;
#pragma unroll
        for (int l = first; l < last && l < LOADS; ++l) {
            const int i = l - T::LOADS_W;
            if (l < T::LOADS_W)
                __builtin_amdgcn_raw_ptr_buffer_load_lds(w_buf, (mx_lds_void*)(st + BM * 128 + (l * SET + sw) * 1024), 16, (int)(in ? w_off + at + l * SET * 8 * K : kBehind), 0, 0, COLD ? 2 : 0);
            else
                __builtin_amdgcn_raw_ptr_buffer_load_lds(a_buf, (mx_lds_void*)(st + (i * SET + sw) * 1024), 16, (int)(in ? a_off[i] + at : kBehind), 0, 0, 0);
        }
        if (first <= T::LOADS_W && T::LOADS_W < last && scaler)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(s_buf, (mx_lds_void*)(st + (BM + BN) * 128 + sw * 256), 4, (int)(in ? s_off + 4u * (uint32_t)k : kBehind), 0, 0, 0);
    };
    // The weights' scales: one a slab, 64 slabs of them in the lanes of a register.  (As scalar loads they would share their counter with the reads of
    // LDS, and return out of order: every wait for a fragment would be one for all.)
    const int c0 = t.n0 + 16 * CG * wn;
    const float* const ws = t.s + (int64_t)min(c0 >> 7, (N - 1) >> 7) * KB;
    float held = begin + lane < end ? ws[begin + lane] : 0.0f;      // (the first ones: in front of all requests)
    MxBias<CG, 16> bias;
    bias.fetch(p, t, c0 + 4 * q);
    auto weight_scale = [&](int s) { return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, held), s & 63)); };
    auto hold = [&](int s) {
        held = begin + s + lane < end ? ws[begin + s + lane] : 0.0f;
        asm volatile("" : "+v"(held));            // (the wait for it is here, not in every slab)
    };

    mx_f32x4 acc[NT][CG];
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int g = 0; g < CG; ++g) acc[i][g] = mx_f32x4{0.f, 0.f, 0.f, 0.f};

    // A slab, a group of 16 columns at a time: the next group's fragments are read, and the last one's products folded, under this one's.
    auto slab = [&](const unsigned char* st, float s_w, auto request) {       // request(g): in front of group g
        const unsigned char* xb = st + (wm * 16 * NT + idx) * 128;
        const unsigned char* wb = st + (BM + wn * 16 * CG + idx) * 128;
        const float* sb = reinterpret_cast<const float*>(st + (BM + BN) * 128) + wm * 16 * NT + idx;
        const int at0 = (q ^ (idx >> 1)) << 4, at1 = ((4 + q) ^ (idx >> 1)) << 4;
        mx_i32x8 x[NT], w[2];
        float sc[NT];
        mx_f32x4 part[2][NT];
        auto read = [&](const unsigned char* b, int i) {
            return rows_operand(*reinterpret_cast<const mx_u32x4*>(b + i * 16 * 128 + at0), *reinterpret_cast<const mx_u32x4*>(b + i * 16 * 128 + at1));
        };
        w[0] = read(wb, 0);
#pragma unroll
        for (int i = 0; i < NT; ++i) x[i] = read(xb, i);
#pragma unroll
        for (int i = 0; i < NT; ++i) sc[i] = sb[16 * i] * s_w;
#pragma unroll
        for (int g = 0; g <= CG; ++g) {
            if (g < CG) request(g);
            if (g + 1 < CG) w[(g + 1) & 1] = read(wb, g + 1);
#pragma unroll
            for (int i = 0; i < NT; ++i) {
                if (g < CG) part[g & 1][i] = rows_mfma(w[g & 1], x[i]);
                if (g > 0) {
#pragma unroll
                    for (int r = 0; r < 4; ++r) acc[i][g - 1][r] = __builtin_fmaf(part[(g - 1) & 1][i][r], sc[i], acc[i][g - 1][r]);
                }
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    auto after = [&](unsigned char* st) { return st + T::STAGE == stages + T::STAGES * T::STAGE ? stages : st + T::STAGE; };
    auto meet = [&] {                             // (a slab's requests are LOADS, and one more of the wavefronts that bring scales)
        if (AHEAD > 1 && scaler) mx_meet<(AHEAD - 1) * (LOADS + 1)>();
        else mx_meet<(AHEAD - 1) * LOADS>();
    };
    unsigned char* now = stages;                  // the stage of the slab that is next; the one in front of it is filled next
    unsigned char* fill = stages + AHEAD * T::STAGE;
    // (columns first: of rows that are fetched by index the indices have to come before)
    issue(0, stages, 0, T::LOADS_W);
#pragma unroll
    for (int i = 0; i < T::LOADS_A; ++i) {
        const uint32_t src = rows_source(p, t, 8 * (i * SET + sw) + lrow);
        a_off[i] = src == kNoRow ? kBehind : src * K + 16 * chunk;
    }
    if (scaler) {
        const uint32_t src = rows_source(p, t, 64 * sw + lane);
        s_off = src == kNoRow ? kBehind : src * (uint32_t)KB * 4;
    }
    issue(0, stages, T::LOADS_W, LOADS);
#pragma unroll
    for (int s = 1; s < AHEAD; ++s) issue(s, stages + s * T::STAGE, 0, LOADS);
    constexpr int PER = (LOADS + CG - 1) / CG;
    asm volatile("" : "+v"(held));
    if (t.rows > wm * 16 * NT) {
        for (int s = 0; s < slabs; ++s) {
            if ((s & 63) == 0 && s > 0) hold(s);
            const float s_w = weight_scale(s);
            meet();
            slab(now, s_w, [&](int g) { issue(s + AHEAD, fill, g * PER, g * PER + PER); });
            now = after(now), fill = after(fill);
        }
    } else {                                      // no rows for this wavefront: it brings the others theirs
        for (int s = 0; s < slabs; ++s) {
            meet();
            issue(s + AHEAD, fill, 0, LOADS);
            fill = after(fill);
        }
    }
    if (!mx_join<KS, SET, NT, CG>(acc, ks, sw, smem, lane)) return;
    if constexpr (KS == 1) {
        mx_meet();                                // (requests for slabs behind the last one: zeros, but they write to LDS)
        mx_store_rows<NT, CG, 16, 16>(p, t, smem + sw * mx_rows_lds<NT, CG, 16, 16>(), lane, idx, 4 * q, 16 * wm * NT, c0, acc, &bias);
    } else {
        mx_store_tile<NT, CG>(p, t, 16 * wm * NT + idx, c0 + 4 * q, acc, &bias);
    }
}

template <class T, bool COLD>
__global__ __launch_bounds__(T::THREADS, T::WAVES_PER_SIMD) void rows_tile_kernel(RowsProduct p) {
    extern __shared__ __align__(16) unsigned char smem[];
    RowsTask t;
    if (rows_task<T::BM>(p, T::BN, t)) rows_tile<T, COLD>(p, t, smem);
}

// -- large tiles: halves of a slab --
//
// What bounded the tiles above at these sizes were their loads: two stages are all that LDS has room for, a stage could be filled again once the whole
// slab in it was multiplied, and a slab ended in a wait for the slowest of its lines (8192 x 14336 x 14336 by 256 x 256: 1457 us; without the loads 928,
// without the products 1374).  Here a slab is consumed in halves -- all token rows and the first half of every wavefront's columns, then the second half
// -- with a meeting in front of each, and what a half leaves is filled for the slab after the next at once: requests are a slab and a half
// ahead instead of three quarters.  The last group's products wait for the next slab's meeting and run under its first reads.
//
// A slab of a 256 x 256 tile takes 1.75 us on random data, 1.47 on zeros; its loads alone 1.25, of which the rows' scales, 4 bytes of each row, are 0.25.
// (Scales of eight slabs at a time, 32 bytes of a row, gave 1.74 and 1.37 for long contractions but were slower for short ones.)
template <int RH_, int NT_, int CW_, int CG_>
struct RowsDeep {
    static constexpr int RH = RH_, NT = NT_, CW = CW_, CG = CG_, KS = 1;
    static constexpr int BM = 16 * NT * RH, BN = 16 * CG * CW;
    static constexpr int SET = RH * CW, THREADS = 64 * SET;
    static constexpr int HALF = CG / 2;
    static constexpr int LOADS_A = BM / 8 / SET, LOADS_H = BN / 16 / SET;      // an instruction of a wavefront brings 8 rows, or 8 columns of a half
    static constexpr int STAGE = (BM + BN) * 128 + SET * 256;  // (a place for scales for every wavefront, so that all of them make as many requests)
    static constexpr int LDS = std::max(2 * STAGE, SET * mx_rows_lds<NT, CG, 16, 16>());
    static constexpr int BLOCKS = std::min(160 * 1024 / LDS, 8 / SET);
    static constexpr int WAVES_PER_SIMD = BLOCKS * THREADS / 256;
    static_assert(CG % 2 == 0 && SET % 2 == 0 && BM % (8 * SET) == 0 && BN % (16 * SET) == 0 && BM <= 64 * SET && NT == 4, "every wavefront brings as many rows and columns");
    static_assert(128 % (16 * CG) == 0 && LDS <= 160 * 1024, "columns of one scale; LDS of a compute unit");
};

template <class T, bool COLD>
__device__ __forceinline__ void rows_deep(const RowsProduct& p, const RowsTask& t, unsigned char* smem) {
    constexpr int NT = T::NT, CG = T::CG, SET = T::SET, BM = T::BM, BN = T::BN, HALF = T::HALF;
    const int lane = threadIdx.x & 63, sw = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = sw / T::CW, wn = sw % T::CW;
    const int idx = lane & 15, q = lane >> 4;
    const int N = p.N, KB = p.K >> 7;
    const uint32_t K = (uint32_t)p.K;

    const int lrow = lane >> 3;
    const uint32_t chunk = (lane & 7) ^ (((8 * sw + lrow) >> 1) & 7);         // (rows_tile_kernel)
    const int64_t rows_all = p.token ? p.tokens : t.rows;
    const __amdgpu_buffer_rsrc_t a_buf = mx_buffer(t.a, (uint32_t)(rows_all * K)), w_buf = mx_buffer(t.w, (uint32_t)N * K),
                                 s_buf = mx_buffer(t.a_scales, (uint32_t)(rows_all * KB * 4));
    // Columns: half h of every wavefront column, eight at a time; in_tile: the first of the eight that instruction l of this wavefront brings.
    auto in_tile = [&](int h, int l) {
        const int j = l * SET + sw;
        return 16 * CG * (j / (2 * HALF)) + 16 * HALF * h + 8 * (j % (2 * HALF));
    };
    uint32_t w_off[2][T::LOADS_H];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int l = 0; l < T::LOADS_H; ++l) w_off[h][l] = (uint32_t)(t.n0 + in_tile(h, l) + lrow) * K + 16 * chunk;
    // Where a slab lies in the rows is a scalar offset (below K, which no buffer is shorter than: the range check compares with what it leaves of the
    // buffer).  Behind the last slab: the last one again, which nobody reads.
    auto issue_columns = [&](int s, int h, int l) {
        __builtin_amdgcn_raw_ptr_buffer_load_lds(w_buf, (mx_lds_void*)(smem + (s & 1) * T::STAGE + (BM + in_tile(h, l)) * 128), 16, (int)w_off[h][l], 128 * min(s, KB - 1), 0, COLD ? 2 : 0);
    };
#pragma unroll
    for (int j = 0; j < 2 * T::LOADS_H; ++j) issue_columns(0, j / T::LOADS_H, j % T::LOADS_H);
    uint32_t a_off[T::LOADS_A];
#pragma unroll
    for (int i = 0; i < T::LOADS_A; ++i) {
        const uint32_t src = rows_source(p, t, 8 * (i * SET + sw) + lrow);
        a_off[i] = src == kNoRow ? kBehind : src * K + 16 * chunk;
    }
    const uint32_t s_src = rows_source(p, t, 64 * sw + lane), s_off = s_src == kNoRow ? kBehind : s_src * (uint32_t)KB * 4;
    auto issue_rows = [&](int s, int i) {
        __builtin_amdgcn_raw_ptr_buffer_load_lds(a_buf, (mx_lds_void*)(smem + (s & 1) * T::STAGE + (i * SET + sw) * 1024), 16, (int)a_off[i], 128 * min(s, KB - 1), 0, 0);
        if (i == 0)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(s_buf, (mx_lds_void*)(smem + (s & 1) * T::STAGE + (BM + BN) * 128 + sw * 256), 4, (int)s_off, 4 * min(s, KB - 1), 0, 0);
    };
    // Requests are one to a group of products: a wavefront whose requests queue at the address unit issues nothing else.  Slab s in its order:
    // the first half of the columns of slab s + 1 behind the first meeting, then the second half of it, and behind the second meeting the
    // rows of slab s + 2.  So behind what the first meeting waits for came a half of columns and a slab's rows, behind the second one's as
    // much and two halves of columns.
    constexpr int ROWS_IN_ALL = T::LOADS_A + 1;
    auto meet_first = [] { mx_meet<T::LOADS_H + ROWS_IN_ALL>(); };
    auto meet_second = [] { mx_meet<2 * T::LOADS_H + ROWS_IN_ALL>(); };
    const int c0 = t.n0 + 16 * CG * wn;
    const float* const ws = t.s + (int64_t)min(c0 >> 7, (N - 1) >> 7) * KB;
    float held = lane < KB ? ws[lane] : 0.0f;     // the weights' scales of 64 slabs (rows_tile_kernel)
    constexpr bool EARLY = CG <= 4;               // (the widest tile has no registers for its bias)
    MxBias<CG, 16> bias;
    if (EARLY) bias.fetch(p, t, c0 + 4 * q);
    auto hold = [&](int s) {
        held = s + lane < KB ? ws[s + lane] : 0.0f;
        asm volatile("" : "+v"(held));            // (the wait for it is here, not in every slab)
    };

    mx_f32x4 acc[NT][CG];
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int g = 0; g < CG; ++g) acc[i][g] = mx_f32x4{0.f, 0.f, 0.f, 0.f};

    auto request = [&](int s, int g) {            // in front of group g of slab s (group CG - 1: that of the slab before, behind the first meeting)
        // order: CG - 1, 0, .. HALF - 2 | HALF - 1, .. CG - 2
        const int n = g == CG - 1 ? 0 : g + 1;
        if (n < HALF) {
#pragma unroll
            for (int j = 2 * T::LOADS_H * n / HALF; j < 2 * T::LOADS_H * (n + 1) / HALF; ++j) issue_columns(s + 1, j / T::LOADS_H, j % T::LOADS_H);
        } else {
#pragma unroll
            for (int j = T::LOADS_A * (n - HALF) / HALF; j < T::LOADS_A * (n - HALF + 1) / HALF; ++j) issue_rows(s + 2, j);
        }
    };
    // what slabs -1 and -2 would have asked for, columns first: of rows that are fetched by index the indices have to come before
#pragma unroll
    for (int i = 0; i < T::LOADS_A; ++i) issue_rows(0, i);
#pragma unroll
    for (int i = 0; i < T::LOADS_A; ++i) issue_rows(1, i);
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(ROWS_IN_ALL) : "memory");      // (slab 0's rows came behind its columns)
    asm volatile("" : "+v"(held));
    if (t.rows > wm * 16 * NT) {
        mx_i32x8 x[NT], w[2];
        float sc[NT], sc_next[NT];
        mx_f32x4 part[NT];
#pragma unroll
        for (int i = 0; i < NT; ++i) {
            x[i] = mx_i32x8{};
            sc[i] = 0.0f;
            part[i] = mx_f32x4{0.f, 0.f, 0.f, 0.f};
        }
        w[0] = w[1] = mx_i32x8{};
        const int at0 = (q ^ (idx >> 1)) << 4, at1 = ((4 + q) ^ (idx >> 1)) << 4;
        auto read = [&](const unsigned char* b, int i) {
            return rows_operand(*reinterpret_cast<const mx_u32x4*>(b + i * 16 * 128 + at0), *reinterpret_cast<const mx_u32x4*>(b + i * 16 * 128 + at1));
        };
        // Products of group g.  A product is folded three instructions later, so the first three here fold what is left of group `last`.
        auto fold = [&](int i, int g, float scale) {
#pragma unroll
            for (int r = 0; r < 4; ++r) acc[i][g][r] = __builtin_fmaf(part[i][r], scale, acc[i][g][r]);
        };
        auto group = [&](int g, int last, const float (&last_scale)[NT], const float (&scale)[NT]) {
#pragma unroll
            for (int i = 0; i < NT; ++i) {
                part[i] = rows_mfma(w[g & 1], x[i]);
                if (i + 1 < NT) fold(i + 1, last, last_scale[i + 1]);
                else fold(0, g, scale[0]);
            }
#pragma unroll
            for (int i = 0; i < NT; ++i) {
                __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);      // a matrix instruction,
                __builtin_amdgcn_sched_group_barrier(0x2, 4, 0);      // four of the vector ALU
            }
            __builtin_amdgcn_sched_barrier(0);
        };
        for (int s = 0; s < KB; ++s) {
            if ((s & 63) == 0 && s > 0) hold(s);
            const float s_w = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, held), s & 63));
            const unsigned char* st = smem + (s & 1) * T::STAGE;
            const unsigned char* xb = st + (wm * 16 * NT + idx) * 128;
            const unsigned char* wb = st + (BM + wn * 16 * CG + idx) * 128;
            const float* sb = reinterpret_cast<const float*>(st + (BM + BN) * 128) + wm * 16 * NT + idx;
            meet_first();
            w[0] = read(wb, 0);
            request(s, CG - 1);
            __builtin_amdgcn_sched_barrier(0);
            group(CG - 1, CG - 2, sc, sc);        // of the slab before
#pragma unroll
            for (int i = 0; i < NT; ++i) x[i] = read(xb, i);
#pragma unroll
            for (int i = 0; i < NT; ++i) sc_next[i] = sb[16 * i] * s_w;
            w[1] = read(wb, 1);
            request(s, 0);
            __builtin_amdgcn_sched_barrier(0);
            group(0, CG - 1, sc, sc_next);
#pragma unroll
            for (int i = 0; i < NT; ++i) sc[i] = sc_next[i];
#pragma unroll
            for (int g = 1; g < CG - 1; ++g) {
                if (g == HALF - 1) meet_second();
                w[(g + 1) & 1] = read(wb, g + 1);
                request(s, g);
                __builtin_amdgcn_sched_barrier(0);
                group(g, g - 1, sc, sc);
            }
        }
        group(CG - 1, CG - 2, sc, sc);
#pragma unroll
        for (int i = 1; i < NT; ++i) fold(i, CG - 1, sc[i]);
    } else {                                      // no rows for this wavefront: it brings the others theirs
        for (int s = 0; s < KB; ++s) {
            meet_first();
#pragma unroll
            for (int n = 0; n < CG; ++n) {
                if (n == HALF) meet_second();
                request(s, n == 0 ? CG - 1 : n - 1);
            }
        }
    }
    mx_meet();                                    // (the requests behind the last slab write to LDS)
    mx_store_rows<NT, CG, 16, 16>(p, t, smem + sw * mx_rows_lds<NT, CG, 16, 16>(), lane, idx, 4 * q, 16 * wm * NT, c0, acc, EARLY ? &bias : nullptr);
}

// The last round of blocks of 256 rows in halves, and what such blocks leave of an expert or of the one matrix, by smaller tiles behind the large ones.  Large
// tiles for all / this, us: 2037 x 10624 x 4608 115 / 103, 3678 x 9216 x 3840 150 / 137, 1435 x 14336 x 5376 129 / 113; 8 experts of 6016 x 5760, 3104 rows 150 /
// 132, of 4096 x 14336, 16384 rows 950 / 925 (its pieces take 40 us, and the eight matrices' way from
// memory 45: so much less where all of them lie at one address; the rest is 2.3 PFLOP/s).
typedef RowsDeep<2, 4, 4, 4> RowsLeft;
typedef RowsTile<1, 4, 4, 2, 2, 2> RowsPiece;
template <class T>
constexpr int rows_lds() { return T::BM == 256 ? std::max(T::LDS, std::max(RowsLeft::LDS, RowsPiece::LDS)) : T::LDS; }

template <class T, bool COLD>
__global__ __launch_bounds__(T::THREADS, T::WAVES_PER_SIMD) void rows_deep_kernel(RowsProduct p) {
    extern __shared__ __align__(16) unsigned char smem[];
    RowsTask t;
    if (!rows_task<T::BM>(p, T::BN, t)) return;
    if constexpr (T::BM == 256) {
        static_assert(RowsLeft::BM == kLeftRows && RowsLeft::BN == T::BN && RowsLeft::THREADS == T::THREADS && RowsPiece::BM == kPieceRows && 2 * RowsPiece::BN == T::BN && RowsPiece::THREADS == T::THREADS, "");
        if (t.kind == kLeftTask) return rows_deep<RowsLeft, COLD>(p, t, smem);
        if (t.kind == kPieceTask) return rows_tile<RowsPiece, COLD>(p, t, smem);
    }
    rows_deep<T, COLD>(p, t, smem);
}

// ---- launches ----

// Workgroups of a launch: blocks of BM rows times column tiles, in eight equal shares.  Experts' blocks are counted on the device; M rows on n experts
// that have any fill (M + n (BM - 1)) / BM of them at most; with pieces, the blocks in front of those and a workgroup for each of them; with
// halves, half a round more.
int64_t rows_grid(const RowsProduct& p, int BM, int BN) {
    if (!p.count) {
        const RowsDense d = rows_dense(p, BM, BN);
        return 8 * (d.share + d.halved + d.left_share);
    }
    const int64_t ncol = (p.N + BN - 1) / BN, n = std::min<int64_t>(p.E, p.M);
    int64_t tiles = (p.M + n * (BM - 1)) / BM * ncol;
    if (BM == 256) tiles = std::max(tiles, (p.M + n * (BM - 1 - kLeftRows)) / BM * ncol + kGroupedUnits) + kGroupedUnits / 2;
    return (tiles + 7) / 8 * 8 + 16;
}

// Weights that are not kept behind their one reading: more than the memory-side cache would hold for the next call, and about one block of
// rows for each.  Kept / not, us: 65536 x 4096 for one row 51.5 / 46.4; 256 experts of 2048 x 7168, 128 rows 303 / 277, 512 rows 624 / 563; 8 of 14336 x
// 4096, 128 rows 98 / 86 -- but 14336 x 4096 for 48 rows, which the cache holds, 12.4 / 15.3, and many rows on 8 of 4096 x 14336 1225 / 1640.  Between two
// calls with an expert's matrix come those with the layer's others, so half of the cache is enough: 64 of 1408 x 2048, three layers in
// turn, 30 rows each 39.8 / 35.5, 94 rows 50.1 / 48.7, 32 of 2048 x 4096, 12 rows 62.9 / 56.2 (a single matrix again and again 30.4 / 35.2, 40 / 44.5, 40.7 / 53.7).
bool rows_cold(const RowsProduct& p, int block_rows) {
    const int64_t experts = p.count ? std::min<int64_t>(p.E, p.M) : 1;
    return p.M <= experts * block_rows && experts * p.N * p.K > ((int64_t)(p.count ? 128 : 256) << 20);
}

struct RowsCut {
    bool wide;
    int KS;
    int64_t waves;
    int chunks;                 // of a wavefront, whole turns
};
RowsCut rows_cut(const RowsProduct& p) {
    const int64_t blocks = p.count ? std::min<int64_t>(p.E, p.M) : (p.M + 15) / 16, groups = blocks * ((p.N + 15) / 16);
    const int chunks = p.K / 128;
    RowsCut c{groups >= 512, 1, 0, 0};
    c.waves = c.wide ? (groups + 1) / 2 : groups;
    while (c.KS < kRowsWaves && 2 * kDepth * c.KS <= chunks && c.waves * 2 <= 4096) c.KS *= 2, c.waves *= 2;
    c.chunks = ((chunks + c.KS - 1) / c.KS + kDepth - 1) / kDepth * kDepth;
    return c;
}
hipError_t launch_rows_stream(const RowsProduct& p, hipStream_t st) {
    const RowsCut c = rows_cut(p);
    const bool cold = rows_cold(p, 16);
    const unsigned grid = (unsigned)rows_grid(p, 16, 16 * (c.wide ? 2 : 1) * (kRowsWaves / c.KS));
    auto launch = [&](auto kernel) {
        kernel<<<grid, 64 * kRowsWaves, 0, st>>>(p, c.KS);
        return hipGetLastError();
    };
    const bool more = p.count || p.M > 8;
    auto rows = [&](auto g, auto m) { return cold ? launch(rows_stream_kernel<decltype(g)::value, decltype(m)::value, true>) : launch(rows_stream_kernel<decltype(g)::value, decltype(m)::value, false>); };
    auto columns = [&](auto g) { return more ? rows(g, std::true_type{}) : rows(g, std::false_type{}); };
    return c.wide ? columns(std::integral_constant<int, 2>{}) : columns(std::integral_constant<int, 1>{});
}
template <class T, bool COLD>
struct RowsKernel { static constexpr void (*kernel)(RowsProduct) = rows_tile_kernel<T, COLD>; };
template <int RH, int NT, int CW, int CG, bool COLD>
struct RowsKernel<RowsDeep<RH, NT, CW, CG>, COLD> { static constexpr void (*kernel)(RowsProduct) = rows_deep_kernel<RowsDeep<RH, NT, CW, CG>, COLD>; };
template <class T, bool COLD>
hipError_t launch_rows_tile(const RowsProduct& p, hipStream_t st) {
    const hipError_t e = allow_lds(RowsKernel<T, COLD>::kernel, rows_lds<T>());
    if (e != hipSuccess) return e;
    RowsKernel<T, COLD>::kernel<<<(unsigned)rows_grid(p, T::BM, T::BN), T::THREADS, rows_lds<T>(), st>>>(p);
    return hipGetLastError();
}

// Forms: 0 the streamer, from 1 on these tiles.  f(the tile's type, as a pointer to nothing).
template <class F>
auto with_rows_tile(int form, F f) {
    switch (form) {
        case 1: return f((RowsTile<1, 1, 2, 2, 4, 2>*)nullptr);      // 16 x 64
        case 2: return f((RowsTile<1, 2, 4, 1, 2, 3>*)nullptr);      // 32 x 64
        case 3: return f((RowsTile<1, 4, 4, 1, 2, 2>*)nullptr);      // 64 x 64
        case 4: return f((RowsTile<1, 4, 4, 2, 1, 2>*)nullptr);      // 64 x 128
        case 5: return f((RowsDeep<2, 4, 2, 4>*)nullptr);            // 128 x 128
        case 6: return f((RowsDeep<2, 4, 4, 4>*)nullptr);            // 128 x 256
        default: return f((RowsDeep<4, 4, 2, 8>*)nullptr);           // 256 x 256
    }
}

// What a tile costs, in us: a launch of its form; a slab of the contraction where a compute unit has one tile; the same for every further tile of the
// unit.  Fitted to 575 products of 1 to 6000 rows, 4 to 1000 us, dense and of experts, evenly and not, each with every form: the choice by
// these was 1.0 % behind the best of the forms on average.  Over some 1500 others it is 0.8 % behind for one matrix and 2.0 % for experts
// (a fit to those alone 0.7 and 1.2), 50 % at worst (23 rows on 4 experts of 1152 x 7168, 16.4 us).
struct RowsCost {
    int rows, columns;
    float launch, slab, more;
};
constexpr RowsCost kRowsTiles[] = {{}, {16, 64, 3.88f, 0.153f, 0.458f}, {32, 64, 3.63f, 0.252f, 0.493f}, {64, 64, 4.54f, 0.25f, 0.969f}, {64, 128, 3.92f, 0.37f, 0.483f},
                                   {128, 128, 5.16f, 0.754f, 0.553f}, {128, 256, 4.3f, 0.866f, 1.41f}, {256, 256, 6.36f, 1.467f, 1.478f}};

// The form that should take least; 0: the streamer.  Of experts' rows the host knows how many there are, not whose: a block an expert where the
// mean is small for it, else half a block more than the mean fills.
int block_form(const RowsProduct& p) {
    const int64_t experts = p.count ? std::min<int64_t>(p.E, p.M) : 1;
    const double each = (double)p.M / experts;
    const RowsCut c = rows_cut(p);
    auto row_blocks = [&](int rows) { return !p.count ? (double)((p.M + rows - 1) / rows) : each > 0.6 * rows ? (double)p.M / rows + 0.5 * experts : (double)experts; };
    const double rounds = std::max(1.0, c.waves / 2048.0) * (p.count ? row_blocks(16) / experts : 1.0);
    double best = each > 16 ? 1e30 : 2.83 + 0.0545 * each + c.chunks * rounds * ((c.wide ? 1.565 : 0.868) + 0.0135 * each);
    int form = 0;
    for (int f = 1; f < (int)(sizeof kRowsTiles / sizeof kRowsTiles[0]); ++f) {
        const RowsCost& t = kRowsTiles[f];
        double tiles = std::ceil(row_blocks(t.rows) * ((p.N + t.columns - 1) / t.columns) / 256.0);      // of the compute unit that has most
        if (t.rows == 256 && tiles - row_blocks(t.rows) * ((p.N + t.columns - 1) / t.columns) / 256.0 >= 0.5) tiles -= 0.4;      // halves in the last round
        const double cost = t.launch + p.K / 128 * (t.slab + t.more * (tiles - 1));
        if (cost < best) best = cost, form = f;
    }
    return form;
}
int64_t block_workgroups(const RowsProduct& p, int form) {
    return form == 0 ? rows_grid(p, 16, 16) : rows_grid(p, kRowsTiles[form].rows, kRowsTiles[form].columns);
}

}  // namespace

// What the kernels read and write at a time, their 32-bit offsets and the launches' sizes; and the kernel that the product takes.
int check_product_block128(const RowsProduct& p, int* form) {
    auto off = [](const void* a, uintptr_t n) { return (uintptr_t)a % n != 0; };
    if (p.M < 0 || p.tokens < 0 || p.N < 1 || p.K < 128 || p.K % 128 || !p.w || !p.s) return MOE_ERR_BAD_ARGUMENT;
    if (p.act != MOE_ACT_RELU && p.act != MOE_ACT_GELU && p.act != MOE_ACT_NONE) return MOE_ERR_BAD_ARGUMENT;
    if (p.M > 0 && (!p.a || !p.a_scales || !p.out)) return MOE_ERR_BAD_ARGUMENT;
    if (off(p.a, 16) || off(p.w, 16) || off(p.out, 16) || off(p.a_scales, 4) || off(p.s, 4) || off(p.bias, 2) || off(p.token, 4)) return MOE_ERR_BAD_ARGUMENT;
    if (p.K > (1 << 20) || (int64_t)p.N * p.K >= kBufferBytes || p.M > INT32_MAX) return MOE_ERR_UNSUPPORTED;
    if (p.token && (p.tokens > INT32_MAX || p.tokens * p.K >= kBufferBytes)) return MOE_ERR_UNSUPPORTED;
    *form = block_form(p);
    return block_workgroups(p, *form) < ((int64_t)1 << 22) ? MOE_OK : MOE_ERR_UNSUPPORTED;      // 512 threads each: 2^31
}

hipError_t launch_product_block128(const RowsProduct& p, int form, hipStream_t st) {
    if (p.M == 0) return hipSuccess;
    if (form == 0) return launch_rows_stream(p, st);
    return with_rows_tile(form, [&](auto* t) {
        typedef std::remove_pointer_t<decltype(t)> T;
        return rows_cold(p, T::BM) ? launch_rows_tile<T, true>(p, st) : launch_rows_tile<T, false>(p, st);
    });
}

}  // namespace moe355

using namespace moe355;

extern "C" int moe_gemm_block128(const void* a, const float* a_scales, const void* w, const float* w_scales, const void* bias, void* out, int64_t M, int64_t N,
                                 int64_t K, int32_t act, void* stream) {
    if (M < 0 || N < 1 || K < 1) return MOE_ERR_BAD_ARGUMENT;
    if (N > INT32_MAX / 2 || K > INT32_MAX / 2) return MOE_ERR_UNSUPPORTED;
    const RowsProduct p{(const uint8_t*)a, a_scales, (const uint8_t*)w, w_scales, (const uint16_t*)bias, nullptr, nullptr, nullptr, (uint16_t*)out, M, M, (int)N, (int)K, 1, act};
    int form;
    const int rc = check_product_block128(p, &form);
    if (rc) return rc;
    return launch_product_block128(p, form, (hipStream_t)stream) == hipSuccess ? MOE_OK : MOE_ERR_HIP;
}

extern "C" int moe_gemm_block128_plan(int64_t M, int64_t N, int64_t K, int32_t experts, int32_t* rows, int32_t* columns, int32_t* parts) {
    if (M < 1 || N < 1 || K < 1 || experts < 0 || experts > kMaxExperts || !rows || !columns || !parts) return MOE_ERR_BAD_ARGUMENT;
    if (N > INT32_MAX / 2 || K > INT32_MAX / 2) return MOE_ERR_UNSUPPORTED;
    // an operand that is there, as far as the choice looks at it
    alignas(16) static const uint8_t some[16] = {};
    alignas(16) static uint16_t result[8];
    const int32_t* const table = experts ? reinterpret_cast<const int32_t*>(some) : nullptr;
    const float* const scales = reinterpret_cast<const float*>(some);
    const RowsProduct p{some, scales, some, scales, nullptr, table, table, nullptr, result, M, M, (int)N, (int)K, experts ? experts : 1, MOE_ACT_NONE};
    int form;
    const int rc = check_product_block128(p, &form);
    if (rc) return rc;
    if (form == 0) {
        const RowsCut c = rows_cut(p);
        *rows = 16, *columns = c.wide ? 32 : 16, *parts = c.KS;
    } else {
        with_rows_tile(form, [&](auto* t) {
            typedef std::remove_pointer_t<decltype(t)> T;
            *rows = T::BM, *columns = T::BN, *parts = T::KS;
        });
    }
    return MOE_OK;
}
