// Which tile of a grouped product (packed rows, a matrix per expert) a workgroup takes, from the experts' row counts alone.
#pragma once

#include "ffn_common.hpp"

namespace moe355 {
namespace {

constexpr int kShareSlack = 14;      // workgroups without a tile, at most: the two lists are rounded up to eight equal shares
// Row blocks of an expert that are taken at a time, all column tiles of those: the 32 tiles that an XCD works on then share 8 row
// blocks and 4 weight tiles instead of one weight tile.  One expert's row blocks all at a time / 8, us: one expert of 4096 x 4096, 8192
// rows, up projection 220 / 208, its data gradient 236 / 225; 2 of them 251 / 246; 8 of 1408 x 2048, 4096 rows 201 / 197; 4 of 2048 x 2048,
// 3072 rows 113 / 109; 4 of 2560 x 2048, 4096 rows 144 / 146; a layer of one expert of 2048 x 2048, SwiGLU, 8192 rows 218 / 212.
constexpr int kRowChunk = 8;
struct GroupedTask {
    int expert, row0, rows, ctile;
    bool piece;      // (with PIECE) a remainder's piece: ctile counts half tiles
};
// The sum over this lane and those in front of it: DPP moves within rows of 16 lanes, then the last lane of one row to the next, and of one half
// to the other.  (Six steps through LDS by __shfl_up take some 600 cycles, in which nothing of the tile is on its way.)
__device__ __forceinline__ int lanes_before(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);
    return v;
}
// Which tile workgroup `id` of a grouped product takes, from the experts' row counts alone; false: none.  Order: the row blocks of
// full height, expert by expert, column tile by column tile, an expert's row blocks (kRowChunk of them) fastest (few row blocks stay in the
// caches while its column tiles pass by); with 256-row blocks, behind them the remainders of at most 128 rows: the long tasks start
// first, and the short ones fill the compute units that the last round of long ones leaves idle.  Workgroups go to the eight XCDs in
// turn: each XCD takes an eighth of either list in a row, so that the tiles that share a weight tile or token rows share an L2.
// Every wavefront works it out for itself, an expert a lane, which takes less time than a launch in front that writes tables.
// One product, bf16, the launch and table in front of 256-row blocks alone against this: 16 experts of 2048 x 2048, about 512 rows each
// 109 -> 80 us; 8 of 4096 x 2048, 2048 rows 274 -> 234; 64 of 2048 x 1408, 94 rows 94 -> 89; 16 of 2048 x 1408, 750 rows 91 -> 73.
// The share of an XCD in a row, against the list dealt out to them: whole layers as two launches, 8 experts of 4096 x 14336, 2048 rows
// 4679 -> 4431 us, 1024 rows 2860 -> 2484; 64 of 2048 x 1408, 1536 rows 1863 -> 1662, 750 rows 1089 -> 907; 12 of 1344 x 2752, 444 rows
// 174 -> 165, 150 rows 125 -> 107.
// PIECE > 0: the last round of an XCD's compute units in smaller tiles, where it has a unit for each of those: blocks in halves, or, where no block is
// in it, remainders in pieces of so many rows and half a tile's columns.
constexpr int kGroupedUnits = 256, kXcdUnits = kGroupedUnits / 8;      // compute units
__host__ __device__ __forceinline__ int64_t halved_blocks(int64_t share, int64_t left_share) {      // of the tiles of an XCD, the last ones
    const int64_t rest = share % kXcdUnits;
    return 2 * rest + left_share <= kXcdUnits ? rest : 0;
}
template <int BIG, int PIECE = 0>
__device__ __forceinline__ bool grouped_task(const int32_t* __restrict__ count, const int32_t* __restrict__ offset, int E, int ncol, int id, GroupedTask& t) {
    constexpr int LEFT = BIG == 256 ? 128 : 0;          // rows up to which what is left of an expert is a block of its own kind
    const int lane = threadIdx.x & 63;
    // (the first 64 experts' counts and offsets in one trip to memory)
    const int first_rows = lane < E ? max(count[lane], 0) : 0, first_offset = lane < E ? offset[lane] : 0;
    auto rows_of = [&](int c) { return c == 0 ? first_rows : c + lane < E ? max(count[c + lane], 0) : 0; };
    auto offset_of = [&](int c) { return c == 0 ? first_offset : c + lane < E ? offset[c + lane] : 0; };
    auto big_of = [&](int n) { return (n + BIG - 1 - LEFT) / BIG; };
    int big_sum = 0, left_sum = 0, piece_sum = 0;         // full row blocks and remainders of all experts
    for (int c = 0; c < E; c += kWave) {
        const int n = rows_of(c), big = big_of(n);
        big_sum += __builtin_amdgcn_readlane(lanes_before(big), kWave - 1);
        left_sum += __popcll(__ballot(n > big * BIG));
        if (PIECE) piece_sum += __popcll(__ballot(n > big * BIG)) + __popcll(__ballot(n > big * BIG + PIECE));
    }
    const bool pieces = PIECE && (big_sum * ncol + 7) / 8 % kXcdUnits == 0 && 2 * piece_sum * ncol <= kGroupedUnits;
    const int left_cols = pieces ? 2 * ncol : ncol, bigs = big_sum * ncol, lefts = (pieces ? piece_sum : left_sum) * left_cols;
    const int big_share = (bigs + 7) / 8, left_share = (lefts + 7) / 8, halved = PIECE ? (int)halved_blocks(big_share, left_share) : 0;
    int half = -1;
    if (id < 8 * (big_share + halved)) {
        int i = id >> 3;
        const int whole = big_share - halved;
        if (PIECE && i >= whole) half = (i - whole) & 1, i = whole + ((i - whole) >> 1);
        id = (id & 7) * big_share + i;
        if (id >= bigs) return false;
    } else {
        id -= 8 * (big_share + halved);
        if ((id >> 3) >= left_share) return false;
        id = (id & 7) * left_share + (id >> 3) + bigs;
        if (id >= bigs + lefts) return false;
    }
    int base = 0;                          // full row blocks of the experts in front
    for (int c = 0; c < E; c += kWave) {
        const int n = rows_of(c), o = offset_of(c), big = big_of(n);
        const int inc = lanes_before(big);
        const int total = __builtin_amdgcn_readlane(inc, kWave - 1);
        if (id < (base + total) * ncol) {
            const int l = __builtin_ctzll(__ballot((base + inc) * ncol > id));
            const int blocks = __builtin_amdgcn_readlane(big, l), first = base + __builtin_amdgcn_readlane(inc, l) - blocks;
            int local = id - first * ncol, rb = 0, width = blocks;
            if (blocks > kRowChunk) {
                rb = local / (kRowChunk * ncol) * kRowChunk;
                width = min(kRowChunk, blocks - rb);
                local -= rb * ncol;
            }
            t.ctile = local / width;
            rb += local - t.ctile * width;
            t.expert = c + l;
            t.rows = min(BIG, __builtin_amdgcn_readlane(n, l) - rb * BIG);
            t.row0 = __builtin_amdgcn_readlane(o, l) + rb * BIG;
            t.piece = false;
            if (PIECE && half >= 0) t.row0 += half * (BIG / 2), t.rows = min(t.rows - half * (BIG / 2), BIG / 2);
            return true;
        }
        base += total;
    }
    if constexpr (LEFT > 0) {
        static_assert(PIECE == 0 || LEFT <= 2 * PIECE, "two pieces a remainder");
        int before = (id - base * ncol) / left_cols;      // remainders, or pieces' rows, in front of this one
        t.ctile = (id - base * ncol) - before * left_cols;
        t.piece = pieces;
        for (int c = 0; c < E; c += kWave) {
            const int n = rows_of(c), o = offset_of(c), left = max(n - big_of(n) * BIG, 0);
            unsigned long long m = __ballot(left > 0);
            const int first = __popcll(m);
            const unsigned long long m2 = pieces ? __ballot(left > PIECE) : 0;
            const int here = first + __popcll(m2);
            if (before < here) {
                const int behind = before < first ? 0 : PIECE;      // rows of the remainder in front
                if (before >= first) m = m2, before -= first;
                const int rank = __popcll(m & ((1ull << lane) - 1ull));
                const int l = __builtin_ctzll(__ballot(((m >> lane) & 1) && rank == before));
                t.expert = c + l;
                t.rows = __builtin_amdgcn_readlane(left, l);
                t.row0 = __builtin_amdgcn_readlane(o, l) + (__builtin_amdgcn_readlane(n, l) - t.rows) + behind;
                t.rows -= behind;
                if (pieces) t.rows = min(t.rows, PIECE);
                return true;
            }
            before -= here;
        }
    }
    return false;
}

}  // namespace
}  // namespace moe355
