// Products whose weights are MXFP4 (mxfp4.hpp): out = act(a . w^T + bias), w [N][K] codes with a scale for 32 values of a row, the rows a
// in bf16 or in MXFP4 too; one matrix, or a matrix per expert over packed rows.  Sums in fp32, rounded once on store.
//
// Three kinds of kernel: a weight streamer for up to 16 rows a block; tiles for bf16 rows, on the bf16 instructions, the weights widened between
// LDS and them; tiles for MXFP4 rows, on the scaled instructions.  product_form() takes the one whose fitted cost is least.
#include "grouped_task.hpp"
#include "product_rows.hpp"

namespace moe355 {
namespace {

struct MxTask {
    const char* a;            // the block's first row
    const uint8_t* a_scales;  // ... and its scales (rows in MXFP4)
    const char* w;            // the expert's matrix
    const uint8_t* s;
    const uint16_t* bias;     // of the expert, or null
    uint16_t* out;            // at the block's first row
    int64_t row0;
    int rows, n0;
};

// Which block of BM rows and which BN columns a workgroup takes.
template <int BM, bool ROWS4>
__device__ __forceinline__ bool mx_task(const MxProduct& p, int BN, MxTask& t) {
    const int ncol = (p.N + BN - 1) / BN;
    int expert = 0, ctile, rows;
    int64_t row0;
    if (p.count) {
        GroupedTask g;
        if (!grouped_task<BM>(p.count, p.offset, p.E, ncol, (int)blockIdx.x, g)) return false;
        expert = g.expert, ctile = g.ctile, row0 = g.row0, rows = g.rows;
        if (row0 < 0 || row0 + rows > p.M) return false;          // tables that are not this layer's: nothing behind the buffers is touched
    } else {
        // an eighth of the tiles in a row for each XCD, kRowChunk row blocks at a time, as for the experts
        const int blocks = (int)((p.M + BM - 1) / BM);
        const int64_t total = (int64_t)blocks * ncol, share = (total + 7) / 8;
        const int64_t id = (int64_t)(blockIdx.x & 7) * share + (blockIdx.x >> 3);
        if ((int64_t)(blockIdx.x >> 3) >= share || id >= total) return false;
        int rb = (int)(id / ((int64_t)kRowChunk * ncol)) * kRowChunk;
        const int width = min(kRowChunk, blocks - rb), local = (int)(id - (int64_t)rb * ncol);
        ctile = local / width;
        rb += local - ctile * width;
        row0 = (int64_t)rb * BM;
        rows = (int)min((int64_t)BM, p.M - row0);
    }
    // the same in every lane, and said so
    row0 = mx_uniform(row0), expert = __builtin_amdgcn_readfirstlane(expert), ctile = __builtin_amdgcn_readfirstlane(ctile), rows = __builtin_amdgcn_readfirstlane(rows);
    const int64_t arow = ROWS4 ? p.K >> 1 : 2 * (int64_t)p.K;
    t.row0 = row0;
    t.a = static_cast<const char*>(p.a) + row0 * arow;
    t.a_scales = ROWS4 ? p.a_scales + row0 * (p.K >> 5) : nullptr;
    t.w = static_cast<const char*>(p.w) + (int64_t)expert * p.N * (p.K >> 1);
    t.s = p.s + (int64_t)expert * p.N * (p.K >> 5);
    t.bias = p.bias ? p.bias + (int64_t)expert * p.N : nullptr;
    t.out = p.out + row0 * p.N;
    t.rows = rows;
    t.n0 = ctile * BN;
    return true;
}

// ---- up to 16 rows a block: a weight streamer ----
constexpr int kStreamWaves = 8;

// KS wavefronts share a contraction, a share in a row each, 8 / KS sets of 16 CG columns a workgroup.  rows_most: token rows that LDS is there for.
// Bound by memory (skinny.hpp).  One row times 4096 x 14336: 8.9 us, 2.4 of them the launch; 16 rows 13.7.
template <bool ROWS4, int CG, bool COLD>
__global__ __launch_bounds__(64 * kStreamWaves) void mx_stream_kernel(MxProduct p, int KS, int rows_most) {
    typedef WeightsMx<ROWS4> W;
    extern __shared__ __align__(16) unsigned char smem[];
    __shared__ mx_f32x4 red[(kStreamWaves - 1) * CG * 64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int ks = wave % KS, set = wave / KS;
    MxTask t;
    if (!mx_task<16, ROWS4>(p, 16 * CG * (kStreamWaves / KS), t)) return;
    const int n0 = t.n0 + 16 * CG * set, K = p.K;
    Skinny<W, CG, COLD> st;
    st.init(smem + wave * skinny_lds<W>(rows_most), rows_most, K);
#pragma unroll
    for (int g = 0; g < CG; ++g) {
        st.w_buf[g] = mx_buffer(t.w, (uint32_t)p.N * st.row);
        st.s_at[g] = t.s;
    }
    st.x_buf = mx_buffer(t.a, (uint32_t)t.rows * st.x_row);
    st.aim_weights(n0, p.N, 16);
    st.aim_tokens(t.rows, [](int r) { return r; });
    if constexpr (ROWS4) {
        st.sx_at = p.a_scales;                    // (the whole array: the eight bytes at the end of a block's may lie behind it)
        st.sx_base = t.row0 * (K >> 5);
        st.sx_end = p.M * (K >> 5) - 8;
        st.sx_row = (uint32_t)min(lane >> 2, t.rows - 1) * (uint32_t)(K >> 5);
    }
    const int chunks = (K + W::K - 1) / W::K, share = (chunks + KS - 1) / KS;
    const int begin = min(ks * share, chunks), end = min(begin + share, chunks), n = (end - begin + kUnit - 1) / kUnit;
    mx_f32x4 acc[1][CG] = {};
    st.run(n, acc[0], [&](int u) { st.chunk0 = begin + kUnit * u, st.chunk_end = u < n ? end : 0; }, [](int) {});
    if (!skinny_join<CG>(acc[0], ks, KS, red + set * (KS - 1) * CG * 64, lane)) return;
    mx_store_tile<1, CG>(p, t, lane & 15, n0 + 4 * (lane >> 4), acc);
}

// A matrix of fewer than 256 values, which has no eight scales in a row to fetch: a value of the result a thread.
template <bool ROWS4>
__global__ __launch_bounds__(256) void mx_small_kernel(MxProduct p) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= p.M * p.N) return;
    const int64_t m = i / p.N;
    const int n = (int)(i - m * p.N);
    int e = 0;
    if (p.count) {
        while (e < p.E && (m < p.offset[e] || m >= (int64_t)p.offset[e] + p.count[e])) ++e;
        if (e == p.E) return;                     // no expert's row
    }
    auto value = [&](const void* codes, const uint8_t* scales, int64_t row, int k) {
        const uint32_t c = static_cast<const uint8_t*>(codes)[row * (p.K >> 1) + (k >> 1)] >> (4 * (k & 1));
        return __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c & 15u, mx_scale(scales[row * (p.K >> 5) + (k >> 5)]), 0)[0];
    };
    float sum = 0.0f;
    for (int k = 0; k < p.K; ++k) {
        const float a = ROWS4 ? value(p.a, p.a_scales, m, k) : bf16_bits_to_f32(static_cast<const uint16_t*>(p.a)[m * p.K + k]);
        sum = __builtin_fmaf(a, value(p.w, p.s, (int64_t)e * p.N + n, k), sum);
    }
    if (p.bias) sum += bf16_bits_to_f32(p.bias[(int64_t)e * p.N + n]);
    p.out[i] = (uint16_t)pack2_bf16(p.act == MOE_ACT_GELU ? gelu16(sum) : p.act == MOE_ACT_RELU && sum < 0.0f ? 0.0f : sum, 0.0f);
}

// ---- more rows: tiles ----
//
// RH x CW wavefronts of 16 NT rows x 16 CG columns each, KS sets of them that share the contraction.  Operands go straight into LDS a slab of
// the contraction at a time, AHEAD slabs ahead, and are read through buffers that end where they end: rows behind the block's last one,
// columns behind the matrix's and what lies behind K are zeros without a branch.  Every slab takes the same path: what is requested behind
// the last one lies behind the operands' ends, and every set runs as many slabs as the longest (of zeros).  Where paths with and without
// requests met, every wait would be one for all of them.
// -- rows in bf16 --
// A slab is 128 values: 256 bytes of a token row, 64 of a weight row, of which a lane's 16 are a whole block and, widened, four fragments
// (skinny.hpp).  Scales go through registers: two stages of a 128 x 128 tile's operands are half of the LDS to the byte.
// What bounds it: on large products the matrix instructions, 8192 x 14336 x 4096 by 256 x 256 in 657 us, 1.46 PFLOP/s (a product of bf16
// by the library: 1.45; widening costs an eighth of the products' issue and hides behind the other wavefront of the SIMD).  On few rows, the way
// of a slab from memory, with one workgroup a compute unit to wait for it: 48 x 14336 x 4096 13.5 us, in which the matrix units and LDS are busy a
// fifth of the cycles each and wavefronts wait for half of theirs.  On experts of some ninety rows, weights that come from memory for one
// row block each: 6016 rows, 64 experts of 1408 x 2048, 54 us; some ten less with the weights in the memory-side cache.  Neither a third stage, nor twice
// the wavefronts, nor one that asks for weight lines ahead of the others shortens that.
template <int RH_, int NT_, int CW_, int CG_, int KS_, int AHEAD_ = 1>
struct MxTile {
    static constexpr bool ROWS4 = false;
    static constexpr int RH = RH_, NT = NT_, CW = CW_, CG = CG_, KS = KS_, AHEAD = AHEAD_;      // AHEAD: slabs that are on their way while one is multiplied
    static constexpr int STAGES = AHEAD + 1;
    static constexpr int BM = 16 * NT * RH, BN = 16 * CG * CW;
    static constexpr int SET = RH * CW;                        // wavefronts of a set
    static constexpr int THREADS = 64 * SET * KS;
    static constexpr int LOADS_A = BM / 4 / SET, LOADS_W = BN / 16 / SET;      // an instruction of a wavefront brings 4 and 16 rows
    static constexpr int RB = NT % 4 == 0 ? 4 : NT % 3 == 0 ? 3 : NT;      // groups of 16 rows whose fragments are in registers at once (twice)
    static constexpr int STAGE = BM * 256 + BN * 64;
    static constexpr int SUMS = (KS - 1) * SET * NT * CG * 1024;
    static constexpr int LDS = STAGES * KS * STAGE > SUMS ? STAGES * KS * STAGE : SUMS;
    static constexpr int BLOCKS = NT * CG >= 32 ? 1 : NT * CG >= 16 ? 2 : 160 * 1024 / LDS;      // workgroups of a compute unit
    static constexpr int WAVES_PER_SIMD = BLOCKS * THREADS / 256 < 4 ? BLOCKS * THREADS / 256 : 4;
    static_assert(SET % 4 == 0 && BM % (4 * SET) == 0 && BN % (16 * SET) == 0, "every wavefront of a set brings as many rows, in steps of 16");
    static_assert(LDS <= 160 * 1024, "LDS of a compute unit");
};

template <class T>
__global__ __launch_bounds__(T::THREADS, T::WAVES_PER_SIMD) void mx_tile_kernel(MxProduct p) {
    extern __shared__ __align__(16) unsigned char smem[];
    constexpr int NT = T::NT, CG = T::CG, RB = T::RB, KS = T::KS;
    MxTask t;
    if (!mx_task<T::BM, false>(p, T::BN, t)) return;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int ks = wave / T::SET, sw = wave % T::SET;            // set and place in it
    const int wm = sw / T::CW, wn = sw % T::CW;
    const int idx = lane & 15, q = lane >> 4;
    const int K = p.K, N = p.N;
    const uint32_t arow = 2 * (uint32_t)K, wrow = (uint32_t)K >> 1, srow = (uint32_t)K >> 5;

    // Rows into LDS: an instruction of a wavefront writes 1 KB of LDS in the order of its lanes, so what a slot holds is decided by the
    // address its lane reads: piece j of segment q (64 bytes, block q) of a row lies in slot 4 (q ^ turn) + (j ^ row) (skinny.hpp, sk_turn).
    const int arow_of = 4 * sw + q;               // (of 16: all that the permutation depends on)
    const uint32_t chunk = 4 * ((idx >> 2) ^ sk_turn(arow_of)) + ((idx ^ arow_of) & 3), a_off = (uint32_t)arow_of * arow;
    unsigned char* const stages = smem + ks * T::STAGES * T::STAGE;
    const int slabs_all = (K + 127) >> 7, slabs = (slabs_all + KS - 1) / KS, begin = ks * slabs;       // of a row; the set's
    // (a weight row's block lies in slot q ^ turn, for the same reason)
    const int c0 = t.n0 + 16 * CG * wn;
    const uint32_t w_chunk = (lane & 3) ^ sk_turn(lane >> 2), w_off = (uint32_t)(t.n0 + 16 * sw + (lane >> 2)) * wrow;
    const __amdgpu_buffer_rsrc_t a_buf = mx_buffer(t.a, (uint32_t)t.rows * arow), w_buf = mx_buffer(t.w, (uint32_t)N * wrow);
    constexpr int LOADS = T::LOADS_A + T::LOADS_W;
    auto issue = [&](int s, unsigned char* st, int first, int last) {  // requests [first, last) of slab number s of this set
        const uint32_t slab = begin + s, at = slab * 256 + 16 * chunk, w_at = slab * 64 + 16 * w_chunk;
        const uint32_t v = at < arow ? a_off + at : kBehind, vw = w_at < wrow ? w_off + w_at : kBehind;
#pragma unroll
        for (int l = first; l < last && l < LOADS; ++l) {
            const int i = l - T::LOADS_W;
            if (l < T::LOADS_W)
                __builtin_amdgcn_raw_ptr_buffer_load_lds(w_buf, (mx_lds_void*)(st + T::BM * 256 + (l * T::SET + sw) * 1024), 16, (int)(vw + l * T::SET * 16 * wrow), 0, 0, 0);
            else
                __builtin_amdgcn_raw_ptr_buffer_load_lds(a_buf, (mx_lds_void*)(st + (i * T::SET + sw) * 1024), 16, (int)(v + i * T::SET * 4 * arow), 0, 0, 0);
        }
    };
    // Scales, of UNIT slabs at a time: lane LPR r + j has eight bytes, those of slabs 2 j and 2 j + 1, of row r of the wavefront's 16 CG.
    // (The address unit takes as long over a byte a lane as over sixteen: a fetch of single bytes for every group and slab took as many of
    // its cycles as half of the operands.)
    constexpr int LPR = 4 / CG, UNIT = 2 * LPR;
    const uint32_t s_row = (uint32_t)min(c0 + lane / LPR, N - 1) * srow, s_last = (uint32_t)N * srow - 8;
    uint64_t raw, held;
    uint32_t early;                               // bytes that the fetch lies in front of what was wanted
    auto fetch_scales = [&](int s) {
        const uint32_t want = s_row + min(4 * (uint32_t)(begin + s) + 8 * (lane % LPR), srow), o = min(want, s_last);
        early = want - o;
        __builtin_memcpy(&raw, t.s + o, 8);
    };
    float scale[CG];
    auto settle_scales = [&](int s, int u) {      // of slab s + u, the unit's u-th; behind the row's end: 0
        const bool in = 4 * (uint32_t)(begin + s + u) + q < srow;
        const int mine = (int)(uint32_t)(u & 1 ? held >> 32 : held);
#pragma unroll
        for (int g = 0; g < CG; ++g) {
            const uint32_t four = (uint32_t)__builtin_amdgcn_ds_bpermute(4 * ((16 * g + idx) * LPR + u / 2), mine);
            scale[g] = mx_scale(in ? four >> (8 * q) & 255u : 0u);
        }
    };

    mx_f32x4 acc[NT][CG];
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int g = 0; g < CG; ++g) acc[i][g] = mx_f32x4{0.f, 0.f, 0.f, 0.f};

    // A slab, in blocks of RB groups of rows of a quarter (32 values a lane group): the next block's fragments are read, and the next quarter's
    // weights widened, under the products of the one before.
    constexpr int NB = NT / RB, SEQ = 4 * NB, STEP = (LOADS + SEQ - 1) / SEQ;
    auto slab = [&](const unsigned char* st, auto request) {      // request(n): in front of block n
        const unsigned char* base = st + (wm * 16 * NT + idx) * 256;
        mx_u32x4 x[2][RB], w[CG];
        mx_bf16x8 wf[2][CG];
#pragma unroll
        for (int g = 0; g < CG; ++g) w[g] = *reinterpret_cast<const mx_u32x4*>(st + T::BM * 256 + (wn * 16 * CG + 16 * g + idx) * 64 + ((q ^ sk_turn(idx)) << 4));
        auto read = [&](int n) {
            const int at = (4 * (q ^ sk_turn(idx)) + ((n / NB) ^ (idx & 3))) << 4;
#pragma unroll
            for (int i = 0; i < RB; ++i) x[n & 1][i] = *reinterpret_cast<const mx_u32x4*>(base + (n % NB * RB + i) * 16 * 256 + at);
        };
        auto widen = [&](int quarter) {
#pragma unroll
            for (int g = 0; g < CG; ++g) {
                const uint32_t codes = w[g][quarter];
                wf[quarter & 1][g] = mx_widen8(codes, scale[g]);
            }
        };
        read(0);
        widen(0);
#pragma unroll
        for (int n = 0; n < SEQ; ++n) {
            const int quarter = n / NB, ib = n % NB;
            request(n);
            if (n + 1 < SEQ) read(n + 1);
            if (ib == NB - 1 && quarter < 3) widen(quarter + 1);
#pragma unroll
            for (int i = 0; i < RB; ++i)
#pragma unroll
                for (int g = 0; g < CG; ++g)
                    acc[ib * RB + i][g] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wf[quarter & 1][g], __builtin_bit_cast(mx_bf16x8, x[n & 1][i]), acc[ib * RB + i][g], 0, 0, 0);
            __builtin_amdgcn_sched_barrier(0);
        }
    };

    constexpr int AHEAD = T::AHEAD, REQUESTS = LOADS;
    auto after = [&](unsigned char* st) { return st + T::STAGE == stages + T::STAGES * T::STAGE ? stages : st + T::STAGE; };
    unsigned char* now = stages;                  // the stage of the slab that is next; the one in front of it is filled next
    unsigned char* fill = stages + AHEAD * T::STAGE;
    if (t.rows > wm * 16 * NT) {
        fetch_scales(0);
#pragma unroll
        for (int s = 0; s < AHEAD; ++s) issue(s, stages + s * T::STAGE, 0, LOADS);
        for (int s = 0; s < slabs; s += UNIT) {
#pragma unroll
            for (int u = 0; u < UNIT; ++u) {
                if (u > 0 && s + u >= slabs) break;
                mx_meet<(AHEAD - 1) * REQUESTS>();
                if (u == 0) held = raw >> (4 * early) >> (4 * early);
                if (u == 0) fetch_scales(s + UNIT);
                settle_scales(s, u);
                slab(now, [&](int n) { issue(s + u + AHEAD, fill, STEP * n, STEP * (n + 1)); });
                now = after(now), fill = after(fill);
            }
        }
    } else {                                      // no rows for this wavefront: it brings the others theirs
        for (int s = 0; s < AHEAD; ++s) issue(s, stages + s * T::STAGE, 0, LOADS);
        for (int s = 0; s < slabs; ++s) {
            mx_meet<(AHEAD - 1) * REQUESTS>();
            issue(s + AHEAD, fill, 0, LOADS);
            fill = after(fill);
        }
    }
    if (!mx_join<KS, T::SET, NT, CG>(acc, ks, sw, smem, lane)) return;
    if constexpr (KS == 1) {
        constexpr int OWN = mx_rows_lds<NT, CG, 16, 16>();
        static_assert(T::SET * OWN <= T::LDS, "a place for every wavefront");
        mx_meet();
        mx_store_rows<NT, CG, 16, 16>(p, t, smem + sw * OWN, lane, idx, 4 * q, 16 * wm * NT, c0, acc);
    } else {
        mx_store_tile<NT, CG>(p, t, 16 * wm * NT + idx, c0 + 4 * q, acc);
    }
}

// -- rows in MXFP4 too --
// A slab is 256 values, 128 bytes of every row, both operands in LDS.  Products are 32 x 32 over 64 values: the scaled instruction of that
// shape takes 33 cycles, that of 16 x 16 over 128 values, half as much work, 31 (measured).  A lane's 16 bytes are the block of its
// row that it multiplies.  NT, CG: 32-row and 32-column blocks of a wavefront.
// 8192 x 14336 x 4096 by 256 x 256: 275 us, 3.5 PFLOP/s, where the instruction's own rate is 10 at 2.4 GHz (7.6 at the 1.8 GHz that this runs at).
// No unit bounds it: the matrix units are busy 45 % of the cycles, LDS a quarter, and wavefronts wait for 30 % of theirs -- every slab of 256 values
// ends in a wait for all requests and a meeting, with one slab under way and two wavefronts a SIMD; the way of a tile's first slab and of its results
// is a small part (workgroups that went from tile to tile gained 4 %).
template <int RH_, int NT_, int CW_, int CG_, int KS_>
struct MxTile4 {
    static constexpr bool ROWS4 = true;
    static constexpr int RH = RH_, NT = NT_, CW = CW_, CG = CG_, KS = KS_;
    static constexpr int BM = 32 * NT * RH, BN = 32 * CG * CW;
    static constexpr int SET = RH * CW;
    static constexpr int THREADS = 64 * SET * KS;
    static constexpr int LOADS_A = BM / 8 / SET, LOADS_W = BN / 8 / SET;       // an instruction of a wavefront brings 8 rows
    static constexpr int STAGE = (BM + BN) * (128 + 8);
    static constexpr int SUMS = (KS - 1) * SET * NT * CG * 4096;
    static constexpr int LDS = 2 * KS * STAGE > SUMS ? 2 * KS * STAGE : SUMS;
    static constexpr int BLOCKS = NT * CG >= 8 ? 1 : NT * CG >= 4 ? 2 : 160 * 1024 / LDS;
    static constexpr int WAVES_PER_SIMD = BLOCKS * THREADS / 256 < 1 ? 1 : BLOCKS * THREADS / 256 < 4 ? BLOCKS * THREADS / 256 : 4;
    static_assert(SET % 2 == 0 && BM % (8 * SET) == 0 && BN % (8 * SET) == 0 && BM + BN <= 64 * SET, "every wavefront of a set brings as many rows, in steps of 16, and a lane the scales of one");
    static_assert(LDS <= 160 * 1024, "LDS of a compute unit");
};
typedef float mx_f32x16 __attribute__((ext_vector_type(16)));
// The scaled instruction, 32 x 32 over 64 values; a scale is byte B of its register.
template <int B>
__device__ __forceinline__ mx_f32x16 mx_mfma32(mx_u32x4 a, uint32_t sa, mx_u32x4 b, uint32_t sb, mx_f32x16 c) {
    // (the upper half, which 4-bit operands do not have, is left open)
    const mx_i32x8 av = __builtin_bit_cast(mx_i32x8, __builtin_shufflevector(a, a, 0, 1, 2, 3, -1, -1, -1, -1));
    const mx_i32x8 bv = __builtin_bit_cast(mx_i32x8, __builtin_shufflevector(b, b, 0, 1, 2, 3, -1, -1, -1, -1));
    return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(av, bv, c, 4 /* e2m1 */, 4, B, (int)sa, B, (int)sb);
}

template <class T>
__global__ __launch_bounds__(T::THREADS, T::WAVES_PER_SIMD) void mx_tile4_kernel(MxProduct p) {
    extern __shared__ __align__(16) unsigned char smem[];
    constexpr int NT = T::NT, CG = T::CG, KS = T::KS, SET = T::SET, BM = T::BM, BN = T::BN;
    MxTask t;
    if (!mx_task<BM, true>(p, BN, t)) return;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int ks = wave / SET, sw = wave % SET;
    const int wm = sw / T::CW, wn = sw % T::CW;
    const int r32 = lane & 31, b = lane >> 5;
    const int K = p.K, N = p.N;
    const uint32_t row = (uint32_t)K >> 1, srow = (uint32_t)K >> 5;

    // Chunk c (16 bytes: a block) of a row lies in slot c ^ (row / 2): the reads below meet no bank twice in a cycle.
    const uint32_t chunk = (lane & 7) ^ (((8 * sw + (lane >> 3)) >> 1) & 7), off = (uint32_t)(8 * sw + (lane >> 3)) * row;
    unsigned char* const stages = smem + ks * 2 * T::STAGE;
    const int slabs_all = (K + 255) >> 8, slabs = (slabs_all + KS - 1) / KS;
    const __amdgpu_buffer_rsrc_t a_buf = mx_buffer(t.a, (uint32_t)t.rows * row), w_buf = mx_buffer(t.w, (uint32_t)N * row);
    // requests [first, last) of a slab's, weights first
    constexpr int LOADS = T::LOADS_A + T::LOADS_W;
    auto issue = [&](int s, int first, int last) {
        unsigned char* const st = stages + (s & 1) * T::STAGE;
        const uint32_t at = (uint32_t)(s * KS + ks) * 128 + 16 * chunk;
        const uint32_t v = at < row ? off + at : kBehind, vw = at < row ? off + at + (uint32_t)t.n0 * row : kBehind;
#pragma unroll
        for (int l = first; l < last && l < LOADS; ++l) {
            const int i = l - T::LOADS_W;
            if (l < T::LOADS_W)
                __builtin_amdgcn_raw_ptr_buffer_load_lds(w_buf, (mx_lds_void*)(st + BM * 128 + (l * SET + sw) * 1024), 16, (int)(vw + l * SET * 8 * row), 0, 0, 0);
            else
                __builtin_amdgcn_raw_ptr_buffer_load_lds(a_buf, (mx_lds_void*)(st + (i * SET + sw) * 1024), 16, (int)(v + i * SET * 8 * row), 0, 0, 0);
        }
    };
    // The scales, eight of a row a lane (token rows, then weight rows), through registers: their addresses have no alignment.
    const int my = min((int)threadIdx.x - ks * SET * 64, BM + BN - 1);
    const bool of_w = my >= BM;
    const uint8_t* const sc = of_w ? t.s : p.a_scales;
    const int64_t sc_last = (of_w ? (int64_t)N : p.M) * srow - 8;                // the last eight bytes of the whole array
    const int64_t sc_row = (of_w ? min(t.n0 + my - BM, N - 1) : t.row0 + min(my, t.rows - 1)) * (int64_t)srow;
    uint64_t raw;
    auto scales_at = [&](int s) { return sc_row + min((s * KS + ks) * 8, (int)srow); };
    auto load_scales = [&](int s) { __builtin_memcpy(&raw, sc + min(scales_at(s), sc_last), 8); };      // inside the array, which has eight
    auto store_scales = [&](int s) {              // those behind the row's end: 0
        const int64_t want = scales_at(s);
        const int early = (int)(want - min(want, sc_last)) * 4, over = (8 - min(max((int)srow - (s * KS + ks) * 8, 0), 8)) * 4;      // half of the bits, up to 32
        const uint64_t held = raw >> early >> early << over << over >> over >> over;      // without a condition: the load would move behind it, and wait there
        *reinterpret_cast<uint64_t*>(stages + (s & 1) * T::STAGE + (BM + BN) * 128 + my * 8) = held;
    };

    mx_f32x16 acc[NT][CG];
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int g = 0; g < CG; ++g)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][g][r] = 0.0f;

    // A slab in quarters of 64 values: the next quarter's fragments are read under the products of the one before.  Of a row's eight scales a
    // lane takes those of its blocks, the even or the odd ones; quarter j's is byte j.
    auto slab = [&](const unsigned char* st, auto request) {       // request(j): in front of quarter j
        const unsigned char* xb = st + (wm * 32 * NT + r32) * 128;
        const unsigned char* wb = st + (BM + wn * 32 * CG + r32) * 128;
        const uint2* scales = reinterpret_cast<const uint2*>(st + (BM + BN) * 128);
        const uint32_t pick = 0x06040200u + 0x01010101u * b;
        mx_u32x4 x[2][NT], w[2][CG];
        uint32_t xs[NT], ws[CG];
        auto read = [&](int j) {
            const int at = ((2 * j + b) ^ ((r32 >> 1) & 7)) << 4;
#pragma unroll
            for (int g = 0; g < CG; ++g) w[j & 1][g] = *reinterpret_cast<const mx_u32x4*>(wb + g * 32 * 128 + at);
#pragma unroll
            for (int i = 0; i < NT; ++i) x[j & 1][i] = *reinterpret_cast<const mx_u32x4*>(xb + i * 32 * 128 + at);
        };
        read(0);
#pragma unroll
        for (int g = 0; g < CG; ++g) {
            const uint2 v = scales[BM + wn * 32 * CG + g * 32 + r32];
            ws[g] = __builtin_amdgcn_perm(v.y, v.x, pick);
        }
#pragma unroll
        for (int i = 0; i < NT; ++i) {
            const uint2 v = scales[wm * 32 * NT + i * 32 + r32];
            xs[i] = __builtin_amdgcn_perm(v.y, v.x, pick);
        }
        auto quarter = [&](auto j_c) {
            constexpr int J = decltype(j_c)::value;
            request(J);
            if constexpr (J < 3) read(J + 1);
            __builtin_amdgcn_sched_barrier(0);    // (the compiler would put the reads last)
#pragma unroll
            for (int i = 0; i < NT; ++i)
#pragma unroll
                for (int g = 0; g < CG; ++g) acc[i][g] = mx_mfma32<J>(w[J & 1][g], ws[g], x[J & 1][i], xs[i], acc[i][g]);
            __builtin_amdgcn_sched_barrier(0);
        };
        quarter(std::integral_constant<int, 0>{});
        quarter(std::integral_constant<int, 1>{});
        quarter(std::integral_constant<int, 2>{});
        quarter(std::integral_constant<int, 3>{});
    };

    constexpr int PER = (LOADS + 2) / 3;          // requests in front of a quarter but the last
    issue(0, 0, LOADS);
    load_scales(0);
    store_scales(0);
    if (t.rows > wm * 32 * NT) {
        for (int s = 0; s < slabs; ++s) {
            mx_meet();
            load_scales(s + 1);
            slab(stages + (s & 1) * T::STAGE, [&](int j) { issue(s + 1, j * PER, j * PER + PER); });
            store_scales(s + 1);
        }
    } else {
        for (int s = 0; s < slabs; ++s) {
            mx_meet();
            issue(s + 1, 0, LOADS);
            load_scales(s + 1);
            store_scales(s + 1);
        }
    }
    // In four pieces as the 16 x 16 products leave them: 4 b .. + 3 of eight columns each, token row r32.
    mx_f32x4 sum[NT][4 * CG];
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int g = 0; g < 4 * CG; ++g) sum[i][g] = mx_f32x4{acc[i][g / 4][4 * (g % 4)], acc[i][g / 4][4 * (g % 4) + 1], acc[i][g / 4][4 * (g % 4) + 2], acc[i][g / 4][4 * (g % 4) + 3]};
    if (!mx_join<KS, SET, NT, 4 * CG>(sum, ks, sw, smem, lane)) return;
    if constexpr (KS == 1) {
        constexpr int OWN = mx_rows_lds<NT, 4 * CG, 32, 8>();
        static_assert(SET * OWN <= T::LDS, "a place for every wavefront");
        mx_meet();
        mx_store_rows<NT, 4 * CG, 32, 8>(p, t, smem + sw * OWN, lane, r32, 4 * b, wm * 32 * NT, t.n0 + wn * 32 * CG, sum);
    } else {
        mx_store_tile<NT, 4 * CG, 32, 8>(p, t, wm * 32 * NT + r32, t.n0 + wn * 32 * CG + 4 * b, sum);
    }
}

// Workgroups of a launch: blocks of BM rows (an expert's last one is its own) times column tiles, in eight equal shares.
int64_t mx_grid(const MxProduct& p, int BM, int BN) {
    const int64_t ncol = (p.N + BN - 1) / BN, blocks = p.count ? p.M / BM + p.E : (p.M + BM - 1) / BM;
    return (blocks * ncol + 7) / 8 * 8 + (p.count ? 16 : 0);
}

template <class T>
hipError_t launch_tile(const MxProduct& p, hipStream_t st) {
    void (*const kernel)(MxProduct) = [] {
        if constexpr (T::ROWS4) return mx_tile4_kernel<T>;
        else return mx_tile_kernel<T>;
    }();
    const hipError_t e = allow_lds(kernel, T::LDS);
    if (e != hipSuccess) return e;
    kernel<<<(unsigned)mx_grid(p, T::BM, T::BN), T::THREADS, T::LDS, st>>>(p);
    return hipGetLastError();
}

template <bool ROWS4, int CG>
hipError_t launch_stream_form(const MxProduct& p, int KS, bool cold, hipStream_t st) {
    const int rows = (int)(p.count ? 16 : std::min<int64_t>(p.M, 16)), lds = kStreamWaves * skinny_lds<WeightsMx<ROWS4>>(rows);
    const unsigned grid = (unsigned)mx_grid(p, 16, 16 * CG * (kStreamWaves / KS));
    const hipError_t e = cold ? allow_lds(mx_stream_kernel<ROWS4, CG, true>, lds) : allow_lds(mx_stream_kernel<ROWS4, CG, false>, lds);
    if (e != hipSuccess) return e;
    if (cold) mx_stream_kernel<ROWS4, CG, true><<<grid, 64 * kStreamWaves, lds, st>>>(p, KS, rows);
    else mx_stream_kernel<ROWS4, CG, false><<<grid, 64 * kStreamWaves, lds, st>>>(p, KS, rows);
    return hipGetLastError();
}

// How a streamer's launch is cut.  About eight wavefronts a compute unit keep the memory busy; more only start pipelines, each of which a
// chunk or two do not pay for.  14336 x 4096, us, one wavefront a contraction / 2 / 4 / 8: 12.0 / 8.3 / 8.8 / 13.3; 4096 x 14336: 32.5 / 18.4 / 12.0 / 8.8.
// Two groups of columns a wavefront halve the token rows' reads, where there are columns enough: 65536 x 4096 for 16 rows 48 -> 37.
struct StreamCut {
    bool wide;
    int KS;
    int64_t waves;
    int chunks;                 // of a wavefront, whole units
};
StreamCut stream_cut(const MxProduct& p) {
    const int64_t blocks = p.count ? std::min<int64_t>(p.E, p.M) : (p.M + 15) / 16, groups = blocks * ((p.N + 15) / 16);
    const int chunks = (p.K + 255) / 256;
    StreamCut c{groups >= 2048, 1, 0, 0};
    c.waves = c.wide ? (groups + 1) / 2 : groups;
    while (c.KS < kStreamWaves && 4 * c.KS <= chunks && c.waves * 2 <= 2048) c.KS *= 2, c.waves *= 2;
    c.chunks = ((chunks + c.KS - 1) / c.KS + kUnit - 1) / kUnit * kUnit;
    return c;
}
template <bool ROWS4>
hipError_t launch_stream(const MxProduct& p, hipStream_t st) {
    const StreamCut c = stream_cut(p);
    const bool cold = (p.count ? std::min<int64_t>(p.E, p.M) : 1) * p.N * p.K / 2 > ((int64_t)256 << 20);      // more than the memory-side cache holds
    return c.wide ? launch_stream_form<ROWS4, 2>(p, c.KS, cold, st) : launch_stream_form<ROWS4, 1>(p, c.KS, cold, st);
}

template <bool ROWS4>
hipError_t launch_small(const MxProduct& p, hipStream_t st) {
    mx_small_kernel<ROWS4><<<(unsigned)((p.M * p.N + 255) / 256), 256, 0, st>>>(p);
    return hipGetLastError();
}

// Forms: 0 the streamer, from 1 on the tiles of the tables below.  f(the tile's type, as a pointer to nothing).
template <class F>
auto with_tile(bool rows4, int form, F f) {
    if (rows4) {
        switch (form) {
            case 1: return f((MxTile4<1, 1, 2, 1, 4>*)nullptr);     // 32 x 64
            case 2: return f((MxTile4<1, 1, 2, 1, 2>*)nullptr);
            case 3: return f((MxTile4<1, 2, 2, 1, 2>*)nullptr);     // 64 x 64
            case 4: return f((MxTile4<1, 2, 4, 1, 1>*)nullptr);     // 64 x 128
            case 5: return f((MxTile4<2, 2, 2, 2, 1>*)nullptr);     // 128 x 128
            case 6: return f((MxTile4<2, 2, 4, 2, 1>*)nullptr);     // 128 x 256
            default: return f((MxTile4<4, 2, 2, 4, 1>*)nullptr);    // 256 x 256
        }
    }
    switch (form) {
        case 1: return f((MxTile<1, 1, 4, 1, 2, 4>*)nullptr);       // 16 x 64
        case 2: return f((MxTile<1, 2, 4, 1, 2, 2>*)nullptr);       // 32 x 64
        case 3: return f((MxTile<1, 3, 4, 1, 2, 3>*)nullptr);       // 48 x 64
        case 4: return f((MxTile<1, 4, 4, 1, 2>*)nullptr);          // 64 x 64
        case 5: return f((MxTile<1, 4, 4, 2, 1>*)nullptr);          // 64 x 128
        case 6: return f((MxTile<1, 6, 4, 2, 1>*)nullptr);          // 96 x 128
        case 7: return f((MxTile<1, 8, 4, 2, 1>*)nullptr);          // 128 x 128
        default: return f((MxTile<2, 8, 4, 4, 1>*)nullptr);         // 256 x 256
    }
}

// What a tile costs, in us: a launch of its form; a slab of the contraction where a compute unit has one tile; the same for every further
// tile of the unit.  Fitted to products of 17 to 6000 rows, 5 to 800 us, dense and of experts, each with every form that was near: over 240 of
// them the choice by these is 1.2 % behind the best of the forms on average, over 68 more of experts with 20 to 130 rows each, evenly and not,
// 3.3 %; 38 % at worst (35 rows for each of 8 experts).
struct TileCost {
    int rows, columns;
    float launch, slab, more;
};
constexpr TileCost kTiles16[] = {{}, {16, 64, 3.2f, 0.158f, 0.187f}, {32, 64, 3.0f, 0.208f, 0.241f}, {48, 64, 3.3f, 0.25f, 0.409f}, {64, 64, 3.1f, 0.343f, 0.352f},
                                 {64, 128, 3.1f, 0.621f, 0.482f}, {96, 128, 2.8f, 0.805f, 0.684f}, {128, 128, 4.4f, 0.822f, 0.836f}, {256, 256, 10.4f, 2.17f, 2.11f}};
constexpr TileCost kTiles4[] = {{}, {32, 64, 4.3f, 0.179f, 0.524f}, {32, 64, 3.2f, 0.231f, 0.281f}, {64, 64, 3.3f, 0.284f, 0.449f}, {64, 128, 2.6f, 0.538f, 0.559f},
                                {128, 128, 3.3f, 0.682f, 0.862f}, {128, 256, 3.8f, 0.963f, 1.70f}, {256, 256, 4.9f, 1.39f, 2.58f}};

// The form that should take least; 0: the streamer.  Of experts' rows the host knows how many there are, not whose: a block an expert where the
// mean is small for it, else half a block more than the mean fills.
int product_form(const MxProduct& p) {
    const bool rows4 = p.a_scales != nullptr;
    const int64_t experts = p.count ? std::min<int64_t>(p.E, p.M) : 1;
    const double each = (double)p.M / experts;
    // (a chunk of a wavefront, with one or two groups of columns; and what its token rows add)
    const StreamCut c = stream_cut(p);
    const double rows = std::min(each, 16.0);
    auto row_blocks = [&](int rows) { return !p.count ? (double)((p.M + rows - 1) / rows) : each > 0.6 * rows ? (double)p.M / rows + 0.5 * experts : (double)experts; };
    const double rounds = std::max(1.0, c.waves / 2048.0) * (p.count ? row_blocks(16) / experts : 1.0);
    double best = 3.8 + (rows4 ? 0.03 : 0.2) * rows + c.chunks * rounds * ((c.wide ? 1.3 : 0.5) + (rows4 ? 0.003 : 0.017) * rows);
    if (p.count && each > 16) best = 1e30;               // a row block an expert, at most
    int form = 0;
    // (whose cost below is memory's.  Rows in MXFP4, without / with it, us, weights of several calls in turn: 64 experts of 1408 x 2048, 88 MiB, one row
    // each 21.9 / 27.9, 40 rows 24.8 / 31.8; 4 of 4096 x 14336, 112 MiB, one row 27.9 / 25.3; 64 of 2048 x 2048, 128 MiB, 34.7 / 31.0, 80 rows 50.9 / 40.5; 16 of
    // 4096 x 4096 35.1 / 29.0; 8 of 4096 x 14336, 224 MiB, 45.9 / 47.7, 80 rows 91.5 / 83.9; 64 of 2048 x 7168, 448 MiB, 104.9 / 82.1, 80 rows 157.6 / 143.1.
    // Rows in bf16 hardly ever get another form by it.)
    const bool cold = experts * p.N * p.K / 2 > ((int64_t)96 << 20);
    const int forms = rows4 ? (int)(sizeof kTiles4 / sizeof kTiles4[0]) : (int)(sizeof kTiles16 / sizeof kTiles16[0]);
    for (int f = 1; f < forms; ++f) {
        const TileCost& t = rows4 ? kTiles4[f] : kTiles16[f];
        const double tiles = std::ceil(row_blocks(t.rows) * ((p.N + t.columns - 1) / t.columns) / 256.0);      // of the compute unit that has most
        const int slabs = rows4 ? (p.K + 255) / 256 : (p.K + 127) / 128;
        // (and of weights that no cache holds a compute unit is brought some 24 KB a us)
        const double cost = std::max(t.launch + slabs * (t.slab + t.more * (tiles - 1)), cold ? 2.4 + tiles * t.columns * (p.K * 17.0 / 32) / 24e3 : 0.0);
        if (cost < best) best = cost, form = f;
    }
    return form;
}

constexpr int kSmallForm = -1;
bool is_small(const MxProduct& p) { return (int64_t)p.N * p.K < 256 || (p.a_scales && p.M * p.K < 256); }      // eight scales are fetched at a time
int64_t product_workgroups(const MxProduct& p, int form) {
    if (form == kSmallForm) return (p.M * p.N + 255) / 256;
    if (form == 0) return mx_grid(p, 16, 16);               // its narrowest
    const TileCost& t = p.a_scales ? kTiles4[form] : kTiles16[form];
    return mx_grid(p, t.rows, t.columns);
}

}  // namespace

hipError_t launch_product_mxfp4(const MxProduct& p, int form, hipStream_t st) {
    if (p.M == 0) return hipSuccess;
    const bool rows4 = p.a_scales != nullptr;
    if (form == kSmallForm) return rows4 ? launch_small<true>(p, st) : launch_small<false>(p, st);
    if (form == 0) return rows4 ? launch_stream<true>(p, st) : launch_stream<false>(p, st);
    return with_tile(rows4, form, [&](auto* t) { return launch_tile<std::remove_pointer_t<decltype(t)>>(p, st); });
}

// What the kernels read and write at a time, their 32-bit offsets and the launches' sizes; and the kernel that the product takes.
int check_product_mxfp4(const MxProduct& p, int a_dtype, int* form) {
    auto aligned = [](const void* a) { return (uintptr_t)a % 16 == 0; };
    if (p.M < 0 || p.N < 1 || p.K < kMxBlock || p.K % kMxBlock || !p.w || !p.s) return MOE_ERR_BAD_ARGUMENT;
    if (p.act != MOE_ACT_RELU && p.act != MOE_ACT_GELU && p.act != MOE_ACT_NONE) return MOE_ERR_BAD_ARGUMENT;
    if (a_dtype != MOE_DTYPE_BF16 && a_dtype != MOE_DTYPE_MXFP4) return MOE_ERR_UNSUPPORTED;
    if (p.M > 0 && (!p.a || !p.out || (a_dtype == MOE_DTYPE_MXFP4) != (p.a_scales != nullptr))) return MOE_ERR_BAD_ARGUMENT;
    if (!aligned(p.a) || !aligned(p.w) || !aligned(p.out) || (uintptr_t)p.bias % 2) return MOE_ERR_BAD_ARGUMENT;
    if (p.K > (1 << 20) || (int64_t)p.N * (p.K / 2) >= kBufferBytes || p.M > INT32_MAX) return MOE_ERR_UNSUPPORTED;
    *form = is_small(p) ? kSmallForm : product_form(p);
    return product_workgroups(p, *form) < ((int64_t)1 << 22) ? MOE_OK : MOE_ERR_UNSUPPORTED;      // 1024 threads each: 2^32
}

}  // namespace moe355

using namespace moe355;

extern "C" int moe_gemm_mxfp4(const void* a, const uint8_t* a_scales, int32_t a_dtype, const void* w, const uint8_t* w_scales, const void* bias, void* out,
                              int64_t M, int64_t N, int64_t K, int32_t act, void* stream) {
    if (M < 0 || N < 1 || K < 1) return MOE_ERR_BAD_ARGUMENT;
    if (N > INT32_MAX / 2 || K > INT32_MAX / 2) return MOE_ERR_UNSUPPORTED;
    const MxProduct p{a, a_scales, w, w_scales, (const uint16_t*)bias, nullptr, nullptr, (uint16_t*)out, M, (int)N, (int)K, 1, act};
    int form;
    const int rc = check_product_mxfp4(p, a_dtype, &form);
    if (rc) return rc;
    return launch_product_mxfp4(p, form, (hipStream_t)stream) == hipSuccess ? MOE_OK : MOE_ERR_HIP;
}

extern "C" int moe_gemm_mxfp4_plan(int64_t M, int64_t N, int64_t K, int32_t experts, int32_t a_dtype, int32_t* rows, int32_t* columns, int32_t* parts) {
    if (M < 1 || N < 1 || K < 1 || experts < 0 || experts > kMaxExperts || !rows || !columns || !parts) return MOE_ERR_BAD_ARGUMENT;
    if (N > INT32_MAX / 2 || K > INT32_MAX / 2) return MOE_ERR_UNSUPPORTED;
    // an operand that is there, as far as the choice looks at it
    alignas(16) static const uint8_t some[16] = {};
    alignas(16) static uint16_t result[8];
    const int32_t* const table = experts ? reinterpret_cast<const int32_t*>(some) : nullptr;
    const MxProduct p{some, a_dtype == MOE_DTYPE_MXFP4 ? some : nullptr, some, some, nullptr, table, table, result, M, (int)N, (int)K, experts ? experts : 1, MOE_ACT_NONE};
    int form;
    const int rc = check_product_mxfp4(p, a_dtype, &form);
    if (rc) return rc;
    if (form == kSmallForm) {
        *rows = *columns = *parts = 1;
    } else if (form == 0) {
        const StreamCut c = stream_cut(p);
        *rows = 16, *columns = c.wide ? 32 : 16, *parts = c.KS;
    } else {
        with_tile(a_dtype == MOE_DTYPE_MXFP4, form, [&](auto* t) {
            typedef std::remove_pointer_t<decltype(t)> T;
            *rows = T::BM, *columns = T::BN, *parts = T::KS;
        });
    }
    return MOE_OK;
}
