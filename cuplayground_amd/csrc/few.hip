// A whole layer for a few tokens (at most 16): router, selection, expert FFN and combine in two launches, or three where the router is large.
//
// With one to sixteen tokens the layer is its weights, once: those of the experts that are hit, 0.1 to 2 GB in 16 bits or MXFP4, and
// nothing else is worth a launch of its own.  What the general path takes six launches for (logits, selection, slots and task tables, two
// projections, combine) is here
//   few_up    every workgroup finds out for itself which experts are hit and by whom -- the logits where the router is small (else
//             few_logits has left them), the selection a token a wavefront, a mask of tokens an expert -- and streams gate and up rows;
//   few_down  a workgroup owns 16 output columns and goes through all experts that are hit: with the tokens as the columns of the matrix
//             instruction's result, an expert's share of the combine is a multiply-add on the accumulators, in fp32, and out is written
//             once.  No expert's output row is ever rounded or stored.  The intermediate is rounded to the activations' 16 bits, for it is
//             an operand of 16-bit matrix instructions: distance from 64 bits 0.0024 in bf16, 0.0017 of it the output's own rounding (0.0029 on
//             the general path, which rounds the experts' rows too).
// Weights stream as in skinny.hpp.  The router's sums and selection are those of the general path to the bit (the fixed order of 64
// partial sums; topk.hpp), and so are slots, drops and packed rows: the intermediate lies where that path would put it.
//
// Bound by memory.  us in few_logits + few_up + few_down, one token of 4096 x 14336, 8 experts, 2 chosen, SwiGLU, MXFP4 (187 MB): 30 + 17; 16 tokens
// of 7168 x 2048, 256 experts, 8 chosen (about 2.4 GB): 9 + 290 + 154, 5.3 TB/s; 4 tokens of 2048 x 1408, 64 experts, 6 chosen, bf16 (about 0.36 GB):
// 5 + 57 + 27.
#include "act_deriv.hpp"
#include "skinny.hpp"
#include "topk.hpp"

namespace moe355 {
namespace {

constexpr int kFewThreads = 512, kFewWaves = 8;
constexpr int kFewPairs = kFewTokens * kMaxTopK;
static_assert(kFewPairs <= 256, "packed rows in a byte");

// What every workgroup knows of the routing.
struct FewPlan {
    float w[kFewPairs];                // [S, k] gate weights
    int32_t idx[kFewPairs];            // [S, k] experts
    uint32_t mask[kMaxExperts];        // tokens an expert keeps
    int16_t base[kMaxExperts];         // packed row of its first one
    int16_t list[kFewPairs];           // experts that are hit, ascending
    float row_w[kFewPairs];            // gate weight of a packed row
    uint8_t row_t[kFewPairs];          // its token
    int32_t part[3][kFewWaves];        // of 64 experts each: rows, experts that are hit, rows of the one that has most
    int32_t hit, kept, most;           // experts that are hit, rows, rows of the expert that has most
};

template <class ET>
__device__ __forceinline__ float few_widen(uint16_t v) {
    if constexpr (std::is_same<ET, f16_s>::value) return (float)__builtin_bit_cast(_Float16, v);
    else return bf16_bits_to_f32(v);
}
template <class ET>
__device__ __forceinline__ uint32_t few_pack(float lo, float hi) {
    if constexpr (std::is_same<ET, f16_s>::value) {
        const mx_f32x2 v = {lo, hi};
        return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, mx_f16x2));
    } else {
        return pack2_bf16(lo, hi);
    }
}

// Four neighbouring values of a bias, or zeros; one load.
template <class ET>
__device__ __forceinline__ mx_f32x4 few_bias(const uint16_t* b, int col) {
    uint16_t raw[4] = {0, 0, 0, 0};
    if (b) __builtin_memcpy(raw, b + col, 8);
    return mx_f32x4{few_widen<ET>(raw[0]), few_widen<ET>(raw[1]), few_widen<ET>(raw[2]), few_widen<ET>(raw[3])};
}
// Four neighbouring values of an expert's bias for the unit that is multiplied, fetched with the unit's scales: a load where the sums are done
// would be waited for behind all weights that are on their way by then.  A bias that is not there is a buffer of no bytes: zeros.
template <class ET>
struct FewBias {
    typedef uint32_t Pair __attribute__((ext_vector_type(2)));
    Pair now, then;
    __amdgpu_buffer_rsrc_t buf;
    __device__ __forceinline__ void aim(const void* b, int64_t at, int n) {
        buf = mx_buffer(b ? static_cast<const uint16_t*>(b) + at : nullptr, b ? 2u * (uint32_t)n : 0u);
    }
    __device__ __forceinline__ void next(int col) {
        now = then;
        then = __builtin_bit_cast(Pair, __builtin_amdgcn_raw_buffer_load_b64(buf, 2 * col, 0, 0));
    }
    __device__ __forceinline__ mx_f32x4 get() const {
        return mx_f32x4{few_widen<ET>((uint16_t)now[0]), few_widen<ET>((uint16_t)(now[0] >> 16)), few_widen<ET>((uint16_t)now[1]), few_widen<ET>((uint16_t)(now[1] >> 16))};
    }
};

// Logits of one expert for tokens t0 .. t0 + n - 1 (n <= TT) by a wavefront: lane p adds up, in ascending k, the products of every k with
// (k / 8) % 64 == p, one multiply-add each; the partial sums are folded pairwise.  logits[t] at out[t * stride].
template <class ET, int TT>
__device__ __forceinline__ void few_logits(const uint16_t* __restrict__ x, const uint16_t* __restrict__ g, const float* bias, int e, int t0, int n, int H, float* out, int stride, int lane) {
    float p[TT];
#pragma unroll
    for (int t = 0; t < TT; ++t) p[t] = 0.0f;
    union Eight { mx_u32x4 v; uint16_t s[8]; };
    auto load = [&](const uint16_t* row, int k) {
        Eight r;
        r.v = *reinterpret_cast<const mx_u32x4*>(row + k);
        return r;
    };
    auto add = [&](const Eight& xv, const Eight& gv, float& sum) {
#pragma unroll
        for (int i = 0; i < 8; ++i) sum = __builtin_fmaf(few_widen<ET>(xv.s[i]), few_widen<ET>(gv.s[i]), sum);
    };
    const uint16_t* const ge = g + (int64_t)e * H;
    int k = 8 * lane;
    constexpr int U = 4;                       // steps that are fetched together: one trip to memory for them
    for (int k0 = 0; k0 + 512 * U <= H; k0 += 512 * U, k += 512 * U) {
        Eight gv[U], xv[U][TT];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            gv[u] = load(ge, k + 512 * u);
#pragma unroll
            for (int t = 0; t < TT; ++t) xv[u][t] = load(x + (int64_t)(t0 + min(t, n - 1)) * H, k + 512 * u);
        }
        __builtin_amdgcn_sched_barrier(0);     // (or each would move to its use, and be waited for by itself)
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int t = 0; t < TT; ++t) add(xv[u][t], gv[u], p[t]);
    }
    for (; k < H; k += 512) {
        const Eight gv = load(ge, k);
#pragma unroll
        for (int t = 0; t < TT; ++t) add(load(x + (int64_t)(t0 + min(t, n - 1)) * H, k), gv, p[t]);
    }
#pragma unroll
    for (int t = 0; t < TT; ++t) {
        float v = p[t];
#pragma unroll
        for (int off = 32; off >= 1; off >>= 1) v = v + __shfl_xor(v, off, kWave);
        if (bias) v = v + bias[e];
        if (lane == 0 && t < n) out[(t0 + t) * stride] = v;
    }
}

constexpr int kLogitTokens = 4;
template <class ET>
__global__ __launch_bounds__(256) void few_logits_kernel(FewArgs a) {
    const int lane = threadIdx.x & 63, wave = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int groups = (a.S + kLogitTokens - 1) / kLogitTokens;
    const int e = wave / groups, t0 = (wave - e * groups) * kLogitTokens;
    if (e >= a.E) return;
    few_logits<ET, kLogitTokens>((const uint16_t*)a.x, (const uint16_t*)a.gate_w, a.gate_bias, e, t0, min(kLogitTokens, a.S - t0), a.H, a.logits + e, a.E, lane);
}

// From the selection in p.w / p.idx (behind a barrier): masks, packed rows, the list.  Called by the whole workgroup.
__device__ __forceinline__ void few_plan(FewPlan& p, const FewArgs& a) {
    const int tid = threadIdx.x, lane = tid & 63, P = a.S * a.k;
    if (tid < a.E) p.mask[tid] = 0;
    __syncthreads();
    if (tid < P && (unsigned)p.idx[tid] < (unsigned)a.E) atomicOr(&p.mask[p.idx[tid]], 1u << (tid / a.k));     // a token names an expert once
    __syncthreads();
    static_assert(kMaxExperts <= kWave * kFewWaves, "64 experts a wavefront");
    const int wave = tid >> 6, e = tid;
    uint32_t m = e < a.E ? p.mask[e] : 0u;
    if (a.drop)                                        // the first `capacity` tokens stay
        while (__popc(m) > a.capacity) m &= ~(1u << (31 - __clz(m)));
    const int n = __popc(m);
    int inc = n, most = n;
#pragma unroll
    for (int off = 1; off < kWave; off <<= 1) {
        const int o = __shfl_up(inc, off, kWave);
        if (lane >= off) inc += o;
        most = max(most, __shfl_xor(most, off, kWave));
    }
    const unsigned long long any = __ballot(n > 0);
    if (lane == kWave - 1) p.part[0][wave] = inc, p.part[1][wave] = __popcll(any), p.part[2][wave] = most;
    __syncthreads();
    int rows = 0, hit = 0, all_rows = 0, all_hit = 0, all_most = 0;
#pragma unroll
    for (int w = 0; w < kFewWaves; ++w) {
        if (w < wave) rows += p.part[0][w], hit += p.part[1][w];
        all_rows += p.part[0][w], all_hit += p.part[1][w], all_most = max(all_most, p.part[2][w]);
    }
    if (e < a.E) {
        p.mask[e] = m;
        p.base[e] = (int16_t)(rows + inc - n);
    }
    if (n > 0) p.list[hit + __popcll(any & ((1ull << lane) - 1ull))] = (int16_t)e;
    if (tid == 0) p.hit = all_hit, p.kept = all_rows, p.most = all_most;
    __syncthreads();
    if (tid < P) {
        const int e = p.idx[tid], t = tid / a.k;
        if ((unsigned)e < (unsigned)a.E && ((p.mask[e] >> t) & 1u)) {
            const int row = p.base[e] + __popc(p.mask[e] & ((1u << t) - 1u));
            p.row_w[row] = p.w[tid];
            p.row_t[row] = (uint8_t)t;
        }
    }
    __syncthreads();
}

// The routing result as the general path hands it out; by one workgroup.
__device__ __forceinline__ void few_report(const FewPlan& p, const FewArgs& a) {
    const int tid = threadIdx.x, P = a.S * a.k;
    if (tid < P) {
        const int e = p.idx[tid], t = tid / a.k;
        const bool in = (unsigned)e < (unsigned)a.E && ((p.mask[e] >> t) & 1u);
        const int slot = in ? __popc(p.mask[e] & ((1u << t) - 1u)) : -1;
        a.topk_idx[tid] = e;
        a.topk_w[tid] = p.w[tid];
        if (a.r.topk_idx) a.r.topk_idx[tid] = e;
        if (a.r.topk_w) a.r.topk_w[tid] = p.w[tid];
        if (a.r.slot) a.r.slot[tid] = slot;
        if (a.r.token_indices) {
            if (in) a.r.token_indices[p.base[e] + slot] = t;
            if (tid >= p.kept) a.r.token_indices[tid] = -1;
        }
    }
    for (int e = tid; e < a.E; e += blockDim.x) {
        if (a.r.expert_count) a.r.expert_count[e] = __popc(p.mask[e]);
        if (a.r.expert_offset) a.r.expert_offset[e] = p.base[e];
    }
}

// The up (and gate) projection: a task is 16 columns of both matrices of an expert, or 32 of the one, over the whole of H, by KS wavefronts.
// With KS = 1 a wavefront goes from task to task without a pause: the next one's weights are requested under the last ones' products.
//
// Of LDS a wavefront has kRowLds for token rows, so that two workgroups have room on a compute unit; where an expert has more rows than that,
// half of the wavefronts work, with the others' room.  (With KS > 1, where there is little to do, as much as S rows may take.)
constexpr int kRowLds = 8192;
template <class W, class ET, bool GATED, bool COLD>
__global__ __launch_bounds__(kFewThreads, 4) void few_up_kernel(FewArgs a, int KS) {
    extern __shared__ __align__(16) unsigned char smem[];
    __shared__ FewPlan plan;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const float* logits = a.logits;
    if (a.fold) {
        float* own = reinterpret_cast<float*>(smem);
        for (int e = wave; e < a.E; e += kFewWaves)
            if (a.S == 1) few_logits<ET, 1>((const uint16_t*)a.x, (const uint16_t*)a.gate_w, a.gate_bias, e, 0, 1, a.H, own + e, a.E, lane);
            else for (int t0 = 0; t0 < a.S; t0 += kLogitTokens)
                few_logits<ET, kLogitTokens>((const uint16_t*)a.x, (const uint16_t*)a.gate_w, a.gate_bias, e, t0, min(kLogitTokens, a.S - t0), a.H, own + e, a.E, lane);
        logits = own;
        __syncthreads();
    }
    for (int t = wave; t < a.S; t += kFewWaves) {
        if (a.E <= 64) topk_one_token<1>(logits + (int64_t)t * a.E, t, a.E, a.k, a.gate_fn, a.norm, plan.idx, plan.w, lane);
        else if (a.E <= 256) topk_one_token<4>(logits + (int64_t)t * a.E, t, a.E, a.k, a.gate_fn, a.norm, plan.idx, plan.w, lane);
        else topk_one_token<8>(logits + (int64_t)t * a.E, t, a.E, a.k, a.gate_fn, a.norm, plan.idx, plan.w, lane);
    }
    __syncthreads();
    few_plan(plan, a);
    if (blockIdx.x == 0) {
        few_report(plan, a);
        if (a.parts > 1)
            for (int i = threadIdx.x; i < a.H / 16; i += kFewThreads) a.arrived[i] = 0;      // for few_down
    }

    constexpr int G = 2, COLS = GATED ? 16 : 32;
    const int H = a.H, I = a.I, chunks = (H + W::K - 1) / W::K;
    const int ncol = I / COLS, tasks = plan.hit * ncol;
    const bool half = KS == 1 && skinny_lds<W>(plan.most) > kRowLds;
    const int waves = half ? kFewWaves / 2 : kFewWaves;
    const int ks = wave % KS, first = blockIdx.x * (waves / KS) + wave / KS, stride = gridDim.x * (waves / KS);
    const int share = (chunks + KS - 1) / KS, begin = min(ks * share, chunks), end = min(begin + share, chunks);      // chunks of a task that are this wavefront's
    const int units = (end - begin + kUnit - 1) / kUnit;
    const int idx = lane & 15, q = lane >> 4;
    const int64_t mat = W::row_bytes((int64_t)H * I), smat = (int64_t)I * (H >> 5);

    // (with KS > 1 the launch has a set of wavefronts for every task there can be)
    const int mytasks = wave < waves && first < tasks ? (KS > 1 ? 1 : (tasks - 1 - first) / stride + 1) : 0;
    Skinny<W, G, COLD> st;
    const int lds = half ? 2 * kRowLds : KS == 1 ? min(skinny_lds<W>(a.S), kRowLds) : skinny_lds<W>(a.S);
    st.init(smem + wave * lds, plan.most, H);
    st.x_buf = mx_buffer(a.x, (uint32_t)a.S * st.x_row);
    int task = first, unit = 0;          // the next unit to be fetched
    auto next = [&](int u) {
        if (u == mytasks * units) {
            st.chunk_end = 0;
            return;
        }
        if (unit == 0) {
            const int j = task / ncol, n0 = (task - j * ncol) * COLS;
            const int e = __builtin_amdgcn_readfirstlane(plan.list[j]), base = __builtin_amdgcn_readfirstlane(plan.base[e]);
#pragma unroll
            for (int g = 0; g < G; ++g) {
                st.w_buf[g] = mx_buffer(static_cast<const char*>(GATED && g ? a.w_gate : a.w_up) + e * mat, (uint32_t)mat);
                if constexpr (W::MX) st.s_at[g] = (GATED && g ? a.s_gate : a.s_up) + e * smat;
            }
            st.aim_weights(n0, I, GATED ? 0 : 16);
            st.aim_tokens(__builtin_amdgcn_readfirstlane(__popc(plan.mask[e])), [&](int r) { return plan.row_t[base + r]; });
        }
        st.chunk0 = begin + kUnit * unit;
        st.chunk_end = end;
        if (++unit == units) unit = 0, task += stride;
    };
    mx_f32x4 acc[G] = {};
    auto store = [&](int task) {
        const int j = task / ncol, n0 = (task - j * ncol) * COLS;
        const int e = __builtin_amdgcn_readfirstlane(plan.list[j]);
        if (idx >= __popc(plan.mask[e])) return;
        uint16_t* h = (uint16_t*)a.h + (int64_t)(plan.base[e] + idx) * I;
        // (fetched here: kept from the task's beginning they would cost the registers of a second workgroup)
        const uint16_t* bu = a.b_up ? (const uint16_t*)a.b_up + (int64_t)e * I : nullptr;
        const uint16_t* bg = a.b_gate ? (const uint16_t*)a.b_gate + (int64_t)e * I : nullptr;
        auto put = [&](int col, float (&v)[4]) {
            *reinterpret_cast<uint2*>(h + col) = uint2{few_pack<ET>(v[0], v[1]), few_pack<ET>(v[2], v[3])};
        };
        if constexpr (GATED) {
            const int col = n0 + 4 * q;
            const mx_f32x4 up = acc[0] + few_bias<ET>(bu, col), gate = acc[1] + few_bias<ET>(bg, col);
            float v[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) v[r] = silu16(gate[r]) * up[r];
            put(col, v);
        } else {
#pragma unroll
            for (int g = 0; g < G; ++g) {
                const int col = n0 + 16 * g + 4 * q;
                const mx_f32x4 up = acc[g] + few_bias<ET>(bu, col);
                float v[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) v[r] = a.act == MOE_ACT_GELU ? gelu16(up[r]) : (up[r] < 0.0f ? 0.0f : up[r]);
                put(col, v);
            }
        }
    };
    int done_task = first, done_unit = 0;
    st.run(mytasks * units, acc, next, [&](int) {
        if (KS > 1 || ++done_unit < units) return;
        store(done_task);
#pragma unroll
        for (int g = 0; g < G; ++g) acc[g] = mx_f32x4{0.f, 0.f, 0.f, 0.f};
        done_unit = 0, done_task += stride;
    });
    if (KS > 1) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");           // the rows' place is the sums' now
        __syncthreads();
        const bool holds = skinny_join<G>(acc, ks, KS, reinterpret_cast<mx_f32x4*>(smem) + wave / KS * (KS - 1) * G * 64, lane);
        if (holds && mytasks) store(first);
    }
}

// The down projection and the combine: a workgroup owns 16 columns of out; its wavefronts share the (expert, chunk of I) pairs, as many
// each.  LDS as for the up projection: 7168 columns, 448 workgroups, are one round instead of two.
template <class W, class ET, bool COLD>
__global__ __launch_bounds__(kFewThreads, 4) void few_down_kernel(FewArgs a) {
    constexpr int G = 1;
    extern __shared__ __align__(16) unsigned char smem[];
    __shared__ FewPlan plan;
    __shared__ mx_f32x4 red[(kFewWaves - 1) * G * 64];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    if (tid < a.S * a.k) {
        plan.idx[tid] = a.topk_idx[tid];
        plan.w[tid] = a.topk_w[tid];
    }
    __syncthreads();
    few_plan(plan, a);

    const int H = a.H, I = a.I, chunks = (I + W::K - 1) / W::K;      // of an expert
    const int group = (int)blockIdx.x / a.parts, part = (int)blockIdx.x - group * a.parts, n0 = group * 16 * G;
    const int idx = lane & 15, q = lane >> 4;
    const int64_t mat = W::row_bytes((int64_t)H * I), smat = (int64_t)H * (I >> 5);
    const bool half = skinny_lds<W>(plan.most) > kRowLds;
    const int waves = half ? kFewWaves / 2 : kFewWaves;
    const int64_t all = (int64_t)plan.hit * chunks;
    const int64_t shares = (int64_t)waves * a.parts;
    const int first = part * waves + min(wave, waves), begin = (int)(all * first / shares), end = wave < waves ? (int)(all * (first + 1) / shares) : begin;
    int j = begin / chunks, c = begin - j * chunks, next_j = j, next_c = c;
    // units: of the first expert's rest, of whole experts, of the last one's part
    const int head = min(end - begin, chunks - c), rest = end - begin - head;
    auto units_of = [](int n) { return (n + kUnit - 1) / kUnit; };
    const int units = units_of(head) + rest / chunks * units_of(chunks) + units_of(rest % chunks);
    Skinny<W, G, COLD> st;
    const int own = half ? 2 * kRowLds : min(skinny_lds<W>(a.S), kRowLds);
    st.init(smem + wave * own, plan.most, I);
    st.x_buf = mx_buffer(a.h, (uint32_t)plan.kept * st.x_row);
    st.aim_weights(n0, H, 16);
    bool aimed = false;
    FewBias<ET> bias[G] = {};
    auto next = [&](int u) {
        const bool live = u < units;
        if (live && (!aimed || next_c == 0)) {
            const int e = __builtin_amdgcn_readfirstlane(plan.list[next_j]), base = __builtin_amdgcn_readfirstlane(plan.base[e]);
#pragma unroll
            for (int g = 0; g < G; ++g) {
                st.w_buf[g] = mx_buffer(static_cast<const char*>(a.w_down) + e * mat, (uint32_t)mat);
                if constexpr (W::MX) st.s_at[g] = a.s_down + e * smat;
                bias[g].aim(a.b_down, (int64_t)e * H, H);
            }
            st.aim_tokens(__builtin_amdgcn_readfirstlane(__popc(plan.mask[e])), [&](int r) { return base + r; });
            aimed = true;
        }
        st.chunk0 = next_c;
        st.chunk_end = live ? min(chunks, end - next_j * chunks) : 0;
        next_c += kUnit;
        if (next_c >= chunks) next_c = 0, ++next_j;
#pragma unroll
        for (int g = 0; g < G; ++g) bias[g].next(n0 + 16 * g + 4 * q);
    };
    mx_f32x4 out[1][G] = {}, acc[G] = {};
    bool whole = c == 0;                 // the expert's first chunk is among them
    st.run(units, acc, next, [&](int) {
        c += kUnit;
        if (c < min(chunks, end - j * chunks)) return;
        // the columns are the expert's rows in order: lane (row, q) hands its sums to the lane of the row's token
        const int e = __builtin_amdgcn_readfirstlane(plan.list[j]);
        const uint32_t m = plan.mask[e];
        const bool in = (m >> idx) & 1u;
        const int r = __popc(m & ((1u << idx) - 1u)), from = 4 * ((lane & 48) + (in ? r : 0));
        const float w = in ? plan.row_w[plan.base[e] + r] : 0.0f;
#pragma unroll
        for (int g = 0; g < G; ++g) {
            const mx_f32x4 first = whole ? bias[g].get() : mx_f32x4{0.f, 0.f, 0.f, 0.f};      // the bias goes with the first chunk
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float y = __uint_as_float(__builtin_amdgcn_ds_bpermute(from, (int)__float_as_uint(acc[g][i]))) + first[i];
                if (in) out[0][g][i] = __builtin_fmaf(w, y, out[0][g][i]);      // a token that is not the expert's: not even a NaN of it
            }
        }
#pragma unroll
        for (int g = 0; g < G; ++g) acc[g] = mx_f32x4{0.f, 0.f, 0.f, 0.f};
        c = 0, ++j, whole = true;
    });
    if (!skinny_join<G>(out[0], wave, kFewWaves, red, lane)) return;
    if (a.parts > 1) {
        // The sums of workgroups that share these columns, wherever they run: written through, counted, and added up in their order by the
        // last that comes.
        static_assert(G == 1, "a part is 16 columns of 16 tokens");
        uint64_t* const parts = reinterpret_cast<uint64_t*>(a.part) + ((int64_t)group * a.parts * 64 + lane) * 2;
        union { mx_f32x4 v; uint64_t w[2]; } s;
        s.v = out[0][0];
#pragma unroll
        for (int i = 0; i < 2; ++i) __hip_atomic_store(parts + part * 128 + i, s.w[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        int before = 0;
        if (lane == 0) before = __hip_atomic_fetch_add(a.arrived + group, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        if (__builtin_amdgcn_readfirstlane(before) != a.parts - 1) return;
        asm volatile("" ::: "memory");
        out[0][0] = mx_f32x4{0.f, 0.f, 0.f, 0.f};
        for (int z = 0; z < a.parts; ++z) {
#pragma unroll
            for (int i = 0; i < 2; ++i) s.w[i] = __hip_atomic_load(parts + z * 128 + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            out[0][0] += s.v;
        }
    }
    if (idx >= a.S) return;
#pragma unroll
    for (int g = 0; g < G; ++g)
        *reinterpret_cast<uint2*>((uint16_t*)a.out + (int64_t)idx * H + n0 + 16 * g + 4 * q) = uint2{few_pack<ET>(out[0][g][0], out[0][g][1]), few_pack<ET>(out[0][g][2], out[0][g][3])};
}

// Bytes of weights for 16 columns from which workgroups share them, where few_parts() has more than one: each streams some 36 KB a us, and the
// sums' way through memory costs 2 us.  The whole call, us, by one / shared: 4 tokens, 24 of 64 experts of 2048 x 1408, bf16 86.7 / 77.9; 1 token,
// 6 of them (0.26 MB) 42.3 / 40.6, in MXFP4 (0.07 MB) 25.8 / 27.2; 16 tokens, 32 experts of 1024 x 512, bf16, by four 42.2 / 35.4.
constexpr int64_t kShareBytes = 192 << 10;
// Router products up to which every workgroup makes the logits itself instead of a launch in front: an expert a wavefront, about.  One token, the
// whole call in us, launch in front / not: 8 experts, H 4096, 51.2 / 48.3; 64 experts, H 2048, 25.8 / 28.3; 256, H 7168, 67.7 / 159.
constexpr int64_t kFoldProducts = 1 << 16;

template <class W, class ET, bool COLD>
hipError_t launch_few_form(const FewArgs& a, hipStream_t st) {
    const bool gated = a.w_gate != nullptr;
    const int64_t most = std::min<int64_t>(a.E, (int64_t)a.S * a.k) * (a.I / (gated ? 16 : 32));      // tasks there can be
    const int chunks = (a.H + W::K - 1) / W::K, lds = skinny_lds<W>(a.S);
    // Wavefronts of a task: until there are more than a thousand, and no less than a unit of chunks for each.  The whole call for one token, in us,
    // with 1 / 2 / 4 / 8: 528 tasks (64 experts of 1408 x 2048, 6 chosen) MXFP4 31.6 / 28.3 / 32.1 / 42.8, bf16 58 / 45 / 48 / 58; 1024 tasks of 28
    // chunks 67.6 / 57.4 / 56.5 / 61.5; 256 tasks of 16 chunks 33 / 26 / 22 / 22.
    int KS = 1;
    while (KS < kFewWaves && 2 * KS * kUnit <= chunks && most * KS <= 1024) KS *= 2;
    const int64_t sets = (most + kFewWaves / KS - 1) / (kFewWaves / KS);
    // (as many workgroups as there is room for at once: every one of them makes the plan)
    const unsigned grid = (unsigned)(KS > 1 ? sets : std::min<int64_t>(sets, 512));
    const int up_lds = kFewWaves * (KS > 1 ? lds : std::min(lds, kRowLds));
    hipError_t e = gated ? allow_lds(few_up_kernel<W, ET, true, COLD>, up_lds) : allow_lds(few_up_kernel<W, ET, false, COLD>, up_lds);
    if (e != hipSuccess) return e;
    if (gated) few_up_kernel<W, ET, true, COLD><<<grid, kFewThreads, up_lds, st>>>(a, KS);
    else few_up_kernel<W, ET, false, COLD><<<grid, kFewThreads, up_lds, st>>>(a, KS);
    e = hipGetLastError();
    if (e != hipSuccess) return e;
    const int down_lds = kFewWaves * std::min(lds, kRowLds);
    e = allow_lds(few_down_kernel<W, ET, COLD>, down_lds);
    if (e != hipSuccess) return e;
    few_down_kernel<W, ET, COLD><<<a.H / 16 * a.parts, kFewThreads, down_lds, st>>>(a);
    return hipGetLastError();
}
template <class W, class ET>
hipError_t launch_few_weights(const FewArgs& a, hipStream_t st) {
    const int64_t experts = std::min<int64_t>(a.E, (int64_t)a.S * a.k);
    const bool cold = experts * W::row_bytes((int64_t)a.H * a.I) * (a.w_gate ? 3 : 2) > ((int64_t)256 << 20);     // more than the memory-side cache holds
    return cold ? launch_few_form<W, ET, true>(a, st) : launch_few_form<W, ET, false>(a, st);
}

}  // namespace

hipError_t launch_few(FewArgs a, bool f16, bool mxfp4, hipStream_t st) {
    a.fold = (int64_t)a.S * a.E * a.H <= kFoldProducts && a.S * a.E * (int)sizeof(float) <= kFewWaves * 2048;       // (the least LDS that the rows have)
    if (std::min<int64_t>(a.E, (int64_t)a.S * a.k) * 16 * (mxfp4 ? a.I / 2 : 2 * (int64_t)a.I) < kShareBytes) a.parts = 1;
    if (!a.fold) {
        const int waves = a.E * ((a.S + kLogitTokens - 1) / kLogitTokens);
        if (f16) few_logits_kernel<f16_s><<<(waves + 3) / 4, 256, 0, st>>>(a);
        else few_logits_kernel<bf16_s><<<(waves + 3) / 4, 256, 0, st>>>(a);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    if (mxfp4) return launch_few_weights<WeightsMx<false>, bf16_s>(a, st);
    return f16 ? launch_few_weights<Weights16<f16_s>, f16_s>(a, st) : launch_few_weights<Weights16<bf16_s>, bf16_s>(a, st);
}

}  // namespace moe355
