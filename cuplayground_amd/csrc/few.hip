// A whole layer for a few tokens (at most 16): router, selection, expert FFN and combine in two launches, or three where the router is large.
//
// With one to sixteen tokens the layer is its weights, once: those of the experts that are hit, 0.1 to 2 GB in 16 bits or MXFP4, and
// nothing else is worth a launch of its own.  What the general path takes six launches for (logits, selection, slots and task tables, two
// projections, combine) is here
//   few_up    every workgroup finds out for itself which experts are hit and by whom -- the logits where the router is small (else
//             few_logits has left them), the selection a token a wavefront, a mask of tokens an expert -- and streams gate and up rows;
//   few_down  a workgroup owns 16 output columns and goes through all experts that are hit: with the tokens as the columns of the matrix
//             instruction's result, an expert's share of the combine is a multiply-add on the accumulators, in fp32, and out is written
//             once.  No expert's output row is ever rounded or stored.
// Weights stream as in skinny.hpp.  The router's sums and selection are those of the general path to the bit (the fixed order of 64
// partial sums; topk.hpp), and so are slots, drops and packed rows: the intermediate lies where that path would put it.
#include "act_deriv.hpp"
#include "skinny.hpp"
#include "topk.hpp"

namespace moe355 {
namespace {

constexpr int kFewThreads = 512, kFewWaves = 8;
constexpr int kFewPairs = kFewTokens * kMaxTopK;

// What every workgroup knows of the routing.
struct FewPlan {
    float w[kFewPairs];                // [S, k] gate weights
    int32_t idx[kFewPairs];            // [S, k] experts
    uint32_t mask[kMaxExperts];        // tokens an expert keeps
    int16_t base[kMaxExperts];         // packed row of its first one
    int16_t list[kFewPairs];           // experts that are hit, ascending
    float row_w[kFewPairs];            // gate weight of a packed row
    int32_t hit, kept;
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

// Logits of one expert for tokens t0 .. t0 + n - 1 (n <= TT) by a wavefront: lane p adds up, in ascending k, the products of every k with
// (k / 8) % 64 == p, one multiply-add each; the partial sums are folded pairwise.  logits[t] at out[t * stride].
template <class ET, int TT>
__device__ __forceinline__ void few_logits(const uint16_t* __restrict__ x, const uint16_t* __restrict__ g, const float* bias, int e, int t0, int n, int H, float* out, int stride, int lane) {
    float p[TT];
#pragma unroll
    for (int t = 0; t < TT; ++t) p[t] = 0.0f;
    for (int k = 8 * lane; k < H; k += 512) {
        union { mx_u32x4 v; uint16_t s[8]; } gv, xv;
        gv.v = *reinterpret_cast<const mx_u32x4*>(g + (int64_t)e * H + k);
#pragma unroll
        for (int t = 0; t < TT; ++t) {
            xv.v = *reinterpret_cast<const mx_u32x4*>(x + (int64_t)(t0 + min(t, n - 1)) * H + k);
#pragma unroll
            for (int i = 0; i < 8; ++i) p[t] = __builtin_fmaf(few_widen<ET>(xv.s[i]), few_widen<ET>(gv.s[i]), p[t]);
        }
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
    for (int e = tid; e < a.E; e += blockDim.x) p.mask[e] = 0;
    __syncthreads();
    if (tid < P && (unsigned)p.idx[tid] < (unsigned)a.E) atomicOr(&p.mask[p.idx[tid]], 1u << (tid / a.k));     // a token names an expert once
    __syncthreads();
    if (tid < kWave) {
        int hit = 0, rows = 0;
        for (int c = 0; c < a.E; c += kWave) {
            const int e = c + lane;
            uint32_t m = e < a.E ? p.mask[e] : 0u;
            if (a.drop)                                        // the first `capacity` tokens stay
                while (__popc(m) > a.capacity) m &= ~(1u << (31 - __clz(m)));
            const int n = __popc(m);
            int inc = n;
#pragma unroll
            for (int off = 1; off < kWave; off <<= 1) {
                const int o = __shfl_up(inc, off, kWave);
                if (lane >= off) inc += o;
            }
            const unsigned long long any = __ballot(n > 0);
            if (e < a.E) {
                p.mask[e] = m;
                p.base[e] = (int16_t)(rows + inc - n);
            }
            if (n > 0) p.list[hit + __popcll(any & ((1ull << lane) - 1ull))] = (int16_t)e;
            hit += __popcll(any);
            rows += __shfl(inc, kWave - 1, kWave);
        }
        if (lane == 0) p.hit = hit, p.kept = rows;
    }
    __syncthreads();
    if (tid < P) {
        const int e = p.idx[tid], t = tid / a.k;
        if ((unsigned)e < (unsigned)a.E && ((p.mask[e] >> t) & 1u)) p.row_w[p.base[e] + __popc(p.mask[e] & ((1u << t) - 1u))] = p.w[tid];
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

// Runs units [0, n) through a ring of two: load(b) fetches the next unit into buffer b, take(b) multiplies what lies there.  (Loads behind a
// condition in the loop would make every wait one for all of them.)
template <class LOAD, class TAKE>
__device__ __forceinline__ void few_ring(int n, LOAD load, TAKE take) {
    if (n > 0) load(0);
    if (n > 1) load(1);
    int i = 0;
    for (; i + 3 < n; i += 2) {
        take(0);
        load(0);
        take(1);
        load(1);
    }
    if (n - i > 0) take(0);
    if (n - i > 2) load(0);
    if (n - i > 1) take(1);
    if (n - i > 2) take(0);
}

// What both projections hold of a unit: weights of G groups of 16 rows, the token rows' pieces.
template <class W, int G>
struct FewUnit {
    SkinnyChunk<W, G> w;
    mx_u32x4 x[W::FRAGS];
};
template <class W, int G, bool COLD, bool CUT>
__device__ __forceinline__ void few_fetch(FewUnit<W, G>& u, const SkinnyRows (&rows)[G], const uint16_t* x, int c, int full, int left, int lane) {
    if (CUT && c == full) {
        skinny_load_tail<W, G, COLD>(u.w, rows, c, (int)W::row_bytes(left), lane);
        skinny_tokens_tail<W>(u.x, x, c, left, lane);
    } else {
        skinny_load<W, G, COLD>(u.w, rows, c);
        skinny_tokens<W>(u.x, x, c, lane);
    }
}
template <class W, int G, bool CUT>
__device__ __forceinline__ void few_multiply(mx_f32x4 (&acc)[G], FewUnit<W, G>& u, int c, int full, int left, int lane) {
    skinny_settle(u.w);
    if (CUT && c == full) skinny_zero_tail(u.w, (int)W::row_bytes(left), lane);
    skinny_multiply<W, G>(acc, u.w, u.x, lane);
}

// The up (and gate) projection: a task is 16 columns of both matrices of an expert, or 32 of the one, over the whole of H, by KS wavefronts.
// With KS = 1 a wavefront goes from task to task without a pause: the next one's weights are requested under the last ones' products.
template <class W, class ET, bool GATED, bool COLD, bool CUT>
__global__ __launch_bounds__(kFewThreads, 2) void few_up_kernel(FewArgs a, int KS) {
    __shared__ FewPlan plan;
    __shared__ mx_f32x4 red[(kFewWaves - 1) * 2 * 64];           // first the logits of a small router
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const float* logits = a.logits;
    if (a.fold) {
        float* own = reinterpret_cast<float*>(red);
        for (int e = wave; e < a.E; e += kFewWaves)
            for (int t0 = 0; t0 < a.S; t0 += kLogitTokens)
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
    if (blockIdx.x == 0) few_report(plan, a);

    constexpr int G = 2, COLS = GATED ? 16 : 32;
    const int H = a.H, I = a.I, full = H / W::K, left = H - full * W::K, chunks = full + (left ? 1 : 0);
    const int ncol = I / COLS, tasks = plan.hit * ncol;
    const int ks = wave % KS, first = blockIdx.x * (kFewWaves / KS) + wave / KS, stride = gridDim.x * (kFewWaves / KS);
    const int mine = ks < chunks ? (chunks - ks + KS - 1) / KS : 0;                            // chunks of a task that are this wavefront's
    const int idx = lane & 15, q = lane >> 4;
    const int64_t mat = W::row_bytes((int64_t)H * I), smat = (int64_t)I * (H >> 5);

    // (with KS > 1 the launch has a set of wavefronts for every task there can be)
    const int mytasks = first < tasks ? (KS > 1 ? 1 : (tasks - 1 - first) / stride + 1) : 0;
    FewUnit<W, G> u[2];
    SkinnyRows rows[G];
    const uint16_t* x = nullptr;
    int lt = first, lc = ks;             // the next unit to load: its task and chunk
    auto aim = [&]() {
        const int j = lt / ncol, n0 = (lt - j * ncol) * COLS;
        const int e = __builtin_amdgcn_readfirstlane(plan.list[j]);
        const uint32_t m = plan.mask[e];
        uint32_t rest = m;               // the idx-th token of the mask; lanes behind the last one take the first
        for (int i = 0; i < idx && (rest & (rest - 1)); ++i) rest &= rest - 1;
        const int t = __ffs(idx < __popc(m) ? rest : m) - 1;
        x = (const uint16_t*)a.x + (int64_t)t * H;
#pragma unroll
        for (int g = 0; g < G; ++g)
            rows[g] = skinny_rows<W>(static_cast<const char*>(GATED && g ? a.w_gate : a.w_up) + e * mat, W::MX ? (GATED && g ? a.s_gate : a.s_up) + e * smat : nullptr,
                                     n0 + (GATED ? 0 : 16 * g), I, H, lane);
    };
    auto load = [&](int b) {
        if (lc == ks) aim();
        few_fetch<W, G, COLD, CUT>(u[b], rows, x, lc, full, left, lane);
        lc += KS;
        if (lc >= chunks) lc = ks, lt += stride;
    };
    mx_f32x4 acc[G] = {};
    auto store = [&](int task) {
        const int j = task / ncol, n0 = (task - j * ncol) * COLS;
        const int e = __builtin_amdgcn_readfirstlane(plan.list[j]);
        if (idx >= __popc(plan.mask[e])) return;
        uint16_t* h = (uint16_t*)a.h + (int64_t)(plan.base[e] + idx) * I;
        const uint16_t* bu = a.b_up ? (const uint16_t*)a.b_up + (int64_t)e * I : nullptr;
        const uint16_t* bg = a.b_gate ? (const uint16_t*)a.b_gate + (int64_t)e * I : nullptr;
        auto put = [&](int col, float (&v)[4]) {
            *reinterpret_cast<uint2*>(h + col) = uint2{few_pack<ET>(v[0], v[1]), few_pack<ET>(v[2], v[3])};
        };
        if constexpr (GATED) {
            const int col = n0 + 4 * q;
            float v[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float up = acc[0][r] + (bu ? few_widen<ET>(bu[col + r]) : 0.0f), gate = acc[1][r] + (bg ? few_widen<ET>(bg[col + r]) : 0.0f);
                v[r] = silu16(gate) * up;
            }
            put(col, v);
        } else {
#pragma unroll
            for (int g = 0; g < G; ++g) {
                const int col = n0 + 16 * g + 4 * q;
                float v[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const float up = acc[g][r] + (bu ? few_widen<ET>(bu[col + r]) : 0.0f);
                    v[r] = a.act == MOE_ACT_GELU ? gelu16(up) : (up < 0.0f ? 0.0f : up);
                }
                put(col, v);
            }
        }
    };
    int ct = first, cc = ks;             // the next unit to multiply
    auto take = [&](int b) {
        few_multiply<W, G, CUT>(acc, u[b], cc, full, left, lane);
        cc += KS;
        if (cc >= chunks) {
            if (KS == 1) {
                store(ct);
#pragma unroll
                for (int g = 0; g < G; ++g) acc[g] = mx_f32x4{0.f, 0.f, 0.f, 0.f};
            }
            cc = ks, ct += stride;
        }
    };
    few_ring(mytasks * mine, load, take);
    if (KS > 1) {
        const bool holds = skinny_join<G>(acc, ks, KS, red + wave / KS * (KS - 1) * G * 64, lane);
        if (holds && mytasks) store(first);
    }
}

// The down projection and the combine: a workgroup owns 16 G columns of out; its wavefronts share the (expert, chunk of I) units.
template <class W, class ET, int G, bool COLD, bool CUT>
__global__ __launch_bounds__(kFewThreads, 2) void few_down_kernel(FewArgs a) {
    __shared__ FewPlan plan;
    __shared__ mx_f32x4 red[(kFewWaves - 1) * G * 64];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    if (tid < a.S * a.k) {
        plan.idx[tid] = a.topk_idx[tid];
        plan.w[tid] = a.topk_w[tid];
    }
    __syncthreads();
    few_plan(plan, a);

    const int H = a.H, I = a.I, full = I / W::K, left = I - full * W::K, chunks = full + (left ? 1 : 0);
    const int n0 = blockIdx.x * 16 * G;
    const int idx = lane & 15, q = lane >> 4;
    const int64_t mat = W::row_bytes((int64_t)H * I), smat = (int64_t)H * (I >> 5);
    const int units = plan.hit * chunks;
    const int begin = (int)((int64_t)units * wave / kFewWaves), end = (int)((int64_t)units * (wave + 1) / kFewWaves);
    FewUnit<W, G> u[2];
    SkinnyRows rows[G];
    const uint16_t* x = nullptr;
    int lj = begin / max(chunks, 1), lc = begin - lj * chunks;
    auto aim = [&]() {
        const int e = __builtin_amdgcn_readfirstlane(plan.list[lj]);
        const uint32_t m = plan.mask[e];
        // lane idx is token idx; where that is not the expert's, its first row is read and the sum left out
        const int at = (m >> idx) & 1u ? __popc(m & ((1u << idx) - 1u)) : 0;
        x = (const uint16_t*)a.h + (int64_t)(plan.base[e] + at) * I;
#pragma unroll
        for (int g = 0; g < G; ++g) rows[g] = skinny_rows<W>(static_cast<const char*>(a.w_down) + e * mat, W::MX ? a.s_down + e * smat : nullptr, n0 + 16 * g, H, I, lane);
    };
    bool aimed = false;
    auto load = [&](int b) {
        if (!aimed || lc == 0) aim(), aimed = true;
        few_fetch<W, G, COLD, CUT>(u[b], rows, x, lc, full, left, lane);
        if (++lc == chunks) lc = 0, ++lj;
    };
    mx_f32x4 out[G] = {}, acc[G] = {};
    int cj = lj, cc = lc, done = begin;
    auto take = [&](int b) {
        if (cc == 0 && a.b_down) {       // the expert's bias goes with its first chunk
            const uint16_t* bd = (const uint16_t*)a.b_down + (int64_t)__builtin_amdgcn_readfirstlane(plan.list[cj]) * H + n0 + 4 * q;
#pragma unroll
            for (int g = 0; g < G; ++g)
#pragma unroll
                for (int r = 0; r < 4; ++r) acc[g][r] = few_widen<ET>(bd[16 * g + r]);
        }
        few_multiply<W, G, CUT>(acc, u[b], cc, full, left, lane);
        ++done;
        if (++cc == chunks || done == end) {
            const int e = __builtin_amdgcn_readfirstlane(plan.list[cj]);
            const uint32_t m = plan.mask[e];
            if ((m >> idx) & 1u) {
                const float w = plan.row_w[plan.base[e] + __popc(m & ((1u << idx) - 1u))];
#pragma unroll
                for (int g = 0; g < G; ++g)
#pragma unroll
                    for (int r = 0; r < 4; ++r) out[g][r] = __builtin_fmaf(w, acc[g][r], out[g][r]);
            }
#pragma unroll
            for (int g = 0; g < G; ++g) acc[g] = mx_f32x4{0.f, 0.f, 0.f, 0.f};
            cc = 0, ++cj;
        }
    };
    few_ring(end - begin, load, take);
    if (!skinny_join<G>(out, wave, kFewWaves, red, lane) || idx >= a.S) return;
#pragma unroll
    for (int g = 0; g < G; ++g)
        *reinterpret_cast<uint2*>((uint16_t*)a.out + (int64_t)idx * H + n0 + 16 * g + 4 * q) = uint2{few_pack<ET>(out[g][0], out[g][1]), few_pack<ET>(out[g][2], out[g][3])};
}

// Router products up to which every workgroup makes the logits itself instead of a launch in front.
constexpr int64_t kFoldProducts = 1 << 18;

template <class W, class ET, bool COLD, bool CUT_UP, bool CUT_DOWN>
hipError_t launch_few_form(const FewArgs& a, hipStream_t st) {
    const bool gated = a.w_gate != nullptr;
    const int64_t most = std::min<int64_t>(a.E, (int64_t)a.S * a.k) * (a.I / (gated ? 16 : 32));      // tasks there can be
    const int chunks = (a.H + W::K - 1) / W::K;
    int KS = 1;
    while (KS < kFewWaves && 2 * KS <= chunks && most * KS < 1024) KS *= 2;
    const int64_t sets = (most + kFewWaves / KS - 1) / (kFewWaves / KS);
    const unsigned grid = (unsigned)(KS > 1 ? sets : std::min<int64_t>(sets, 512));
    if (gated) few_up_kernel<W, ET, true, COLD, CUT_UP><<<grid, kFewThreads, 0, st>>>(a, KS);
    else few_up_kernel<W, ET, false, COLD, CUT_UP><<<grid, kFewThreads, 0, st>>>(a, KS);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    few_down_kernel<W, ET, 1, COLD, CUT_DOWN><<<a.H / 16, kFewThreads, 0, st>>>(a);
    return hipGetLastError();
}
template <class W, class ET, bool COLD>
hipError_t launch_few_cut(const FewArgs& a, hipStream_t st) {
    const bool up = a.H % W::K, down = a.I % W::K;
    if (up) return down ? launch_few_form<W, ET, COLD, true, true>(a, st) : launch_few_form<W, ET, COLD, true, false>(a, st);
    return down ? launch_few_form<W, ET, COLD, false, true>(a, st) : launch_few_form<W, ET, COLD, false, false>(a, st);
}
template <class W, class ET>
hipError_t launch_few_weights(const FewArgs& a, hipStream_t st) {
    const int64_t experts = std::min<int64_t>(a.E, (int64_t)a.S * a.k);
    const bool cold = experts * W::row_bytes((int64_t)a.H * a.I) * (a.w_gate ? 3 : 2) > ((int64_t)256 << 20);     // more than the memory-side cache holds
    return cold ? launch_few_cut<W, ET, true>(a, st) : launch_few_cut<W, ET, false>(a, st);
}

}  // namespace

hipError_t launch_few(FewArgs a, bool f16, bool mxfp4, hipStream_t st) {
    a.fold = (int64_t)a.S * a.E * a.H <= kFoldProducts && a.S * a.E <= (kFewWaves - 1) * 2 * 64 * 4;
    if (!a.fold) {
        const int waves = a.E * ((a.S + kLogitTokens - 1) / kLogitTokens);
        if (f16) few_logits_kernel<f16_s><<<(waves + 3) / 4, 256, 0, st>>>(a);
        else few_logits_kernel<bf16_s><<<(waves + 3) / 4, 256, 0, st>>>(a);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    if (mxfp4) return launch_few_weights<WeightsMx, bf16_s>(a, st);
    return f16 ? launch_few_weights<Weights16<f16_s>, f16_s>(a, st) : launch_few_weights<Weights16<bf16_s>, bf16_s>(a, st);
}

}  // namespace moe355
