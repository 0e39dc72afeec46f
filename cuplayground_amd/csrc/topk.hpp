// Top-k selection and gate weights of one token by one wavefront; shared by the stand-alone top-k kernel and by the
// single-workgroup router of decode-sized layers.
//
// Bound by its own steps, k times a search for the largest: on integer keys a step is a maximum a lane, four across lanes and a ballot a
// slot; comparing (value, index) pairs through every exchange took four times as long (two tokens of 256 experts, 8 of them: 8 us, now 2).
#pragma once

#include "moe_internal.hpp"

namespace moe355 {

// Logits as integers in their order: a NaN ranks as -inf (and 0 behind that is no logit's), -0 as 0.
__device__ __forceinline__ uint32_t rank_key(float v) {
    const uint32_t u = __float_as_uint(v != v ? -INFINITY : v + 0.0f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
// The largest of the 64 lanes' keys: lanes exchange through the cross-lane data paths of the ALU (within quads, then mirrored within 8
// and 16 lanes), which cost a few cycles each where a shuffle through the LDS crossbar costs a round trip, and the four rows meet
// through scalar registers.
template <int CTRL>
__device__ __forceinline__ uint32_t dpp_max(uint32_t k) {
    return max(k, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)k, CTRL, 0xF, 0xF, false));
}
__device__ __forceinline__ uint32_t wave_max(uint32_t k) {
    k = dpp_max<0xB1>(k);             // quad_perm [1,0,3,2]: lane ^ 1
    k = dpp_max<0x4E>(k);             // quad_perm [2,3,0,1]: lane ^ 2
    k = dpp_max<0x141>(k);            // row_half_mirror: i <-> 7 - i within 8 lanes
    k = dpp_max<0x140>(k);            // row_mirror: i <-> 15 - i within 16 lanes
    const uint32_t a = max((uint32_t)__builtin_amdgcn_readlane((int)k, 0), (uint32_t)__builtin_amdgcn_readlane((int)k, 16));
    const uint32_t b = max((uint32_t)__builtin_amdgcn_readlane((int)k, 32), (uint32_t)__builtin_amdgcn_readlane((int)k, 48));
    return max(a, b);
}

// `row`: the E logits of token t (global memory, or LDS when the logits kernel selects right behind its sums).
// Lane l keeps the logits of experts l, l+64, ... (J of them; J * 64 >= E) in registers.  Called by all 64 lanes of a
// wavefront.  J is a template parameter so that layers with up to 64 experts do not walk eight slots per step.
// The selection is total: a NaN logit ranks as -inf (behind every number, ties to the lower index), so a token row
// that overflowed still gets k distinct, valid experts; its weights are computed from the logits as they are and
// come out NaN, which is what reaches the output of that token and of no other.
template <int J>
__device__ __forceinline__ void topk_one_token(const float* __restrict__ row, int t, int E, int k, int gate_fn,
                                               int norm, int32_t* __restrict__ topk_idx, float* __restrict__ topk_w,
                                               int lane) {
    static_assert(J >= 1 && J <= kMaxExperts / kWave, "slots per lane");
    float v[J];
    uint32_t key[J];                  // 0: no expert, or taken
    unsigned valid = 0;
#pragma unroll
    for (int j = 0; j < J; ++j) {
        const int e = j * kWave + lane;
        v[j] = 0.0f;
        key[j] = 0;
        if (e < E) {
            v[j] = row[e];
            key[j] = rank_key(v[j]);
            valid |= 1u << j;
        }
    }
    int my_i = 0;
    for (int r = 0; r < k; ++r) {
        uint32_t most = key[0];
#pragma unroll
        for (int j = 1; j < J; ++j) most = max(most, key[j]);
        most = wave_max(most);
        int i = 0;                    // the lowest index that has it
#pragma unroll
        for (int j = J - 1; j >= 0; --j) {
            const unsigned long long m = __ballot(key[j] == most);
            if (m) i = j * kWave + __builtin_ctzll(m);
        }
#pragma unroll
        for (int j = 0; j < J; ++j)
            if (j * kWave + lane == i) key[j] = 0;
        if (lane == r) my_i = i;
    }
    // the logits behind the keys, as stored (a NaN ranks as -inf but stays a NaN in the weights)
    float my_l = 0.0f;
#pragma unroll
    for (int j = 0; j < J; ++j) {
        const float l = __shfl(v[j], my_i & (kWave - 1), kWave);
        if ((my_i >> 6) == j) my_l = l;
    }
    const float top_l = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(my_l), 0));
    float p = 0.0f;
    if (gate_fn == MOE_GATE_SOFTMAX) {
        float part = 0.0f;
#pragma unroll
        for (int j = 0; j < J; ++j)
            if ((valid >> j) & 1u) part = part + expf(v[j] - top_l);
#pragma unroll
        for (int off = 32; off >= 1; off >>= 1) part = part + __shfl_xor(part, off, kWave);
        if (lane < k) p = expf(my_l - top_l) / part;
    } else {
        if (lane < k) p = 1.0f / (1.0f + expf(-my_l));
    }
    if (norm) {
        float sum = p;
#pragma unroll
        for (int off = 32; off >= 1; off >>= 1) sum = sum + __shfl_xor(sum, off, kWave);
        p = p / sum;
    }
    if (lane < k) {
        topk_idx[(size_t)t * k + lane] = my_i;
        topk_w[(size_t)t * k + lane] = p;
    }
}

}  // namespace moe355
