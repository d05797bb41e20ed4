// Top-k choice of one token's experts by one warp, shared by the router kernels (route.cu) and the MoE layer for a few tokens
// (moe_decode.cu).
#pragma once

#include "common.cuh"

namespace dq {
namespace route {

// One warp per token. Ranking is by logit (both scoring functions are monotonic),
// value descending then expert id ascending; weights are the selected scores
// normalised to sum 1. Output rows have `slots` >= k entries: entries k.. name the shared
// experts E, E+1, ... (every token, weight 1), which the layer then treats like routed ones.
template <int kPerLane>
__device__ __forceinline__ void topk_of_token(const float* row, int E, int k, int slots, int scoring, int lane, int* indices,
                                              float* weights) {
    float x[kPerLane];
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < kPerLane; ++i) {
        const int e = i * 32 + lane;
        x[i] = e < E ? row[e] : -INFINITY;
        m = fmaxf(m, x[i]);
    }
    m = warp_max(m);
    float sel_score = 0.0f;  // lane j keeps the j-th selected score
    int sel_idx = 0;
    float denom = 0.0f;
    uint32_t taken = 0;      // bit i: this lane's i-th expert has been selected (an expert is chosen at most once,
                             // also when fewer than k logits are above -inf)
    for (int j = 0; j < k; ++j) {
        float bv = -INFINITY;
        int bi = 0x7fffffff;
#pragma unroll
        for (int i = 0; i < kPerLane; ++i) {
            const int e = i * 32 + lane;
            if (e < E && ((taken >> i) & 1u) == 0u && (x[i] > bv || (x[i] == bv && e < bi))) {
                bv = x[i];
                bi = e;
            }
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            const float ov = __shfl_xor_sync(0xffffffffu, bv, o);
            const int oi = __shfl_xor_sync(0xffffffffu, bi, o);
            if (ov > bv || (ov == bv && oi < bi)) {
                bv = ov;
                bi = oi;
            }
        }
        // remove the winner from its owner lane
#pragma unroll
        for (int i = 0; i < kPerLane; ++i)
            if (i * 32 + lane == bi) taken |= 1u << i;
        const float score = scoring == DQMOE_SCORE_SIGMOID ? 1.0f / (1.0f + expf(-bv)) : expf(bv - m);
        denom += score;
        if (lane == j) {
            sel_score = score;
            sel_idx = bi;
        }
    }
    if (lane < k) {
        indices[lane] = sel_idx;
        weights[lane] = sel_score / denom;
    } else if (lane < slots) {
        indices[lane] = E + (lane - k);
        weights[lane] = 1.0f;
    }
}

}  // namespace route
}  // namespace dq
