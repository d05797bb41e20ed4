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
//
// The comparisons are of integers that order like the logits (0 for NaN and for what is taken), so that a round is two redux
// instructions: the largest value, then the lowest id that has it. With floats and ids compared through shuffles (ten of them a round)
// and a score per round, 32 tokens of 128 experts, k 8, took a block of eight warps 14.5 us; now a block of sixteen takes 6.1 with the loads
// of the logits before and the list of the experts hit behind.
template <int kPerLane>
__device__ __forceinline__ void topk_of_token(const float* row, int E, int k, int slots, int scoring, int lane, int* indices,
                                              float* weights) {
    uint32_t x[kPerLane];
#pragma unroll
    for (int i = 0; i < kPerLane; ++i) {
        const int e = i * 32 + lane;
        const float v = e < E ? row[e] + 0.0f : 0.0f;  // -0 counts as 0
        const uint32_t bits = __float_as_uint(v);
        x[i] = e < E && v == v ? (bits & 0x80000000u ? ~bits : bits | 0x80000000u) : 0u;
    }
    float value = -INFINITY;  // lane j keeps the j-th selected
    int index = 0x7fffffff;
    for (int j = 0; j < k; ++j) {
        uint32_t best = 0;
        int id = 0x7fffffff;
#pragma unroll
        for (int i = 0; i < kPerLane; ++i)
            if (x[i] > best) {
                best = x[i];
                id = i * 32 + lane;
            }
        const uint32_t top = __reduce_max_sync(0xffffffffu, best);
        if (top == 0) break;  // nothing left: the last slots keep -inf and an id that is none
        const int bi = int(__reduce_min_sync(0xffffffffu, best == top ? uint32_t(id) : 0x7fffffffu));
        // an expert is chosen at most once, also when fewer than k logits are above -inf
#pragma unroll
        for (int i = 0; i < kPerLane; ++i)
            if (i * 32 + lane == bi) x[i] = 0;
        if (lane == j) {
            value = __uint_as_float(top & 0x80000000u ? top & 0x7fffffffu : ~top);
            index = bi;
        }
    }
    const float m = __shfl_sync(0xffffffffu, value, 0);
    // sigmoid(v) = e^v / (1 + e^v). expf(-v) overflows from v = -88.8 down, where this is 0: a loss below 2^-24 of the largest chosen score as long as
    // that one's m is -72 or more. Below, 1 + e^v is 1 in fp32, and e^(v - m) the same ratios.
    const float score = scoring == DQMOE_SCORE_SIGMOID && !(m < -72.0f) ? 1.0f / (1.0f + expf(-value)) : expf(value - m);
    float denom = 0.0f;
    for (int j = 0; j < k; ++j) denom += __shfl_sync(0xffffffffu, score, j);
    if (lane < k) {
        indices[lane] = index;
        weights[lane] = score / denom;
    } else if (lane < slots) {
        indices[lane] = E + (lane - k);
        weights[lane] = 1.0f;
    }
}

}  // namespace route
}  // namespace dq
