// The whole MoE layer for up to 32 tokens in two launches: x [T, H] and the router's weights in, out [T, H] out.
//
//   route    logits = x Wr^T in fp32 (clusters of eight blocks, slices of H), x laid out as the tensor core's second operand
//   experts  top-k of every token (each block for itself), the experts that are hit, fc1 + SwiGLU, fc2, sum over the experts
//
// What bounds it: the weights of the experts hit, once from HBM. Everything else is arranged around that stream:
//   - The weights are the tensor core's first operand (M = 128 weight rows), all T tokens the second (N), for every expert that any
//     token chose; columns of tokens that did not choose it are computed and dropped. So there is no sort, no gather and no
//     dependence of the weight stream on who chose what. The MMAs take a fraction of the time that the weights take to arrive.
//   - FP8 weights meet activations that are not quantised: a value x of a group of 128 is split into hi + lo / 16, both e4m3, times a
//     power of two s with 128 <= amax / s < 256. e4m3 has four significant bits and the rest of a bf16 value after its first four has
//     four more, so the split is exact down to 2^-13 of the group's largest value and off by at most 2^-21 of that below it. hi and lo
//     are separate columns of the same MMA: N = 2 T, no conversion of weights, which go from memory to the tensor core untouched. The
//     intermediate (fp32) is split the same way, within 2^-9 of each value (bf16's half step is 2^-8); with bf16 weights into two bf16.
//   - Work comes in units of 32 KiB of weights (fc1: 128 gate and 128 value rows x 128 bytes; fc2: 128 rows x 256 bytes) and pieces of
//     several units, which the blocks claim one after the other from a counter: fc1's pieces expert by expert, then fc2's in the same order
//     of experts, ever smaller ones towards the end. fc2's first pieces need only experts that were finished long ago, so the stream does
//     not pause between the two, and no SM waits for a slower one.
//   - What takes trips through L2 - sums over the parts of a tile, the activation, the hand-over to fc2 - is done by four warps of
//     their own beside the stream; the second operand has a thread of its own that may wait for fc1 while weights are still fetched.
// A block waits for an expert's fc1 only when all of fc1 has been claimed by blocks that are running, and those finish it whatever
// happens: so the wait ends also where not all blocks fit the GPU at once (other streams' kernels, several of these among them).
// Sums are added in a fixed order whoever adds them: results do not depend on which block took which piece.
//
// us per call, first with one equal, static share of the units per SM, the sums and the activation on the warps that drain the accumulators and
// fc2 behind all of fc1, then as it is, both over one set of weights (and what a graph over 0.6 GB of them takes, at which bandwidth):
//   block FP8, H 1024, I 2048, 8 experts, k 2, 5 tokens                    44.8 / 22.8 (26.0: 1.3 TB/s)
//   bf16, H 4096, I 14336, 8 experts, k 2, 1 token                         124 / 120 (118: 6.0)
//   FP8 by tensor, H 4096, I 14336, 8 experts, k 2, 16 tokens              267 / 229 (229: 6.1)
//   block FP8, H 7168, I 2048, 32 experts, k 8, 1 shared, 8 tokens         224 / 204 (200: 6.3)
//   FP8 by channel, H 2048, I 768, 128 experts, k 8, 32 tokens             211 / 123 (124: 4.2)
// What is left above the weights' time is the chain of latencies before the first weight (route 3 us, top-k and plan 2 to 5), between fc1's last sum and
// fc2's first MMA (8), and behind the last (5): nearly all of the smallest case. At 32 tokens of many experts another 20 to 30 us are not accounted for.
//
// No counterpart in the reference, whose runner (csrc/moe_kernels.h:770-892) takes routed rows and five launches.
#include <cmath>
#include <mutex>

#include "common.cuh"
#include "gemm_tile.cuh"
#include "ptx_sm100.cuh"
#include "route_topk.cuh"
#include "streamk.cuh"

namespace dq {
namespace moe_decode {

constexpr int kMaxTokens = 32;
constexpr int kMaxExperts = 1024;
constexpr int kMaxTopk = 32;
// warp 0 weights, 1 MMA, 2 tokens, 3 count, warps 4..7 drain, warps 8..11 finish, warps 12..15 drain the second 16 of 32 tokens; all choose the experts
__host__ __device__ constexpr int threads(int tp) { return tp > 16 ? 512 : 384; }
constexpr int kRows = 128;                    // weight rows of an MMA
constexpr int kKBytes = 128;                  // bytes of a K block: one swizzle row
constexpr int kTileBytes = kRows * kKBytes;   // 16 KiB
constexpr int kABytes = 2 * kTileBytes;       // a unit's weights
constexpr int kRingBytes = 205 * 1024;
constexpr int kMaxSplit1 = 6;                 // parts of an fc1 tile
constexpr int kMaxParts = 40;                 // of an fc2 tile: this many at most shrink, the others are equal
constexpr int kMaxShrinking = 16;
constexpr int kGroup = 8;                     // parts that are added to one sum first
constexpr int kGroups = (kMaxParts + kGroup - 1) / kGroup;
constexpr int kMaxStages = 6;
constexpr int kScaleBytes = 1024;             // room behind a stage's second operand for its scales
constexpr int kClaims = 4, kJobs = 4;
constexpr int kStatusRing = 301, kStatusPhase = 302;
constexpr int kSplit = 8;                     // blocks of a route cluster: slices of H
constexpr int kRouteThreads = 256;

__host__ __device__ constexpr int token_rows(int T) { return T <= 8 ? 8 : T <= 16 ? 16 : 32; }
// columns of the second operand: hi and lo (FP8; the intermediate also with bf16 weights), M = 128 wants a multiple of 16
__host__ __device__ constexpr int fc1_cols(bool fp8, int tp) { return fp8 ? 2 * tp : (tp < 16 ? 16 : tp); }
__host__ __device__ constexpr int fc2_cols(int tp) { return 2 * tp; }
__host__ __device__ constexpr int stage_bytes(int tp) { return kABytes + 2 * fc2_cols(tp) * kKBytes + kScaleBytes; }
__host__ __device__ constexpr int stages(int tp) { return kRingBytes / stage_bytes(tp) < kMaxStages ? kRingBytes / stage_bytes(tp) : kMaxStages; }

struct Params {
    const __nv_bfloat16* x;
    const void* w_router;
    const float* b_scale;
    const float* b1_scale;
    __nv_bfloat16* out;
    int T, H, I, E, k, n_shared;
    int scoring, mode;
    int kb1, pairs2;          // K blocks of fc1; pairs of K blocks of fc2
    int tiles1, tiles2;       // tiles of 128 rows of I and H
    int blocks;
    float share, per_share, shrink_rate, even;  // of fc2's parts, see plan_parts2
    int max_hit;              // experts hit at most
    int n_counters;
    size_t rec1, rec2;        // bytes of a unit's second operand with its scales
    int* counters;            // claims; finished fc1 tiles of each expert; parts seen of each fc1 tile, of each group of parts
                              // of an fc2 tile, groups seen of each fc2 tile
    float* logits;            // [T, E]
    uint8_t* xq;              // [kb1] records: [fc1_cols][128 B] swizzled, scales [token_rows]
    uint8_t* aq;              // [experts hit][pairs2] records: two of [fc2_cols][128 B] swizzled, scales [2][token_rows]
    // partial sums, four tokens of a weight row together: [token / 4][128][4]
    float* part1;             // [kJobs of each block, then pieces of split tiles][gate, value]
    float* part2;             // [tile][part]
    float* group2;            // [tile][group]
    int* status;
    long long wait_limit;     // clock cycles before a wait gives up
};

// byte `byte` of row `row` of an operand tile with 128-byte rows, as the 128-byte swizzle places it
__device__ __forceinline__ int swizzled(int row, int byte) { return row * kKBytes + (byte ^ ((row & 7) << 4)); }

// 2^(exponent(amax) - 7) for the largest of a group's magnitudes, given as bits, so that amax / s lies in [128, 256); not below 2^-100, and
// NaN where the group holds an infinity or a NaN (its token's results are NaN then)
__device__ __forceinline__ float split_scale(uint32_t amax_bits, float* inv) {
    if (amax_bits >= 0x7f800000u) {
        *inv = 0.0f;
        return __uint_as_float(0x7fffffffu);
    }
    const int e = max(int(amax_bits >> 23) - 127 - 7, -100);
    *inv = __uint_as_float(uint32_t(127 - e) << 23);
    return __uint_as_float(uint32_t(127 + e) << 23);
}
// two scaled values -> e4m3 pairs hi and lo with x = hi + lo / 16
__device__ __forceinline__ void split_e4m3x2(float x0, float x1, uint32_t* hi, uint32_t* lo) {
    *hi = f2e4m3x2(x0, x1);
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(*hi), __NV_E4M3);
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
    *lo = f2e4m3x2((x0 - f.x) * 16.0f, (x1 - f.y) * 16.0f);
}

// ---------------------------------------------------------------- route

// Three bf16 whose sum is the fp32 value to 2^-24 of it, two values at a time.
__device__ __forceinline__ void split3(float a, float b, uint32_t (&w)[3]) {
#pragma unroll
    for (int i = 0; i < 3; ++i) {
        w[i] = pack_bf16x2(a, b);
        a -= bf16_lo(w[i]);
        b -= bf16_hi(w[i]);
    }
}
// This warp's share of the logits of all tokens and eight experts, over chunks of 32 values of H. A thread loads 16 bytes of a row, eight values
// that follow one another; which of them an MMA takes for its k is the same for x and the weights, and a sum does not mind.
// Each value of x and each weight is read once per cluster. (With a warp per expert and fp32 FMAs each warp read all of x, and the kernel
// took 10.7 us for 32 tokens of H 2048 and 128 experts.)
template <bool kF32, int kM>
__device__ __forceinline__ void partial_logits(const Params& p, int e0, int first, int step, float* part /*[T][8]*/, int lane) {
    const int g = lane >> 2, kk = (lane & 3) * 8;
    float acc[kM][4] = {};
#pragma unroll 4
    for (int k0 = first * 32; k0 < p.H; k0 += step * 32) {
        const int k = k0 + kk;
        const bool in = k < p.H;
        uint4 x[kM][2];
#pragma unroll
        for (int m = 0; m < kM; ++m)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int t = m * 16 + h * 8 + g;
                x[m][h] = in && t < p.T ? *reinterpret_cast<const uint4*>(p.x + size_t(t) * p.H + k) : make_uint4(0, 0, 0, 0);
            }
        uint32_t w[kF32 ? 3 : 1][4] = {};
        if (in && e0 + g < p.E) {
            const size_t at = size_t(e0 + g) * p.H + k;
            if constexpr (kF32) {
                const float4* q = reinterpret_cast<const float4*>(static_cast<const float*>(p.w_router) + at);
                const float4 a = q[0], b = q[1];
                const float f[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    uint32_t s3[3];
                    split3(f[2 * i], f[2 * i + 1], s3);
                    w[0][i] = s3[0], w[1][i] = s3[1], w[2][i] = s3[2];
                }
            } else {
                const uint4 v = *reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(p.w_router) + at);
                w[0][0] = v.x, w[0][1] = v.y, w[0][2] = v.z, w[0][3] = v.w;
            }
        }
#pragma unroll
        for (int m = 0; m < kM; ++m)
#pragma unroll
            for (int i = (kF32 ? 2 : 0); i >= 0; --i) {
                ptx::mma_16x8x16<false>(acc[m], x[m][0].x, x[m][1].x, x[m][0].y, x[m][1].y, w[i][0], w[i][1]);
                ptx::mma_16x8x16<false>(acc[m], x[m][0].z, x[m][1].z, x[m][0].w, x[m][1].w, w[i][2], w[i][3]);
            }
    }
#pragma unroll
    for (int m = 0; m < kM; ++m)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int t = m * 16 + (i >> 1) * 8 + g;
            if (t < p.T) part[t * 8 + (lane & 3) * 2 + (i & 1)] = acc[m][i];
        }
}

// A K block of a token's x into its record.
template <bool kFp8>
__device__ __forceinline__ void lay_out_x(const Params& p, int kb, int t, int tp, int lane) {
    uint8_t* rec = p.xq + size_t(kb) * p.rec1;
    if constexpr (kFp8) {
        const int k = kb * kKBytes + lane * 4;
        uint2 v = make_uint2(0, 0);
        if (k < p.H) v = *reinterpret_cast<const uint2*>(p.x + size_t(t) * p.H + k);
        const uint32_t most = max(max((v.x & 0x7fffu) << 16, v.x & 0x7fff0000u), max((v.y & 0x7fffu) << 16, v.y & 0x7fff0000u));
        float inv;
        const float s = split_scale(__reduce_max_sync(0xffffffffu, most), &inv);
        uint32_t h0, l0, h1, l1;
        split_e4m3x2(bf16_lo(v.x) * inv, bf16_hi(v.x) * inv, &h0, &l0);
        split_e4m3x2(bf16_lo(v.y) * inv, bf16_hi(v.y) * inv, &h1, &l1);
        *reinterpret_cast<uint32_t*>(rec + swizzled(t, lane * 4)) = h0 | (h1 << 16);
        *reinterpret_cast<uint32_t*>(rec + swizzled(tp + t, lane * 4)) = l0 | (l1 << 16);
        if (lane == 0) reinterpret_cast<float*>(rec + fc1_cols(true, tp) * kKBytes)[t] = s;
    } else {
        const int k = kb * (kKBytes / 2) + lane * 2;
        const uint32_t v = k < p.H ? *reinterpret_cast<const uint32_t*>(p.x + size_t(t) * p.H + k) : 0u;
        *reinterpret_cast<uint32_t*>(rec + swizzled(t, lane * 4)) = v;
    }
}

template <bool kF32, bool kFp8>
__global__ void __launch_bounds__(kRouteThreads) moe_decode_route_kernel(const __grid_constant__ Params p) {
    pdl_enter();
    __shared__ float s_part[kRouteThreads / 32][kMaxTokens * 8], s_sum[kMaxTokens * 8];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = int(ptx::cluster_ctarank());
    const int chunk = blockIdx.x / kSplit;
    const int tp = token_rows(p.T);
    const bool working = chunk * 8 < p.E;
    if (working) {
        const int first = rank * (kRouteThreads / 32) + warp, step = kSplit * (kRouteThreads / 32);
        if (tp <= 16) partial_logits<kF32, 1>(p, chunk * 8, first, step, s_part[warp], lane);
        else partial_logits<kF32, 2>(p, chunk * 8, first, step, s_part[warp], lane);
    }
    for (int i = blockIdx.x * kRouteThreads + threadIdx.x; i < p.n_counters; i += gridDim.x * kRouteThreads) p.counters[i] = 0;
    const int warps = gridDim.x * (kRouteThreads / 32);
    for (int u = blockIdx.x * (kRouteThreads / 32) + warp; u < p.kb1 * p.T; u += warps) lay_out_x<kFp8>(p, u / p.T, u % p.T, tp, lane);
    if (!working) return;  // whole clusters
    __syncthreads();
    if (threadIdx.x < p.T * 8) {
        float sum = 0.0f;
#pragma unroll
        for (int w = 0; w < kRouteThreads / 32; ++w) sum += s_part[w][threadIdx.x];
        s_sum[threadIdx.x] = sum;
    }
    __syncthreads();
    ptx::cluster_sync();
    const int mine = chunk * 8 + rank;  // the expert whose slices this block adds
    if (mine < p.E && threadIdx.x < p.T) {
        float sum = 0.0f;
#pragma unroll
        for (int r = 0; r < kSplit; ++r) {
            float v;
            asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(ptx::map_to_cta(&s_sum[threadIdx.x * 8 + rank], r)) : "memory");
            sum += v;
        }
        p.logits[size_t(threadIdx.x) * p.E + mine] = sum;
    }
    __syncthreads();
    ptx::cluster_sync();  // the other blocks read this one's shared memory
}

// ---------------------------------------------------------------- experts

struct alignas(16) Tail {
    uint64_t full[kMaxStages], empty[kMaxStages];
    uint64_t tmem_full[4], tmem_empty[4];
    uint64_t claim_full[kClaims], claim_empty[kClaims];
    uint64_t job_full[kJobs], job_empty[kJobs];  // pieces whose sums are written, from the draining warps to the counting one
    uint64_t last_full[kJobs];                   // those that complete a tile or a group of parts, from there to the finishing warps
    uint64_t meet;                             // the finishing warps
    int claim[kClaims], job[kJobs], last_job[kJobs];
    uint32_t tmem_base;
    int abort_flag;
    int n_hit;
    int whole1, split1, pieces1;               // fc1 tiles in one piece; parts of each of the others; pieces of fc1
    int parts2;                                // of an fc2 tile
    int bound2[kMaxParts + 1];                 // first unit of each part of an fc2 tile
    uint32_t bad_tokens;                       // tokens without a number among their weights
    int last;
    alignas(16) float token_scale[4][2 * kMaxTokens];  // of a unit's tokens, by accumulator buffer; fc2: of its two K blocks
    uint32_t amax[4][kMaxTokens];
    int topk_index[kMaxTokens][kMaxTopk];
    float topk_weight[kMaxTokens][kMaxTopk];
    uint32_t mask[kMaxExperts];                // tokens of an expert
    uint32_t hit_mask[kMaxExperts];            // the same by place in the list of experts hit
    uint16_t hit[kMaxExperts];
};
constexpr size_t kSmemBytes = 1024 + size_t(kRingBytes) + sizeof(Tail);
static_assert(kSmemBytes <= 227 * 1024, "shared memory of one block");

// Pieces of the work, from the experts that are hit, fc1's and fc2's by a warp each. Approximate logarithms and quotients do: all blocks get the same.
// fc1: whole tiles, but the last ones, one per block, in parts of some eight units, three pieces per block at least, so that fc1's end is not
// waited for long. Few short tiles: in as many parts as make the longest block's share shortest, where counting and adding parts stands for
// kCountUnits units.
// fc2: the units of a tile ([expert][pair of K blocks]) in parts, each half of what would be left for a block if all were shared out
// evenly, so that the blocks end together however fast each is: what is left shrinks by a constant factor per part, down to where the parts
// have the least size, from where on they are equal. Parts are not empty: each is a unit or more before rounding. Few units: at most one group
// of equal parts, which saves the second level of sums, unless that costs more units than it stands for.
// Parts without / with regard to what counting them costs, us per call: H 1024, I 2048, 8 experts in block FP8, 5 tokens 26.1 / 23.2, 32 tokens
// 57 / 40. The same for longer tiles or parts lengthens the wait for the slowest block: 16 tokens of 128 experts (H 2048, I 768) 91 / 112,
// one token of 32 experts (H 7168, I 2048) 77.5 / 80.9; in fc2 alone from six units a block on, 4 tokens of the 128 experts 44.4 / 48.5.
constexpr int kShortUnits = 16;
constexpr int kCountUnits = 6;  // a counter, the sums and their hand-over take some 4 us, a unit 0.6
__device__ __forceinline__ void plan_pieces1(const Params& p, Tail& st, int n_hit, int lane) {
    const int tiles1 = n_hit * p.tiles1, cut = min(tiles1, p.blocks);
    const int most = max(1, min(kMaxSplit1, p.kb1 / 2));
    int split = max(1, min(max(p.kb1 / 8, int(__fdividef(float(3 * p.blocks), float(max(tiles1, 1))) + 0.999f)), most));
    if (tiles1 <= p.blocks && p.kb1 <= kShortUnits) {
        const int mine = lane + 1;  // a lane for each number of parts
        const int cost = mine <= most ? (tiles1 * mine + p.blocks - 1) / p.blocks * ((p.kb1 + mine - 1) / mine) + (mine > 1 ? kCountUnits : 0) : 0x7fffff;
        split = int(__reduce_min_sync(0xffffffffu, unsigned(cost) * 32u + lane) & 31u) + 1;
    }
    if (lane == 0) {
        st.n_hit = n_hit;
        st.whole1 = tiles1 - cut;
        st.split1 = split;
        st.pieces1 = tiles1 - cut + cut * split;
    }
}
__device__ __forceinline__ void plan_parts2(const Params& p, Tail& st, int n_hit, int lane) {
    const int units = n_hit * p.pairs2;
    const float all = float(units), log_all = __log2f(all);
    const float least = fmaxf(1.0f, fminf(4.0f, all * p.share));
    float knee = fminf(all, least * p.per_share), log_knee = __log2f(knee);
    int shrinking = knee < all ? min(kMaxShrinking, int((log_all - log_knee) * p.shrink_rate)) : 0;
    if (shrinking == 0) knee = all;
    int equal = max(1, min(kMaxParts - kMaxShrinking, int(__fdividef(knee, least))));
    const int few = min(kGroup, units), few_cost = few > 0 ? (p.tiles2 * few + p.blocks - 1) / p.blocks * ((units + few - 1) / few) : 0;
    const float even = p.even * all;  // units of a block
    if (even <= float(kCountUnits) && float(few_cost) <= even + float(kCountUnits)) {
        shrinking = 0;
        knee = all;
        equal = max(1, few);
    }
    const float step = shrinking > 0 ? __fdividef(log_knee - log_all, float(shrinking)) : 0.0f, each = __fdividef(knee, float(equal));
    for (int q = lane; q < shrinking + equal; q += 32)
        st.bound2[q] = q == 0 ? 0 : int(0.001f +  // against a whole number that came out a little less
                           (q < shrinking ? all * (1.0f - exp2f(step * float(q))) : all - each * float(shrinking + equal - q)));
    if (lane == 0) {
        st.bound2[shrinking + equal] = units;
        st.parts2 = units > 0 ? shrinking + equal : 0;
    }
}
__device__ __forceinline__ int all_pieces(const Params& p, const Tail& st) { return st.pieces1 + st.parts2 * p.tiles2; }

struct Piece {
    int phase;       // 0 fc1, 1 fc2, 2 no more, 3 a wait has run out
    int tile, part;  // fc1: tile = expert's place * tiles1 + tile of I, part -1 for all of it; fc2: tile of H
    int lo, hi;      // units of the tile
};
__device__ __forceinline__ Piece piece_at(const Params& p, const Tail& st, int c) {
    Piece q;
    if (c >= all_pieces(p, st)) return Piece{2, 0, 0, 0, 0};
    if (c < st.pieces1) {
        q.phase = 0;
        const int cut = c - st.whole1;
        if (cut < 0) {
            q.tile = c, q.part = -1;
            q.lo = 0, q.hi = p.kb1;
        } else {
            const int tile = cut / st.split1;
            q.tile = st.whole1 + tile, q.part = cut - tile * st.split1;
            q.lo = q.part * p.kb1 / st.split1, q.hi = (q.part + 1) * p.kb1 / st.split1;
        }
    } else {
        q.phase = 1;
        q.part = (c - st.pieces1) / p.tiles2;
        q.tile = c - st.pieces1 - q.part * p.tiles2;
        q.lo = st.bound2[q.part];
        q.hi = st.bound2[q.part + 1];
    }
    return q;
}

// Where the sums of an fc1 piece stand: places that a block uses in turn, or one for each part of a split tile.
template <size_t kFloats>
__device__ __forceinline__ float* place1(const Params& p, const Tail& st, const Piece& q, int slot) {
    const size_t at = q.part < 0 ? size_t(blockIdx.x) * kJobs + slot : size_t(p.blocks) * kJobs + size_t(q.tile - st.whole1) * st.split1 + q.part;
    return p.part1 + at * kFloats;
}

// The next piece, as the weights' thread announces it to the other roles.
template <bool kWarp>
__device__ __forceinline__ Piece next_piece(const Params& p, Tail& st, int it, int lane, int* code = nullptr) {
    const int slot = it % kClaims, parity = (it / kClaims) & 1;
    const bool ok = kWarp ? ptx::mbar_wait_warp(&st.claim_full[slot], parity, &st.abort_flag, p.wait_limit)
                          : ptx::mbar_wait(&st.claim_full[slot], parity, &st.abort_flag, p.wait_limit);
    if (!ok) return Piece{3, 0, 0, 0, 0};
    const int c = *const_cast<volatile int*>(&st.claim[slot]);
    if constexpr (kWarp) __syncwarp();
    if (!kWarp || lane == 0) ptx::mbar_arrive(&st.claim_empty[slot]);
    if (code != nullptr) *code = c;
    return piece_at(p, st, c);
}

template <bool kFp8, int kTp>
struct Shape {
    static constexpr int kN1 = fc1_cols(kFp8, kTp), kN2 = fc2_cols(kTp);
    static constexpr int kKElems = kFp8 ? kKBytes : kKBytes / 2;
    static constexpr int kStages = stages(kTp);
    static constexpr int kStage = stage_bytes(kTp);
    // FP8: the accumulators of one unit per buffer, handed over unit by unit; bf16: those of one piece and expert
    static constexpr int kBufCols = kFp8 ? 2 * kN1 : (2 * kN1 > kN2 ? 2 * kN1 : kN2);
    static constexpr int kBufs = kFp8 ? 4 : 2;
    static constexpr int kTmemCols = kBufs * kBufCols;  // 128 / 256 / 512 and 64 / 64 / 128
    static_assert((kTmemCols & (kTmemCols - 1)) == 0 && kTmemCols >= 32 && kTmemCols <= 512, "TMEM allocation");
    static constexpr int kDrainTokens = kTp > 16 ? 16 : kTp;  // of four draining warps
    static constexpr int kDrainWarps = 4 * kTp / kDrainTokens;
    static constexpr size_t kPart1 = size_t(2) * kTp * kRows, kPart2 = size_t(kTp) * kRows;  // floats
};

template <bool kFp8, int kTp>
__device__ __forceinline__ void load_weights(const Params& p, const CUtensorMap& map_b, const CUtensorMap& map_b1, Tail& st, uint8_t* ring, int claim) {
    using S = Shape<kFp8, kTp>;
    int it = 0;
    bool ok = true;
    for (int n = 0; ok; ++n) {
        const int slot = n % kClaims;
        const int next = claim < all_pieces(p, st) ? atomicAdd(&p.counters[0], 1) : claim;  // known by the time it is needed
        if (!(ok = ptx::mbar_wait(&st.claim_empty[slot], ((n / kClaims) & 1) ^ 1, &st.abort_flag, p.wait_limit))) break;
        *const_cast<volatile int*>(&st.claim[slot]) = claim;
        ptx::mbar_arrive(&st.claim_full[slot]);
        const Piece q = piece_at(p, st, claim);
        if (q.phase == 2) break;
        for (int u = q.lo; u < q.hi; ++u, ++it) {
            const int s = it % S::kStages;
            if (!(ok = ptx::mbar_wait(&st.empty[s], ((it / S::kStages) & 1) ^ 1, &st.abort_flag, p.wait_limit))) break;
            uint8_t* a = ring + s * S::kStage;
            ptx::mbar_arrive_expect_tx(&st.full[s], kABytes);
            if (q.phase == 0) {
                const int j = q.tile / p.tiles1, row = st.hit[j] * 2 * p.I + (q.tile - j * p.tiles1) * kRows;
                ptx::tma_load_2d(a, &map_b, u * S::kKElems, row, &st.full[s]);
                ptx::tma_load_2d(a + kTileBytes, &map_b, u * S::kKElems, row + p.I, &st.full[s]);
            } else {
                const int j = u / p.pairs2, pair = u - j * p.pairs2, row = st.hit[j] * p.H + q.tile * kRows;
                // a last pair's second block may lie past I, where the copy writes zeros
                ptx::tma_load_2d(a, &map_b1, pair * 2 * S::kKElems, row, &st.full[s]);
                ptx::tma_load_2d(a + kTileBytes, &map_b1, (pair * 2 + 1) * S::kKElems, row, &st.full[s]);
            }
        }
        claim = next;
    }
}

template <bool kFp8, int kTp>
__device__ __forceinline__ void load_tokens(const Params& p, Tail& st, uint8_t* ring) {
    using S = Shape<kFp8, kTp>;
    int it = 0, ready = -1;  // place of the expert whose fc1 was last seen finished
    bool ok = true;
    for (int n = 0; ok; ++n) {
        const Piece q = next_piece<false>(p, st, n, 0);
        if (q.phase >= 2) break;
        for (int u = q.lo; u < q.hi; ++u, ++it) {
            const int s = it % S::kStages;
            if (!(ok = ptx::mbar_wait(&st.empty[s], ((it / S::kStages) & 1) ^ 1, &st.abort_flag, p.wait_limit))) break;
            uint8_t* b = ring + s * S::kStage + kABytes;
            if (q.phase == 0) {
                ptx::mbar_arrive_expect_tx(&st.full[s], uint32_t(p.rec1));
                ptx::bulk_load(b, p.xq + size_t(u) * p.rec1, uint32_t(p.rec1), &st.full[s]);
                continue;
            }
            const int j = u / p.pairs2;
            if (j != ready) {
                const long long t0 = clock64();
                while (streamk::ld_acquire_gpu(&p.counters[1 + j]) < p.tiles1) {
                    if (*const_cast<volatile int*>(&st.abort_flag) != 0) ok = false;
                    if (clock64() - t0 > p.wait_limit) {
                        *const_cast<volatile int*>(&st.abort_flag) = 1;
                        *p.status = kStatusPhase;
                        ok = false;
                    }
                    if (!ok) break;
                }
                if (!ok) break;
                asm volatile("fence.proxy.async;" ::: "memory");
                ready = j;
            }
            ptx::mbar_arrive_expect_tx(&st.full[s], uint32_t(p.rec2));
            ptx::bulk_load(b, p.aq + size_t(u) * p.rec2, uint32_t(p.rec2), &st.full[s]);  // [expert][pair], as the units
        }
    }
}

// The MMAs of every unit, issued by one thread; by the whole warp because it also takes the scales of a unit's tokens out of its stage (FP8), to stand
// beside the accumulators that they belong to: so the stage is free when the MMAs have read it, not when the accumulators have been drained.
template <bool kFp8, int kTp>
__device__ __forceinline__ void multiply(const Params& p, Tail& st, uint8_t* ring, uint32_t tmem, int lane) {
    using S = Shape<kFp8, kTp>;
    constexpr int kKind = kFp8 ? 0 : 1;
    constexpr uint32_t kFormat = kFp8 ? 0 : 1;
    constexpr uint32_t kId1 = ptx::make_idesc(kFormat, kRows, S::kN1), kId2 = ptx::make_idesc(kFormat, kRows, S::kN2);
    int it = 0, buf_it = 0;
    for (int n = 0;; ++n) {
        const Piece q = next_piece<true>(p, st, n, lane);
        if (q.phase >= 2) return;
        bool fresh = true;  // the next unit begins an accumulator buffer
        for (int u = q.lo; u < q.hi; ++u, ++it) {
            const int slot = it % S::kStages, buf = buf_it % S::kBufs;
            if (fresh && !ptx::mbar_wait_warp(&st.tmem_empty[buf], ((buf_it / S::kBufs) & 1) ^ 1, &st.abort_flag, p.wait_limit)) return;
            if (!ptx::mbar_wait_warp(&st.full[slot], (it / S::kStages) & 1, &st.abort_flag, p.wait_limit)) return;
            ptx::tc_fence_after();
            const bool done = kFp8 || u + 1 == q.hi || (q.phase == 1 && (u + 1) % p.pairs2 == 0);
            if (ptx::elect_one()) {
                const uint32_t a = ptx::smem_u32(ring + slot * S::kStage);
                const uint64_t da = ptx::smem_desc_sw128(a), db = ptx::smem_desc_sw128(a + kABytes);
                const uint32_t d = tmem + buf * S::kBufCols;
#pragma unroll
                for (int half = 0; half < 2; ++half)
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const uint64_t ak = ptx::smem_desc_advance(da, half * kTileBytes + k * 32);
                        if (q.phase == 0)  // gate rows, value rows
                            ptx::umma<kKind>(d + half * S::kN1, ak, ptx::smem_desc_advance(db, k * 32), kId1, (!kFp8 && !fresh) || k > 0);
                        else               // two K blocks: with their own scales in FP8, one sum in bf16
                            ptx::umma<kKind>(d + (kFp8 ? half * S::kN2 : 0), ak, ptx::smem_desc_advance(db, half * S::kN2 * kKBytes + k * 32), kId2,
                                             (!kFp8 && (!fresh || half > 0)) || k > 0);
                    }
                ptx::umma_commit(&st.empty[slot]);
                if (done) ptx::umma_commit(&st.tmem_full[buf]);
            }
            __syncwarp();
            if constexpr (kFp8) {
                const float* from = reinterpret_cast<const float*>(ring + slot * S::kStage + kABytes + (q.phase == 0 ? S::kN1 : 2 * S::kN2) * kKBytes);
                if (lane < kTp) {
                    st.token_scale[buf][lane] = from[lane];
                    if (q.phase == 1) st.token_scale[buf][kTp + lane] = from[kTp + lane];
                }
                __syncwarp();
                if (lane == 0) {
                    ptx::mbar_arrive(&st.empty[slot]);
                    ptx::mbar_arrive(&st.tmem_full[buf]);
                }
            }
            if (done) ++buf_it;
            fresh = done;
        }
    }
}

// Scale of a weight row in a unit: constant over the weights (bf16: 1), an expert, a row, or a 128x128 block.
__device__ __forceinline__ float weight_scale(const float* scale, int mode, int e, int rows, int row, int blocks_k, int kb) {
    if (mode == DQMOE_QUANT_FP8_BLOCK) return scale[(size_t(e) * ((rows + 127) / 128) + row / 128) * blocks_k + kb];
    if (mode == DQMOE_QUANT_FP8_CHANNEL) return scale[size_t(e) * rows + row];
    return mode == DQMOE_QUANT_FP8_TENSOR ? scale[e] : 1.0f;
}

__device__ __forceinline__ uint32_t all_tokens(const Params& p) { return p.T == 32 ? 0xffffffffu : (1u << p.T) - 1u; }
// Sums of the tokens of `mask` (and some beside them) of a weight row.
template <int kTp>
__device__ __forceinline__ void put_sums(float* to, int row, uint32_t mask, const float (&sum)[kTp]) {
#pragma unroll
    for (int t = 0; t < kTp; t += 4)
        if ((mask >> t) & 15u) *reinterpret_cast<float4*>(to + t * kRows + row * 4) = make_float4(sum[t], sum[t + 1], sum[t + 2], sum[t + 3]);
}
// Two fp32 values in a register pair, and their FMA in one instruction.
__device__ __forceinline__ uint64_t two(float lo, float hi) {
    uint64_t v;
    asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(lo), "f"(hi));
    return v;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t v;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(v) : "l"(a), "l"(b), "l"(c));
    return v;
}
// Accumulators to scaled sums of a piece, which go to the piece's place in the workspace.
template <bool kFp8, int kTp>
struct Drain {
    using S = Shape<kFp8, kTp>;
    static constexpr int kCols = S::kDrainTokens;
    const Params& p;
    Tail& st;
    uint32_t tmem;
    int warp, lane, row;  // row = TMEM lane = weight row of the tile
    int t0;               // first of this warp's tokens
    int buf_it = 0;

    __device__ __forceinline__ bool acquire() {
        const int buf = buf_it % S::kBufs;
        if (!ptx::mbar_wait_warp(&st.tmem_full[buf], (buf_it / S::kBufs) & 1, &st.abort_flag, p.wait_limit)) return false;
        ptx::tc_fence_after();
        return true;
    }
    __device__ __forceinline__ void release() {
        ptx::tc_fence_before();
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(&st.tmem_empty[buf_it % S::kBufs]);
        ++buf_it;
    }
    __device__ __forceinline__ const float* token_scale() const { return st.token_scale[buf_it % S::kBufs] + t0; }
    // columns of this warp's first token
    __device__ __forceinline__ uint32_t buffer() const { return tmem + (buf_it % S::kBufs) * S::kBufCols + t0; }

    // sum += (hi + lo / 16) * scale, of the tokens of `mask` where the others' columns may hold what is no number
    template <bool kMasked>
    __device__ __forceinline__ void add_scaled(uint32_t taddr, const float* token_scale, float row_scale, uint32_t mask, float (&sum)[kCols]) {
        float hi[kCols], lo[kCols];
        ptx::tmem_read2<kCols>(taddr, taddr + kTp, hi, lo);
        const uint64_t row2 = two(row_scale, row_scale), sixteenth = two(0.0625f, 0.0625f);
#pragma unroll
        for (int t = 0; t < kCols; t += 4) {
            const float4 sc = *reinterpret_cast<const float4*>(token_scale + t);
#pragma unroll
            for (int i = 0; i < 4; i += 2) {
                const uint64_t scale = fma2(i == 0 ? two(sc.x, sc.y) : two(sc.z, sc.w), row2, 0);
                const uint64_t x = fma2(two(lo[t + i], lo[t + i + 1]), sixteenth, two(hi[t + i], hi[t + i + 1]));
                const uint64_t v = fma2(x, scale, two(sum[t + i], sum[t + i + 1]));
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    if (!kMasked || ((mask >> (t + i + h)) & 1u)) sum[t + i + h] = __uint_as_float(uint32_t(v >> (32 * h)));
            }
        }
    }

    __device__ __forceinline__ bool fc1(const Piece& q, float* to) {
        const int j = q.tile / p.tiles1, e = st.hit[j], i = min((q.tile - j * p.tiles1) * kRows + row, p.I - 1);
        const uint32_t mask = (st.hit_mask[j] >> t0) & ((1u << kCols) - 1u);  // the sums of other tokens are not used
        float g[kCols], v[kCols];
        if constexpr (kFp8) {
#pragma unroll
            for (int t = 0; t < kCols; ++t) g[t] = v[t] = 0.0f;
            float sg = weight_scale(p.b_scale, p.mode, e, 2 * p.I, i, p.kb1, q.lo);
            float sv = weight_scale(p.b_scale, p.mode, e, 2 * p.I, p.I + i, p.kb1, q.lo);
            for (int kb = q.lo; kb < q.hi; ++kb) {
                const float gs = sg, vs = sv;
                if (kb + 1 < q.hi) {  // the next unit's, while this one's MMAs are on their way
                    sg = weight_scale(p.b_scale, p.mode, e, 2 * p.I, i, p.kb1, kb + 1);
                    sv = weight_scale(p.b_scale, p.mode, e, 2 * p.I, p.I + i, p.kb1, kb + 1);
                }
                if (!acquire()) return false;
                if (mask != 0) {
                    add_scaled<false>(buffer(), token_scale(), gs, mask, g);
                    add_scaled<false>(buffer() + S::kN1, token_scale(), vs, mask, v);
                }
                release();
            }
        } else {
            if (!acquire()) return false;
            ptx::tmem_read2<kCols>(buffer(), buffer() + S::kN1, g, v);
            release();
        }
        put_sums<kCols>(to + t0 * kRows, row, mask, g);
        put_sums<kCols>(to + (kTp + t0) * kRows, row, mask, v);
        return true;
    }

    __device__ __forceinline__ bool fc2(const Piece& q, float* to) {
        const int kb2 = (p.I + S::kKElems - 1) / S::kKElems;
        const int h = min(q.tile * kRows + row, p.H - 1);
        float sum[kCols];
#pragma unroll
        for (int t = 0; t < kCols; ++t) sum[t] = 0.0f;
        if constexpr (kFp8) {
            auto scale_of = [&](int u, int half) {
                const int j = u / p.pairs2, kb = (u - j * p.pairs2) * 2 + half;
                return kb < kb2 ? weight_scale(p.b1_scale, p.mode, st.hit[j], p.H, h, kb2, kb) : 0.0f;
            };
            float next0 = 0.0f, next1 = 0.0f;
            if (q.lo < q.hi) next0 = scale_of(q.lo, 0), next1 = scale_of(q.lo, 1);
            for (int u = q.lo; u < q.hi; ++u) {
                const int j = u / p.pairs2, kb = (u - j * p.pairs2) * 2;
                const float s0 = next0, s1 = next1;
                if (u + 1 < q.hi) next0 = scale_of(u + 1, 0), next1 = scale_of(u + 1, 1);
                const uint32_t mask = (st.hit_mask[j] >> t0) & ((1u << kCols) - 1u);
                if (!acquire()) return false;
                if (mask != 0) {
                    add_scaled<true>(buffer(), token_scale(), s0, mask, sum);
                    if (kb + 1 < kb2) add_scaled<true>(buffer() + S::kN2, token_scale() + kTp, s1, mask, sum);  // nothing was laid out past I
                }
                release();
            }
        } else {
            for (int u = q.lo; u < q.hi;) {  // expert by expert: only the tokens that chose it take part
                const int j = u / p.pairs2;
                u = min(q.hi, (j + 1) * p.pairs2);
                if (!acquire()) return false;
                float hi[kCols], lo[kCols];
                ptx::tmem_read2<kCols>(buffer(), buffer() + kTp, hi, lo);
                release();
                const uint32_t mask = st.hit_mask[j] >> t0;
#pragma unroll
                for (int t = 0; t < kCols; ++t)
                    if ((mask >> t) & 1u) sum[t] += hi[t] + lo[t];
            }
        }
        put_sums<kCols>(to + t0 * kRows, row, all_tokens(p) >> t0, sum);
        return true;
    }

    __device__ __forceinline__ void run() {
        for (int n = 0;; ++n) {
            int code = 0;
            const Piece q = next_piece<true>(p, st, n, lane, &code);
            // the finishing warps are through with what used this note, and this place for a tile in one part, before
            const int slot = n % kJobs;
            if (q.phase == 3 || !ptx::mbar_wait_warp(&st.job_empty[slot], ((n / kJobs) & 1) ^ 1, &st.abort_flag, p.wait_limit)) return;
            if (q.phase == 0) {
                if (!fc1(q, place1<S::kPart1>(p, st, q, slot))) return;
            } else if (q.phase == 1) {
                if (!fc2(q, p.part2 + (size_t(q.tile) * kMaxParts + q.part) * S::kPart2)) return;
            }
            if (warp == 0 && lane == 0) *const_cast<volatile int*>(&st.job[slot]) = code;
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive(&st.job_full[slot]);
            if (q.phase == 2) return;
        }
    }
};

// Counts the pieces in whose sums are written, and passes those on that complete a tile of fc1 or a group of parts of fc2. A counter takes
// some trips through L2 (2-5 thousand cycles while the weights stream), which nobody else has to wait for.
__device__ __forceinline__ void count_pieces(const Params& p, Tail& st) {
    int passed = 0;
    for (int n = 0;; ++n) {
        const int slot = n % kJobs;
        if (!ptx::mbar_wait(&st.job_full[slot], (n / kJobs) & 1, &st.abort_flag, p.wait_limit)) return;
        const int code = *const_cast<volatile int*>(&st.job[slot]);
        const Piece q = piece_at(p, st, code);
        bool last = true;
        if (q.phase == 0 && q.part >= 0 && st.split1 > 1) {
            last = streamk::atomic_add_acq_rel_gpu(&p.counters[1 + p.max_hit + q.tile], 1) == st.split1 - 1;
        } else if (q.phase == 1) {
            const int group = q.part / kGroup, in_group = min(kGroup, st.parts2 - group * kGroup);
            int* counters = p.counters + 1 + p.max_hit + p.max_hit * p.tiles1;
            if (in_group > 1) last = streamk::atomic_add_acq_rel_gpu(&counters[q.tile * kGroups + group], 1) == in_group - 1;
        }
        if (last) {  // at most kJobs of them are under way, each with its slot of `job`
            *const_cast<volatile int*>(&st.last_job[passed % kJobs]) = code * kJobs + slot;
            ptx::mbar_arrive(&st.last_full[passed % kJobs]);
            ++passed;
        } else {
            for (int i = 0; i < 4; ++i) ptx::mbar_arrive(&st.job_empty[slot]);
        }
        if (q.phase == 2) return;
    }
}

// Sums over the parts of a tile; fc1: the activation, laid out as fc2's second operand; fc2: the output. Eight tokens at a time in a loop:
// unrolled over 32 tokens, of which a tile has two or three, this was 77 KB of code, whose fetches through a busy L2 took up to 69000 cycles
// a tile.
template <bool kFp8, int kTp>
struct Finish {
    using S = Shape<kFp8, kTp>;
    const Params& p;
    Tail& st;
    int warp, lane, row;
    uint32_t meetings = 0;

    // The finishing warps wait for one another at an mbarrier, whose wait ends also where one of them has given up.
    __device__ __forceinline__ bool meet() {
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(&st.meet);
        return ptx::mbar_wait_warp(&st.meet, meetings++ & 1, &st.abort_flag, p.wait_limit);
    }

    // Weight of token t for the expert e (routed ids only), by all lanes together.
    __device__ __forceinline__ float weight_of(int t, int e) const {
        const bool mine = lane < p.k && st.topk_index[t][lane] == e;
        const uint32_t who = __ballot_sync(0xffffffffu, mine);
        return who == 0 ? 1.0f : st.topk_weight[t][__ffs(who) - 1];  // shared experts are not in the list
    }

    // sum of `parts` parts in their order for tokens t0 .. t0 + 7, those of `mask8`; all loads of kAtOnce parts before the first use
    template <int kAtOnce>
    __device__ __forceinline__ void add_parts(const float* part, int parts, size_t stride, int t0, uint32_t mask8, float (&sum)[8]) const {
#pragma unroll
        for (int i = 0; i < 8; ++i) sum[i] = 0.0f;
        float4 v[kAtOnce][2];
#pragma unroll
        for (int o = 0; o < kAtOnce; ++o)
#pragma unroll
            for (int h = 0; h < 2; ++h)
                v[o][h] = o < parts && ((mask8 >> (4 * h)) & 15u) != 0 ? streamk::ld_partial4(part + o * stride + (t0 + 4 * h) * kRows + row * 4)
                                                                        : make_float4(0, 0, 0, 0);
#pragma unroll
        for (int o = 0; o < kAtOnce; ++o)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                sum[4 * h] += v[o][h].x, sum[4 * h + 1] += v[o][h].y;
                sum[4 * h + 2] += v[o][h].z, sum[4 * h + 3] += v[o][h].w;
            }
    }

    __device__ __forceinline__ bool fc1(const Piece& q, const float* part) {
        const int parts = q.part < 0 ? 1 : st.split1;
        const int j = q.tile / p.tiles1, tile = q.tile - j * p.tiles1, e = st.hit[j];
        if (q.part > 0) part -= q.part * S::kPart1;
        const bool inside = tile * kRows + row < p.I;
        uint8_t* rec = p.aq + (size_t(j) * p.pairs2 + (kFp8 ? tile >> 1 : tile)) * p.rec2;
#pragma unroll 1
        for (int t0 = 0; t0 < kTp; t0 += 8) {
            const uint32_t mask8 = (st.hit_mask[j] >> t0) & 255u;  // the same for all threads
            if (mask8 == 0) continue;
            float g[8], v[8];
            add_parts<kMaxSplit1>(part, parts, S::kPart1, t0, mask8, g);
            add_parts<kMaxSplit1>(part + kTp * kRows, parts, S::kPart1, t0, mask8, v);
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if ((mask8 >> i) & 1u) {
                    const float w = weight_of(t0 + i, e);  // all lanes, also those of rows past I
                    g[i] = inside ? w * (silu_approx(g[i]) * v[i]) : 0.0f;
                    if constexpr (kFp8) {
                        const uint32_t most = __reduce_max_sync(0xffffffffu, __float_as_uint(g[i]) & 0x7fffffffu);
                        if (lane == 0) st.amax[warp][t0 + i] = most;
                    }
                }
            if constexpr (kFp8) {
                if (!meet()) return false;
                uint8_t* data = rec + (tile & 1) * S::kN2 * kKBytes;
                float* scales = reinterpret_cast<float*>(rec + 2 * S::kN2 * kKBytes) + (tile & 1) * kTp;
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if ((mask8 >> i) & 1u) {
                        const int t = t0 + i;
                        float inv;
                        const float s = split_scale(max(max(st.amax[0][t], st.amax[1][t]), max(st.amax[2][t], st.amax[3][t])), &inv);
                        uint32_t hi, lo;
                        split_e4m3x2(g[i] * inv, 0.0f, &hi, &lo);
                        data[swizzled(t, row)] = uint8_t(hi);
                        data[swizzled(kTp + t, row)] = uint8_t(lo);
                        if (row == 0) scales[t] = s;
                    }
            } else {
                uint8_t* data = rec + (row >> 6) * S::kN2 * kKBytes;
                const int byte = (row & 63) * 2;
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if ((mask8 >> i) & 1u) {
                        const uint32_t hi = f2bf_bits(g[i]);
                        const float rest = g[i] - __uint_as_float(hi << 16);
                        // an infinite value has no rest
                        const uint32_t lo = (hi & 0x7fffu) < 0x7f80u ? f2bf_bits(rest) : 0u;
                        *reinterpret_cast<uint16_t*>(data + swizzled(t0 + i, byte)) = uint16_t(hi);
                        *reinterpret_cast<uint16_t*>(data + swizzled(kTp + t0 + i, byte)) = uint16_t(lo);
                    }
            }
        }
        asm volatile("fence.proxy.async;" ::: "memory");  // to the bulk copies of other blocks
        if (!meet()) return false;
        if (warp == 0 && lane == 0) streamk::red_add_release_gpu(&p.counters[1 + j], 1);
        return true;
    }

    __device__ __forceinline__ bool fc2(const Piece& q) {
        const int group = q.part / kGroup, groups = (st.parts2 + kGroup - 1) / kGroup, in_group = min(kGroup, st.parts2 - group * kGroup);
        const uint32_t all = all_tokens(p), bad = st.bad_tokens;
        const int h = q.tile * kRows + row;
        float* group_sums = p.group2 + size_t(q.tile) * kGroups * S::kPart2;
        auto put_out = [&](int t0, const float (&sum)[8]) {
            if (h < p.H) {
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (t0 + i < p.T) p.out[size_t(t0 + i) * p.H + h] = __float2bfloat16_rn((bad >> (t0 + i)) & 1u ? __uint_as_float(0x7fffffffu) : sum[i]);
            }
        };
#pragma unroll 1
        for (int t0 = 0; t0 < p.T; t0 += 8) {
            float sum[8];
            add_parts<kGroup>(p.part2 + (size_t(q.tile) * kMaxParts + group * kGroup) * S::kPart2, in_group, S::kPart2, t0, (all >> t0) & 255u, sum);
            if (groups == 1) put_out(t0, sum);
            else put_sums<8>(group_sums + group * S::kPart2 + t0 * kRows, row, 255u, sum);
        }
        if (groups == 1) return true;
        if (!meet()) return false;
        if (warp == 0 && lane == 0)
            st.last = streamk::atomic_add_acq_rel_gpu(p.counters + 1 + p.max_hit + p.max_hit * p.tiles1 + p.tiles2 * kGroups + q.tile, 1) == groups - 1;
        if (!meet()) return false;
        if (*const_cast<volatile int*>(&st.last) == 0) return true;  // read by all before they meet for the next job's
#pragma unroll 1
        for (int t0 = 0; t0 < p.T; t0 += 8) {
            float sum[8];
            add_parts<kGroups>(group_sums, groups, S::kPart2, t0, (all >> t0) & 255u, sum);
            put_out(t0, sum);
        }
        return true;
    }

    __device__ __forceinline__ void run() {
        for (int n = 0;; ++n) {
            if (!ptx::mbar_wait_warp(&st.last_full[n % kJobs], (n / kJobs) & 1, &st.abort_flag, p.wait_limit)) return;
            const int note = *const_cast<volatile int*>(&st.last_job[n % kJobs]), slot = note % kJobs;
            const Piece q = piece_at(p, st, note / kJobs);
            if (q.phase == 2) return;
            if (!(q.phase == 0 ? fc1(q, place1<S::kPart1>(p, st, q, slot)) : fc2(q))) return;
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive(&st.job_empty[slot]);
        }
    }
};

// Chosen experts of every token into shared memory, and the list of experts that any token chose, shared ones at its end.
template <int kPerLane>
__device__ __forceinline__ void choose_topk(const Params& p, Tail& st, int warp, int lane) {
    for (int t = warp; t < p.T; t += int(blockDim.x >> 5)) {
        int* index = st.topk_index[t];
        float* weight = st.topk_weight[t];
        route::topk_of_token<kPerLane>(p.logits + size_t(t) * p.E, p.E, p.k, p.k, p.scoring, lane, index, weight);
        __syncwarp();
        if (lane < p.k) {
            if (index[lane] < p.E) atomicOr(&st.mask[index[lane]], 1u << t);
            if (isnan(weight[lane])) atomicOr(&st.bad_tokens, 1u << t);
        }
    }
}
__device__ __forceinline__ void choose(const Params& p, Tail& st, int warp, int lane) {
    if (p.E <= 32) choose_topk<1>(p, st, warp, lane);
    else if (p.E <= 128) choose_topk<4>(p, st, warp, lane);
    else if (p.E <= 256) choose_topk<8>(p, st, warp, lane);
    else choose_topk<32>(p, st, warp, lane);
    __syncthreads();
    if (warp < 2) {  // each for its part of the plan: one after the other they took 2 us
        int count = 0;
        for (int e0 = 0; e0 < p.E; e0 += 32) {
            const uint32_t m = e0 + lane < p.E ? st.mask[e0 + lane] : 0u;
            const uint32_t hits = __ballot_sync(0xffffffffu, m != 0);
            if (warp == 0 && m != 0) {
                const int at = count + __popc(hits & ((1u << lane) - 1u));
                st.hit[at] = uint16_t(e0 + lane);
                st.hit_mask[at] = m;
            }
            count += __popc(hits);
        }
        if (warp == 0) {
            for (int i = lane; i < p.n_shared; i += 32) {
                st.hit[count + i] = uint16_t(p.E + i);
                st.hit_mask[count + i] = all_tokens(p);
            }
            plan_pieces1(p, st, count + p.n_shared, lane);
        } else {
            plan_parts2(p, st, count + p.n_shared, lane);
        }
    }
}

template <bool kFp8, int kTp>
__global__ void __launch_bounds__(threads(kTp), 1)
moe_decode_experts_kernel(const __grid_constant__ CUtensorMap map_b, const __grid_constant__ CUtensorMap map_b1, const __grid_constant__ Params p) {
    using S = Shape<kFp8, kTp>;
    pdl_launch();
    extern __shared__ uint8_t smem_raw[];
    uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    Tail& st = *reinterpret_cast<Tail*>(ring + kRingBytes);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        for (int i = 0; i < S::kStages; ++i) {
            ptx::mbar_init(&st.full[i], 2);              // weights, tokens
            ptx::mbar_init(&st.empty[i], kFp8 ? 2 : 1);  // the tensor core's reads, and the MMA warp's of the scales
        }
        for (int i = 0; i < 4; ++i) {
            ptx::mbar_init(&st.tmem_full[i], kFp8 ? 2 : 1);  // the MMAs, and the scales
            ptx::mbar_init(&st.tmem_empty[i], S::kDrainWarps);
        }
        for (int i = 0; i < kClaims; ++i) {
            ptx::mbar_init(&st.claim_full[i], 1);
            ptx::mbar_init(&st.claim_empty[i], 2 + S::kDrainWarps);  // tokens, MMA, draining warps
        }
        for (int i = 0; i < kJobs; ++i) {
            ptx::mbar_init(&st.job_full[i], S::kDrainWarps);
            ptx::mbar_init(&st.job_empty[i], 4);   // the finishing warps, or the counting thread for them
            ptx::mbar_init(&st.last_full[i], 1);
        }
        ptx::mbar_init(&st.meet, 4);
        st.abort_flag = 0;
        ptx::fence_barrier_init();
    }
    if (warp == 1) {
        ptx::tmem_alloc(&st.tmem_base, S::kTmemCols);
        ptx::tmem_relinquish();
    }
    for (int i = threadIdx.x; i < p.E; i += threads(kTp)) st.mask[i] = 0;
    if (threadIdx.x == 0) st.bad_tokens = 0;
    ptx::tc_fence_before();
    __syncthreads();
    ptx::tc_fence_after();
    if (threadIdx.x == 32 * 2) ptx::prefetch_tensormap(&map_b);
    if (threadIdx.x == 32 * 3) ptx::prefetch_tensormap(&map_b1);
    pdl_wait();
    int claim = 0;
    if (threadIdx.x == 0) claim = atomicAdd(&p.counters[0], 1);  // looked at behind the choice, which does not need it
    choose(p, st, warp, lane);
    __syncthreads();
    if (warp == 0) claim = __shfl_sync(0xffffffffu, claim, 0);
    const uint32_t tmem = *const_cast<volatile uint32_t*>(&st.tmem_base);

    if (st.n_hit == 0) {  // no token has an expert
        for (int i = blockIdx.x * threads(kTp) + threadIdx.x; i < p.T * p.H; i += gridDim.x * threads(kTp))
            p.out[i] = __float2bfloat16_rn((st.bad_tokens >> (i / p.H)) & 1u ? __uint_as_float(0x7fffffffu) : 0.0f);
    } else if (warp == 0) {
        if (ptx::elect_one()) load_weights<kFp8, kTp>(p, map_b, map_b1, st, ring, claim);
        __syncwarp();
    } else if (warp == 1) {
        multiply<kFp8, kTp>(p, st, ring, tmem, lane);
    } else if (warp == 2) {
        if (ptx::elect_one()) load_tokens<kFp8, kTp>(p, st, ring);
        __syncwarp();
    } else if (warp == 3) {
        if (ptx::elect_one()) count_pieces(p, st);
        __syncwarp();
    } else if (warp >= 8 && warp < 12) {
        Finish<kFp8, kTp> f{p, st, warp - 8, lane, (warp - 8) * 32 + lane};
        f.run();
    } else if (warp >= 4) {
        const int quarter = warp & 3;  // of TMEM's lanes, that a warp may read
        Drain<kFp8, kTp> d{p, st, tmem + (uint32_t(quarter * 32) << 16), warp - 4, lane, quarter * 32 + lane, warp >= 12 ? 16 : 0};
        d.run();
    }
    ptx::settle_after_abort(&st.abort_flag);
    __syncthreads();
    if (threadIdx.x == 0 && st.abort_flag != 0 && *const_cast<volatile int*>(p.status) == 0) *p.status = kStatusRing;
    if (warp == 1) {
        ptx::tc_fence_after();
        ptx::tmem_dealloc(tmem, S::kTmemCols);
    }
}

// ---------------------------------------------------------------- host

struct Layout {
    size_t counters, logits, xq, aq, part1, part2, group2, total;
};
static Layout plan(Params* p, bool fp8) {
    const int tp = token_rows(p->T);
    const int ke = fp8 ? 128 : 64;
    p->max_hit = (p->T * p->k < p->E ? p->T * p->k : p->E) + p->n_shared;
    p->kb1 = ceil_div(p->H, ke);
    p->pairs2 = ceil_div(ceil_div(p->I, ke), 2);
    p->tiles1 = ceil_div(p->I, kRows);
    p->tiles2 = ceil_div(p->H, kRows);
    p->rec1 = size_t(fc1_cols(fp8, tp)) * kKBytes + (fp8 ? size_t(tp) * sizeof(float) : 0);
    p->rec2 = size_t(2) * fc2_cols(tp) * kKBytes + (fp8 ? size_t(2) * tp * sizeof(float) : 0);
    p->blocks = sm_count();
    p->even = float(p->tiles2) / float(p->blocks);
    p->share = p->even < 1.0f ? 0.5f * p->even : 0.5f;  // of what is left, per part
    p->per_share = 1.0f / p->share;
    p->shrink_rate = -1.0f / log2f(1.0f - p->share);
    p->n_counters = 1 + p->max_hit + p->max_hit * p->tiles1 + p->tiles2 * (kGroups + 1);
    Layout L{};
    size_t off = 0;
    auto add = [&](size_t bytes) {
        const size_t at = off;
        off += align_up(bytes, 256);
        return at;
    };
    L.counters = add(size_t(p->n_counters) * sizeof(int));
    L.logits = add(size_t(p->T) * p->E * sizeof(float));
    L.xq = add(size_t(p->kb1) * p->rec1);
    L.aq = add(size_t(p->max_hit) * p->pairs2 * p->rec2);
    L.part1 = add(size_t(p->blocks) * (kJobs + kMaxSplit1) * 2 * tp * kRows * sizeof(float));
    L.part2 = add(size_t(p->tiles2) * kMaxParts * tp * kRows * sizeof(float));
    L.group2 = add(size_t(p->tiles2) * kGroups * tp * kRows * sizeof(float));
    L.total = off;
    return L;
}

static int check_sizes(int T, int H, int I, int E, int k, int n_shared, int quant_mode) {
    DQ_CHECK_FMT(quant_mode == DQMOE_QUANT_NONE || quant_mode == DQMOE_QUANT_FP8_TENSOR || quant_mode == DQMOE_QUANT_FP8_CHANNEL ||
                     quant_mode == DQMOE_QUANT_FP8_BLOCK,
                 "quant_mode=%d: bf16 weights, or FP8 with scales per tensor, channel or block", quant_mode);
    DQ_CHECK_FMT(T >= 0 && T <= kMaxTokens, "T=%d: at most %d tokens (dqmoe_moe_block takes any number)", T, kMaxTokens);
    DQ_CHECK(H > 0 && I > 0 && E > 0 && k > 0 && k <= E && k <= kMaxTopk && n_shared >= 0);
    DQ_CHECK_FMT(int64_t(E) + n_shared <= kMaxExperts, "E=%d and n_shared=%d: at most %d experts", E, n_shared, kMaxExperts);
    DQ_CHECK_FMT(H % 16 == 0 && I % 16 == 0, "hidden_size=%d and inter_size=%d must be multiples of 16", H, I);
    // row numbers of the tensor maps and unit numbers are 32-bit
    DQ_CHECK_FMT(H <= (1 << 17) && I <= (1 << 17) && int64_t(E + n_shared) * (int64_t(2) * I + H) < (int64_t(1) << 31) &&
                     int64_t(E + n_shared) * ceil_div(I, 64) * ceil_div(H, 64) < (int64_t(1) << 30),
                 "H=%d I=%d E=%d: too large", H, I, E);
    return DQMOE_OK;
}

template <class K>
static int opt_in(K kern, int which) {
    static std::mutex mu;
    static bool configured[6][64] = {};
    int dev = 0;
    DQ_CUDA(cudaGetDevice(&dev));
    DQ_CHECK(dev >= 0 && dev < 64);
    std::lock_guard<std::mutex> lk(mu);
    if (!configured[which][dev]) {
        DQ_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, int(kSmemBytes)));
        configured[which][dev] = true;
    }
    return DQMOE_OK;
}

template <bool kFp8, int kTp>
static int launch_experts(const CUtensorMap& b, const CUtensorMap& b1, const Params& p, cudaStream_t stream) {
    DQ_RC(opt_in(moe_decode_experts_kernel<kFp8, kTp>, (kFp8 ? 3 : 0) + (kTp == 8 ? 0 : kTp == 16 ? 1 : 2)));
    return launch_pdl(moe_decode_experts_kernel<kFp8, kTp>, dim3(p.blocks), threads(kTp), kSmemBytes, stream, b, b1, p);
}

template <bool kF32, bool kFp8>
static int launch_route(const Params& p, cudaStream_t stream) {
    // a cluster for eight experts; more of them only lay x out, a K block of a token per warp and turn
    const int clusters = ceil_div(p.E, 8), wanted = ceil_div(p.kb1 * p.T, kSplit * 2 * (kRouteThreads / 32));
    const int most = sm_count() / kSplit;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(unsigned(kSplit * (clusters > wanted ? clusters : wanted < most ? wanted : (clusters > most ? clusters : most))), 1, 1);
    cfg.blockDim = dim3(kRouteThreads, 1, 1);
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = kSplit;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    DQ_CUDA(cudaLaunchKernelEx(&cfg, moe_decode_route_kernel<kF32, kFp8>, p));
    return DQMOE_OK;
}

}  // namespace moe_decode
}  // namespace dq

using namespace dq;

extern "C" {

size_t dqmoe_moe_decode_workspace_bytes(int T, int H, int I, int E, int k, int n_shared, int quant_mode) {
    if (moe_decode::check_sizes(T, H, I, E, k, n_shared, quant_mode) != DQMOE_OK) return 0;
    moe_decode::Params p{};
    p.T = T, p.H = H, p.I = I, p.E = E, p.k = k, p.n_shared = n_shared;
    return moe_decode::plan(&p, quant_mode != DQMOE_QUANT_NONE).total;
}

int dqmoe_moe_decode(const void* x_bf16, const void* w_router, int router_type, const void* b, const float* b_scale, const void* b1,
                     const float* b1_scale, void* out_bf16, void* workspace, size_t workspace_bytes, int T, int H, int I, int E, int k,
                     int n_shared, int scoring, int quant_mode, dqmoe_stream_t stream_) {
    cudaStream_t stream = static_cast<cudaStream_t>(stream_);
    DQ_RC(moe_decode::check_sizes(T, H, I, E, k, n_shared, quant_mode));
    DQ_CHECK(scoring == DQMOE_SCORE_SOFTMAX || scoring == DQMOE_SCORE_SIGMOID);
    DQ_CHECK_FMT(router_type == DQMOE_DT_BF16 || router_type == DQMOE_DT_FLOAT, "router_type=%d: BF16 or FLOAT", router_type);
    if (T == 0) return DQMOE_OK;
    const bool fp8 = quant_mode != DQMOE_QUANT_NONE;
    DQ_CHECK(x_bf16 != nullptr && w_router != nullptr && b != nullptr && b1 != nullptr && out_bf16 != nullptr);
    if (fp8) DQ_CHECK(b_scale != nullptr && b1_scale != nullptr);
    DQ_CHECK(is_aligned(x_bf16, 16) && is_aligned(w_router, 16) && is_aligned(b, 16) && is_aligned(b1, 16) && is_aligned(out_bf16, 2));
    if (fp8) DQ_CHECK(is_aligned(b_scale, 4) && is_aligned(b1_scale, 4));
    DQ_CHECK_FMT(workspace != nullptr && is_aligned(workspace, 256), "workspace pointer %p is not aligned!", workspace);
    moe_decode::Params p{};
    p.T = T, p.H = H, p.I = I, p.E = E, p.k = k, p.n_shared = n_shared;
    const moe_decode::Layout L = moe_decode::plan(&p, fp8);
    if (workspace_bytes != 0 && workspace_bytes < L.total)
        return fail(DQMOE_ERR_WORKSPACE, __FILE__, __LINE__, "workspace_bytes >= dqmoe_moe_decode_workspace_bytes(...)",
                    "workspace has %zu bytes, the layer needs %zu", workspace_bytes, L.total);
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    p.x = static_cast<const __nv_bfloat16*>(x_bf16);
    p.w_router = w_router;
    p.b_scale = b_scale;
    p.b1_scale = b1_scale;
    p.out = static_cast<__nv_bfloat16*>(out_bf16);
    p.scoring = scoring;
    p.mode = quant_mode;
    p.counters = reinterpret_cast<int*>(ws + L.counters);
    p.logits = reinterpret_cast<float*>(ws + L.logits);
    p.xq = ws + L.xq;
    p.aq = ws + L.aq;
    p.part1 = reinterpret_cast<float*>(ws + L.part1);
    p.part2 = reinterpret_cast<float*>(ws + L.part2);
    p.group2 = reinterpret_cast<float*>(ws + L.group2);
    p.status = device_status_word();
    if (p.status == nullptr) return DQMOE_ERR_CUDA;
    p.wait_limit = wait_limit();
    const int esz = fp8 ? 1 : 2;
    CUtensorMap map_b, map_b1;
    DQ_RC(gemm::make_map(&map_b, b, esz, uint64_t(E + n_shared) * 2 * I, uint64_t(H), moe_decode::kRows));
    DQ_RC(gemm::make_map(&map_b1, b1, esz, uint64_t(E + n_shared) * H, uint64_t(I), moe_decode::kRows));
    const bool f32 = router_type == DQMOE_DT_FLOAT;
    DQ_RC(f32 ? (fp8 ? moe_decode::launch_route<true, true>(p, stream) : moe_decode::launch_route<true, false>(p, stream))
              : (fp8 ? moe_decode::launch_route<false, true>(p, stream) : moe_decode::launch_route<false, false>(p, stream)));
    switch (moe_decode::token_rows(T)) {
        case 8: return fp8 ? moe_decode::launch_experts<true, 8>(map_b, map_b1, p, stream) : moe_decode::launch_experts<false, 8>(map_b, map_b1, p, stream);
        case 16: return fp8 ? moe_decode::launch_experts<true, 16>(map_b, map_b1, p, stream) : moe_decode::launch_experts<false, 16>(map_b, map_b1, p, stream);
        default: return fp8 ? moe_decode::launch_experts<true, 32>(map_b, map_b1, p, stream) : moe_decode::launch_experts<false, 32>(map_b, map_b1, p, stream);
    }
}

}  // extern "C"
