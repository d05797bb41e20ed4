// A projection that many requests share, each row with its request's low-rank adapter beside it, in two launches:
//   y[t] = x[t] W^T + bias + scale_a (x[t] A_a^T) B_a^T,   a = ids[t]; rows whose id is outside [0, L) have no adapter.
//
//   shrink    z[t] = scale_a x[t] A_a^T, [T, R] in the operands' type
//   project   y = x W^T + z B_a^T, summed in fp32
//
// What bounds it: with few rows the weights W and the adapters in use from HBM, and a chain of latencies (shrink, the last sums, the sums over
// parts); with hundreds the way from L2 to the SMs, some 60 bytes a cycle and SM (a K block of a tile of 128 x 256 takes 820 cycles to
// arrive, its MMAs 512); with thousands the tensor cores at the clock that the power limit leaves. project runs with W on the tensor core's first
// operand (M = 128 rows of W) and up to 256 rows of x on the second, so that a decode batch computes few columns too many; large batches take
// pairs of blocks, each with half of the rows of x for both. Tiles that do not fill the chip are cut along K into equal parts (plan_tiles).
//
// The adapters' part has two forms, by chunk of 16 rows. Where a chunk has one adapter - prefill, where a request's rows stand together - B_a is
// the first operand and z the second of MMAs on top of x W^T, for all such chunks that follow one another at once. Where it has several,
// the epilogue's warps multiply m16n8k16 fragments, each adapter by itself, and take the columns whose rows have that adapter: masks on a mixed
// product would let one adapter's infinities reach the rows of another. A block whose tile is its only one does that while the tensor core
// still sums. The list of these products is made from the ids by a warp of each block, and divided among the parts of a tile like its K.
// Forms of the second kind, us per call, for 64 rows of 64 adapters (K 4096, N 6144, R 16), and 333 fp16 rows of 40 requests (2880 x 2880, R 64):
//   rows of B in threads, z B^T by FMAs                                                                      70, 489
//   B and 16 rows of z through the stages into accumulators of their own, whose columns the epilogue picks   28, 38: 460 cycles of the
//                                                                               one thread that issues the copies for each product
//   fragments straight from L2, behind the sums / while the tensor core sums                                 24, 37 / 20, 31
//   B through shared memory in slots of their own                                                            20, 28.5
//
// project starts while shrink runs: it reads only x, W, ids and B until a tile's K is through. That is sound because shrink lets it start
// behind its own wait for the kernels before, which wrote those. No counterpart in the reference.
//
// us per call over 0.6 GB of inputs: one row, 4096 x 4096, R 16 13.3 (2.5 TB/s; floor 5.2); 64 rows as above 22.9 (3.0 TB/s; floor 10.8); 333 as above 30.4
// (floor 6.4); 4096 rows of 6 requests, 4096 x 4096, R 32 117 (1.2 PFLOP/s); 8191 rows of 24, K 7168, N 4096, R 16 357 (1.35 PFLOP/s). The figures further up
// are of calls over one set of inputs, which L2 partly holds: as built 10.7, 20.2 and 28.7.
#include <mutex>

#include "common.cuh"
#include "gemm_tile.cuh"
#include "ptx_sm100.cuh"
#include "streamk.cuh"

namespace dq {
namespace lora {

constexpr int kKBytes = 128;                    // bytes of a K block: one swizzle row, 64 values
constexpr int kKElems = 64;
constexpr int kRows = 128;                      // rows of W, or of stacked A, of an MMA
constexpr int kABytes = kRows * kKBytes;        // 16 KiB
constexpr int kMaxRank = 128;
constexpr int kStatusShrink = 311, kStatusProject = 312;

// ---------------------------------------------------------------- shrink

constexpr int kShrinkTok = 64;                  // rows of x per tile
constexpr int kShrinkThreads = 256;             // warp 0 TMA, warp 1 MMA, warps 4..7 epilogue
constexpr int kShrinkXBytes = kShrinkTok * kKBytes;
constexpr int kShrinkStages = 8;                // at most
constexpr int kMaxSplit = 8;                    // blocks of a cluster: slices of K

__device__ __forceinline__ uint16_t to_bits(float f, bool half) {
    return half ? __half_as_ushort(__float2half_rn(f)) : uint16_t(f2bf_bits(f));
}
template <bool kHalf>
__device__ __forceinline__ float2 unpack2(uint32_t w) {
    if constexpr (kHalf) return __half22float2(*reinterpret_cast<const __half2*>(&w));
    else return make_float2(bf16_lo(w), bf16_hi(w));
}

struct ShrinkParams {
    const uint16_t* x;      // rows form
    int64_t ldx;
    const uint16_t* lora_a; // [L, R, K]
    const int* ids;
    const float* scale;     // [L] or null
    uint16_t* z;            // [T, R] in the operands' type
    float* z_scale;         // [T], fp16: z counts times this power of two (1 but where a row's z lies near an end of fp16's range)
    int* counters;          // project's, cleared here
    int n_counters;
    int T, K, L, R;
    int half;               // operands fp16, else bf16
    int cap;                // tile form: adapters of a product,
    int stages;             // stages of the ring,
    int slots;              // clusters that share a tile's groups of adapters
    int* status;
    long long wait_limit;   // clock cycles before a wait gives up
};

// A row's z in the operands' type, by a warp whose lanes hold four values each (lane * 4 < R).
__device__ __forceinline__ void put_z(const ShrinkParams& p, int64_t t, float scale, float4 v, int lane) {
    v.x *= scale, v.y *= scale, v.z *= scale, v.w *= scale;
    if (p.half) {
        // Above 2^15 values would leave the range; below R 2^-14 what R values lose that are not normal numbers any more, 2^-25 each, would
        // be more than the rounding of the row's largest. Such rows have a power of two that brings the largest into [2^14, 2^15). The others do
        // without, so that chunks of one adapter can be summed on top of x W^T. us per call without / with: 4096 rows of 6 requests (4096 x 4096, R 32)
        // 120 / 157, of R 128 129 / 180, 64 rows of 64 (K 4096, N 6144, R 16; never summed so) 21.1 / 21.9.
        const float most = warp_max(lane * 4 < p.R ? fmaxf(fmaxf(fabsf(v.x), fabsf(v.y)), fmaxf(fabsf(v.z), fabsf(v.w))) : 0.0f);
        float up = 1.0f, down = 1.0f;
        if (most > 0.0f && most <= 3.402823466e38f && (most > 32768.0f || most < float(p.R) * 0x1p-14f)) {
            const int e = max(int(__float_as_uint(most) >> 23) - 127 - 14, -126);
            up = __uint_as_float(uint32_t(127 + e) << 23), down = __uint_as_float(uint32_t(127 - e) << 23);
        }
        v.x *= down, v.y *= down, v.z *= down, v.w *= down;
        if (lane == 0) p.z_scale[t] = up;
    }
    if (lane * 4 < p.R)
        *reinterpret_cast<uint2*>(p.z + t * p.R + lane * 4) =
            make_uint2(to_bits(v.x, p.half) | (uint32_t(to_bits(v.y, p.half)) << 16), to_bits(v.z, p.half) | (uint32_t(to_bits(v.w, p.half)) << 16));
}

// Rows form, for few rows: a block per row and 16 ranks (fp16: all ranks, whose common power of two it needs), a warp per rank. A warp has
// all its loads of A on their way at once, before project, which starts beside it, fills the path to memory.
constexpr int kRowWarps = 16;
constexpr int kRowValues = 4096;                // of K at a time: 16 loads of 16 bytes per lane
template <bool kHalf>
__global__ void __launch_bounds__(kRowWarps * 32) lora_shrink_rows_kernel(const __grid_constant__ ShrinkParams p) {
    pdl_wait();    // x, ids and the workspace
    pdl_launch();  // project: what is there before this kernel, it may read from now on
    __shared__ alignas(16) uint16_t s_x[kRowValues];
    __shared__ alignas(16) float s_z[kMaxRank];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (int i = (blockIdx.y * gridDim.x + blockIdx.x) * kRowWarps * 32 + threadIdx.x; i < p.n_counters; i += gridDim.x * gridDim.y * kRowWarps * 32)
        p.counters[i] = 0;
    const int t = blockIdx.x, id = p.ids[t];
    if (id < 0 || id >= p.L) return;
    const int first = blockIdx.y * kRowWarps, ranks = gridDim.y > 1 ? min(p.R, first + kRowWarps) : p.R;
    for (int r0 = first; r0 < ranks; r0 += kRowWarps) {
        const int r = r0 + warp;
        float sum = 0.0f;
        for (int k0 = 0; k0 < p.K; k0 += kRowValues) {
            const uint16_t* a = p.lora_a + (size_t(id) * p.R + r) * p.K + k0 + lane * 8;
            uint4 w[kRowValues / 256];
#pragma unroll
            for (int i = 0; i < kRowValues / 256; ++i)
                w[i] = r < ranks && k0 + i * 256 + lane * 8 < p.K ? *reinterpret_cast<const uint4*>(a + i * 256) : make_uint4(0, 0, 0, 0);
            const int k = k0 + threadIdx.x * 8;
            const uint4 x = k < p.K ? *reinterpret_cast<const uint4*>(p.x + t * p.ldx + k) : make_uint4(0, 0, 0, 0);
            __syncthreads();  // the values before have been read
            *reinterpret_cast<uint4*>(s_x + threadIdx.x * 8) = x;
            __syncthreads();
            static_assert(kRowValues == kRowWarps * 32 * 8, "a thread's share of x");
#pragma unroll
            for (int i = 0; i < kRowValues / 256; ++i) {
                if (k0 + i * 256 + lane * 8 >= p.K) continue;  // past K, where x may not be finite in the place of nothing
                const uint4 v = *reinterpret_cast<const uint4*>(s_x + i * 256 + lane * 8);
                const uint32_t xs[4] = {v.x, v.y, v.z, v.w}, ws[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float2 f = unpack2<kHalf>(xs[j]), g = unpack2<kHalf>(ws[j]);
                    sum = fmaf(f.x, g.x, sum);
                    sum = fmaf(f.y, g.y, sum);
                }
            }
        }
        sum = warp_sum(sum);
        if (lane == 0 && r < ranks) s_z[r] = sum;
    }
    __syncthreads();
    if (warp > 0) return;
    if (gridDim.y == 1) {
        put_z(p, t, p.scale != nullptr ? p.scale[id] : 1.0f, lane * 4 < p.R ? *reinterpret_cast<const float4*>(s_z + lane * 4) : make_float4(0, 0, 0, 0), lane);
    } else if (lane < ranks - first) {  // bf16: no power of two
        const float scale = p.scale != nullptr ? p.scale[id] : 1.0f;
        p.z[int64_t(t) * p.R + first + lane] = to_bits(s_z[first + lane] * scale, false);
    }
}

struct alignas(16) ShrinkTail {
    uint64_t full[kShrinkStages], empty[kShrinkStages], tmem_full[2], tmem_empty[2];
    uint32_t tmem_base;
    int abort_flag;
    int distinct;                               // adapters of the tile
    alignas(16) int id[kShrinkTok];             // -1 where there is none
    float scale[kShrinkTok];
    alignas(16) int place[kShrinkTok];          // place of a row's adapter among the tile's
    int adapter[kShrinkTok];                    // the tile's adapters in the order of their first rows
    uint32_t firsts[2];
};
// x first, so that an MMA's 128 rows of A, of which a stage has cap * R, end inside shared memory: behind the last stage lie the sums and what
// is left of an A tile.
static size_t shrink_smem(int R, int cap, int stages) {
    const size_t behind = size_t(kShrinkTok) * R * sizeof(float) + sizeof(ShrinkTail), tile = kABytes - size_t(cap) * R * kKBytes;
    return 1024 + size_t(stages) * (kShrinkXBytes + cap * R * kKBytes) + (behind > tile ? behind : tile);
}

__device__ __forceinline__ uint32_t cluster_nctarank() {
    uint32_t n;
    asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(n));
    return n;
}

// Tile form: 64 rows of x against all adapters among them, several adapters' A stacked on M = 128; of the product is kept what belongs together.
// K over a cluster of blocks where there are few tiles.
__global__ void __launch_bounds__(kShrinkThreads)
lora_shrink_tiles_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_a, const __grid_constant__ ShrinkParams p) {
    const int stage = kShrinkXBytes + p.cap * p.R * kKBytes;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    float* part = reinterpret_cast<float*>(ring + p.stages * stage);  // [64][R] of this block's slice of K
    ShrinkTail& st = *reinterpret_cast<ShrinkTail*>(part + kShrinkTok * p.R);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int i = 0; i < p.stages; ++i) {
            ptx::mbar_init(&st.full[i], 1);
            ptx::mbar_init(&st.empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            ptx::mbar_init(&st.tmem_full[i], 1);
            ptx::mbar_init(&st.tmem_empty[i], 4);
        }
        st.abort_flag = 0;
        ptx::fence_barrier_init();
    }
    if (warp == 1) {
        ptx::tmem_alloc(&st.tmem_base, 2 * kShrinkTok);
        ptx::tmem_relinquish();
    }
    pdl_wait();    // x, ids and the workspace
    pdl_launch();
    const int rank = int(ptx::cluster_ctarank()), split = int(cluster_nctarank());
    const int cluster = blockIdx.x / split, tile = cluster / p.slots, slot = cluster - tile * p.slots;
    for (int i = blockIdx.x * kShrinkThreads + threadIdx.x; i < p.n_counters; i += gridDim.x * kShrinkThreads) p.counters[i] = 0;
    if (threadIdx.x < kShrinkTok) {
        const int t = tile * kShrinkTok + threadIdx.x;
        const int id = t < p.T ? p.ids[t] : -1;
        st.id[threadIdx.x] = id >= 0 && id < p.L ? id : -1;
    }
    ptx::tc_fence_before();
    __syncthreads();
    ptx::tc_fence_after();
    const uint32_t tmem = *const_cast<volatile uint32_t*>(&st.tmem_base);
    // the distinct adapters, in the order of their first rows
    int first = kShrinkTok;  // this row's adapter appears first in row `first`
    if (threadIdx.x < kShrinkTok) {
        const int mine = st.id[threadIdx.x];
#pragma unroll
        for (int t = kShrinkTok - 4; t >= 0; t -= 4) {
            const int4 ids = *reinterpret_cast<const int4*>(st.id + t);
            first = ids.x == mine ? t : ids.y == mine ? t + 1 : ids.z == mine ? t + 2 : ids.w == mine ? t + 3 : first;
        }
        const uint32_t firsts = __ballot_sync(0xffffffffu, mine >= 0 && first == int(threadIdx.x));
        if (lane == 0) st.firsts[warp] = firsts;
    }
    __syncthreads();
    if (threadIdx.x < kShrinkTok) {
        const uint32_t lo = st.firsts[0], hi = st.firsts[1];
        const int mine = st.id[threadIdx.x];
        const int at = first < 32 ? __popc(lo & ((1u << first) - 1u)) : __popc(lo) + __popc(hi & ((1u << (first - 32)) - 1u));
        st.place[threadIdx.x] = mine >= 0 ? at : -1;
        if (mine >= 0 && first == int(threadIdx.x)) st.adapter[at] = mine;
        if (threadIdx.x == 0) st.distinct = __popc(lo) + __popc(hi);
    }
    __syncthreads();

    const int cap = p.cap, groups = (st.distinct + cap - 1) / cap;  // adapters of a product, products of the tile
    const int kbs = (p.K + kKElems - 1) / kKElems;
    const int kb0 = rank * kbs / split, kb1 = (rank + 1) * kbs / split;
    if (kb0 == kb1)
        for (int i = threadIdx.x; i < kShrinkTok * p.R; i += kShrinkThreads) part[i] = 0.0f;
    if (warp == 0 && kb0 < kb1) {
        if (ptx::elect_one()) {
            int it = 0;
            bool ok = true;
            for (int g = slot; ok && g < groups; g += p.slots) {
                const int n = min(cap, st.distinct - g * cap);
                for (int kb = kb0; kb < kb1; ++kb, ++it) {
                    const int s = it % p.stages;
                    if (!(ok = ptx::mbar_wait(&st.empty[s], ((it / p.stages) & 1) ^ 1, &st.abort_flag, p.wait_limit))) break;
                    uint8_t* a = ring + s * stage + kShrinkXBytes;
                    ptx::mbar_arrive_expect_tx(&st.full[s], uint32_t(n * p.R + kShrinkTok) * kKBytes);
                    ptx::tma_load_2d(ring + s * stage, &map_x, kb * kKElems, tile * kShrinkTok, &st.full[s]);
                    for (int i = 0; i < n; ++i)
                        ptx::tma_load_2d(a + i * p.R * kKBytes, &map_a, kb * kKElems, st.adapter[g * cap + i] * p.R, &st.full[s]);
                }
            }
        }
        __syncwarp();
    } else if (warp == 1 && kb0 < kb1) {
        if (ptx::elect_one()) {
            const uint32_t idesc = ptx::make_idesc(p.half ? 0 : 1, kRows, kShrinkTok);
            int it = 0, acc = 0;
            bool ok = true;
            for (int g = slot; ok && g < groups; g += p.slots, ++acc) {
                if (!ptx::mbar_wait(&st.tmem_empty[acc & 1], ((acc >> 1) & 1) ^ 1, &st.abort_flag, p.wait_limit)) break;
                for (int kb = kb0; kb < kb1; ++kb, ++it) {
                    const int s = it % p.stages;
                    if (!(ok = ptx::mbar_wait(&st.full[s], (it / p.stages) & 1, &st.abort_flag, p.wait_limit))) break;
                    ptx::tc_fence_after();
                    const uint64_t da = ptx::smem_desc_sw128(ptx::smem_u32(ring + s * stage + kShrinkXBytes));
                    const uint64_t db = ptx::smem_desc_sw128(ptx::smem_u32(ring + s * stage));
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        ptx::umma<1>(tmem + (acc & 1) * kShrinkTok, ptx::smem_desc_advance(da, k * 32), ptx::smem_desc_advance(db, k * 32), idesc,
                                     kb > kb0 || k > 0);
                    ptx::umma_commit(&st.empty[s]);
                }
                ptx::umma_commit(&st.tmem_full[acc & 1]);
            }
        }
        __syncwarp();
    } else if (warp == 2 || warp == 3) {
        const int t = threadIdx.x - 2 * 32, id = st.id[t];
        st.scale[t] = p.scale != nullptr && id >= 0 ? p.scale[id] : 1.0f;
    } else if (warp >= 4 && kb0 < kb1) {
        const int row = (warp - 4) * 32 + lane, mine = row / p.R, r = row - mine * p.R;
        int acc = 0;
        for (int g = slot; g < groups; g += p.slots, ++acc) {
            if (!ptx::mbar_wait_warp(&st.tmem_full[acc & 1], (acc >> 1) & 1, &st.abort_flag, p.wait_limit)) break;
            ptx::tc_fence_after();
            const int rows = min(kShrinkTok, p.T - tile * kShrinkTok);
#pragma unroll 1
            for (int c = 0; c < rows; c += 16) {
                int place[16];  // all of them before the first sum is put down, which might be one of them for all the compiler knows
#pragma unroll
                for (int i = 0; i < 16; i += 4) {
                    const int4 four = *reinterpret_cast<const int4*>(st.place + c + i);
                    place[i] = four.x, place[i + 1] = four.y, place[i + 2] = four.z, place[i + 3] = four.w;
                }
                float v[16];
                ptx::tmem_read(tmem + (uint32_t((warp - 4) * 32) << 16) + (acc & 1) * kShrinkTok + c, v);
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (mine < cap && place[i] == g * cap + mine) part[(c + i) * p.R + r] = v[i];
            }
            ptx::tc_fence_before();
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive(&st.tmem_empty[acc & 1]);
        }
    }
    ptx::settle_after_abort(&st.abort_flag);
    __syncthreads();
    if (threadIdx.x == 0 && st.abort_flag != 0) *p.status = kStatusShrink;
    if (warp == 1) {
        ptx::tc_fence_after();
        ptx::tmem_dealloc(tmem, 2 * kShrinkTok);
    }
    __syncwarp();
    // the slices of K in their order; each block of the cluster adds its share of the rows, a warp per row
    ptx::cluster_sync();
    for (int t = warp * split + rank; t < kShrinkTok; t += split * (kShrinkThreads / 32)) {
        const int place = st.place[t];
        if (place < 0 || (place / cap) % p.slots != slot) continue;
        float4 v[kMaxSplit], sum = make_float4(0, 0, 0, 0);
#pragma unroll
        for (int c = 0; c < kMaxSplit; ++c) {
            v[c] = make_float4(0, 0, 0, 0);
            if (c < split && lane * 4 < p.R)
                asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v[c].x), "=f"(v[c].y), "=f"(v[c].z), "=f"(v[c].w)
                             : "r"(ptx::map_to_cta(part + t * p.R + lane * 4, c)) : "memory");
        }
#pragma unroll
        for (int c = 0; c < kMaxSplit; ++c) sum.x += v[c].x, sum.y += v[c].y, sum.z += v[c].z, sum.w += v[c].w;
        put_z(p, int64_t(tile) * kShrinkTok + t, st.scale[t], sum, lane);
    }
    __syncthreads();
    ptx::cluster_sync();  // the others read this block's shared memory until here
}

// ---------------------------------------------------------------- project

constexpr int kThreads = 384;                   // warp 0 TMA, warp 1 MMA, warp 2 list of the adapters' products, warp 3 B of mixed rows, warps 4..11 epilogue
constexpr int kMaxTok = 256;
constexpr int kTmemCols = 512;                  // two accumulators
constexpr int kRingBytes = 216 * 1024;          // stages, and B of mixed rows
constexpr int kMaxStages = 10;
constexpr int kChunk = 16;                      // rows of x that are looked at together
constexpr int kMaxSlots = 8;                    // adapters' B on their way to each half of the epilogue
constexpr int kMaxParts = 16;

struct Params {
    const int* ids;
    const uint16_t* lora_b;   // [L, N, R]
    const uint16_t* z;        // [T, R]
    const float* z_scale;     // null unless fp16
    const float* bias;        // [N] or null
    uint16_t* y;
    int64_t ldy;
    int T, N, K, L, R;
    int tok;                  // rows of x per tile, a multiple of 16, on pairs of 32
    int stages;
    int slots;                // for B of mixed rows, of each half of the epilogue
    int n_tiles, tiles;       // tiles along N, and in all
    int kbs;
    int groups;               // blocks, or pairs of them
    int whole;                // tiles that are not split: group g takes g, g + groups, ...
    int parts;                // of each of the others, a group each
    int* counters;            // parts seen of each split tile, on pairs of each half of it
    float* part;              // [block] sums of a part of a tile, four rows of x together: [tok / 4][128][4]
    int* status;
    long long wait_limit;     // clock cycles before a wait gives up
};

// Products of a part of a tile. Direct: adapter, first chunk | chunks << 8, all of whose rows have it. Mixed, by the half of the epilogue that has
// the chunk: adapter, chunk | its rows << 16.
struct List {
    int direct0, direct1, mixed0[2], mixed1[2];
    uint2 direct[kMaxTok / kChunk], mixed[2][kMaxTok / 2];
};
struct alignas(16) Tail {
    uint64_t full[kMaxStages], empty[kMaxStages], tmem_full[2], tmem_empty[2];
    uint64_t list_full[2], list_empty[2];
    uint64_t b_full[2][kMaxSlots], b_empty[2][kMaxSlots];  // by half of the epilogue
    uint64_t meet;            // the epilogue warps
    uint32_t tmem_base;
    int abort_flag;
    int last_part;
    List list[2];
};
constexpr size_t kSmemBytes = 1024 + size_t(kRingBytes) + sizeof(Tail);  // at most: a launch asks for the stages that it has
static_assert(kSmemBytes <= 227 * 1024, "shared memory of one block");

struct Piece {
    int tile, kb0, kb1;
    int index, of;            // which of how many parts of its tile
};
// The pieces of a group, in order: its whole tiles, then its part of one of the others.
struct Pieces {
    const Params& p;
    int group, tile;
    __device__ __forceinline__ Pieces(const Params& p_, int group_) : p(p_), group(group_), tile(group_) {}
    __device__ __forceinline__ bool next(Piece* q) {
        if (tile < p.whole) {
            *q = Piece{tile, 0, p.kbs, 0, 1};
            tile += p.groups;
            return true;
        }
        if (left() == 0) return false;
        const int split = group / p.parts, index = group - split * p.parts;
        *q = Piece{p.whole + split, index * p.kbs / p.parts, (index + 1) * p.kbs / p.parts, index, p.parts};
        tile = 0x7fffffff;
        return true;
    }
    __device__ __forceinline__ int left() const { return tile < p.whole || (tile != 0x7fffffff && group < (p.tiles - p.whole) * p.parts) ? 1 : 0; }  // 0: none
};

__device__ __forceinline__ float load_f32(const float* from) {  // past L1: written while this kernel was here already
    float v;
    asm volatile("ld.relaxed.gpu.global.f32 %0, [%1];" : "=f"(v) : "l"(from) : "memory");
    return v;
}

// The adapters' products of a tile's rows, by one warp, and which of them belong to this part.
// scaled_rows: bit c where this lane's row of the c-th pair of chunks has a power of two.
template <bool kPair>
__device__ __forceinline__ void make_list(const Params& p, List& l, int t0, const Piece& q, int lane, const int (&ids)[kMaxTok / 32], uint32_t scaled_rows) {
    int direct = 0, mixed0 = 0, mixed1 = 0, last = -1, last_end = -1, last_first = 0;
    const int rows = min(p.tok, p.T - t0), half = lane >> 4;
#pragma unroll
    for (int pair = 0; pair < kMaxTok / 32; ++pair) {  // two chunks at a time, half a warp each
        const int c = 2 * pair;
        if (c * kChunk >= rows) break;
        int id = ids[pair];  // -2: no row
        if (id != -2 && (id < 0 || id >= p.L)) id = -1;
        if (c * kChunk + lane < rows && id == -2) id = -1;
        const bool scaled = ((scaled_rows >> pair) & 1u) != 0;
        const uint32_t present = __ballot_sync(0xffffffffu, id >= -1), with = __ballot_sync(0xffffffffu, id >= 0);
        if (with == 0) continue;
        const uint32_t scales = __ballot_sync(0xffffffffu, scaled);
        const uint32_t peers = __match_any_sync(0xffffffffu, 2 * id + half) >> (16 * half);  // of this half
        bool whole[2], mixes[2];  // whether a chunk has one adapter; whether it has any and is not a direct product
        int a[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const uint32_t here = 0xffffu << (16 * h);
            a[h] = __shfl_sync(0xffffffffu, id, (with & here) != 0 ? __ffs(with & here) - 1 : 0);
            const uint32_t same = __ballot_sync(0xffffffffu, id == a[h]) & here;
            whole[h] = (with & here) != 0 && same == (present & here) && (scales & here) == 0;
        }
        if constexpr (kPair) {  // both or neither: such products have 32 rows at least
            const bool both = whole[0] && (whole[1] ? a[0] == a[1] : (present >> 16) == 0);
            whole[0] = whole[1] = both;
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            mixes[h] = (with & (0xffffu << (16 * h))) != 0 && !whole[h];
            if (!whole[h]) continue;
            if (a[kPair ? 0 : h] != last || c + h != last_end) {
                last = a[kPair ? 0 : h];
                last_first = c + h;
                ++direct;
            }
            last_end = c + h + 1;
            if (lane == 0) l.direct[direct - 1] = make_uint2(uint32_t(last), uint32_t(last_first | ((last_end - last_first) << 8)));
        }
        const bool leads = id >= 0 && (lane & 15) == __ffs(peers) - 1 && (half ? mixes[1] : mixes[0]);
        const uint32_t leaders = __ballot_sync(0xffffffffu, leads);
        const int at = (half ? mixed1 : mixed0) + __popc((leaders >> (16 * half)) & ((1u << (lane & 15)) - 1u));
        if (leads) l.mixed[half][at] = make_uint2(uint32_t(id), uint32_t(c + half) | (peers << 16));
        mixed0 += __popc(leaders & 0xffffu);
        mixed1 += __popc(leaders >> 16);
    }
    if (lane == 0) {
        l.direct0 = direct * q.index / q.of;
        l.direct1 = direct * (q.index + 1) / q.of;
        l.mixed0[0] = mixed0 * q.index / q.of;
        l.mixed1[0] = mixed0 * (q.index + 1) / q.of;
        l.mixed0[1] = mixed1 * q.index / q.of;
        l.mixed1[1] = mixed1 * (q.index + 1) / q.of;
    }
}

template <bool kHalf, bool kPair>
struct Epilogue {
    const Params& p;
    Tail& st;
    uint32_t tmem;            // this warp's lanes
    int warp, lane, row;      // warp 0..7, row = TMEM lane = row of W among the block's 128 of the tile
    int rank;                 // of the block in its pair
    const uint8_t* b_ring;
    int b_it = 0;             // B's of this half so far
    uint32_t meetings = 0;

    __device__ __forceinline__ bool meet() {
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(&st.meet);
        return ptx::mbar_wait_warp(&st.meet, meetings++ & 1, &st.abort_flag, p.wait_limit);
    }

    __device__ __forceinline__ void store(float (&v)[kChunk], int t0, int n) {
        if (n >= p.N) return;
        const float bias = p.bias != nullptr ? p.bias[n] : 0.0f;
        uint16_t* y = p.y + int64_t(t0) * p.ldy + n;
#pragma unroll
        for (int j = 0; j < kChunk; ++j)
            if (t0 + j < p.T) y[j * p.ldy] = to_bits(v[j] + bias, kHalf);
    }

    // The same from the accumulators of m16n8k16 products, of the 32 rows of W from n0 on.
    __device__ __forceinline__ void store_fragments(const float (&v)[kChunk], int t0, int n0) {
#pragma unroll
        for (int i = 0; i < kChunk; ++i) {
            const int n = n0 + (i >> 3) * 16 + ((i >> 1) & 1) * 8 + (lane >> 2), t = t0 + ((i >> 2) & 1) * 8 + (lane & 3) * 2 + (i & 1);
            if (n < p.N && t < p.T) p.y[int64_t(t) * p.ldy + n] = to_bits(v[i] + (p.bias != nullptr ? p.bias[n] : 0.0f), kHalf);
        }
    }

    // The adapters' products of the mixed rows of a chunk, from place `e` of the list on: B's rows are the products' rows, z's rows their columns, of
    // which each takes the columns that have its adapter. 16 bytes of a row are eight values that follow one another; which of them a product takes
    // for its k is the same for both, and a sum does not mind. Returns the place behind them, -1 where a wait has run out.
    __device__ __forceinline__ int products(const List& l, int half, int e, int chunk, int t0, float (&v)[kChunk]) {
        const int k_lane = (lane & 3) * 8, g = lane >> 2;
        uint4 z[kMaxRank / 32][2];
        float scale[4] = {1.0f, 1.0f, 1.0f, 1.0f};  // of this lane's columns
#pragma unroll
        for (int k = 0; k < kMaxRank / 32; ++k)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int t = t0 + h * 8 + g;  // a row without an adapter, whose z is nothing, has a column that nobody takes
                z[k][h] = k * 32 + k_lane < p.R && t < p.T ? load16(p.z + size_t(t) * p.R + k * 32 + k_lane) : make_uint4(0, 0, 0, 0);
            }
        if constexpr (kHalf) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int t = t0 + (j >> 1) * 8 + (lane & 3) * 2 + (j & 1);
                if (t < p.T) scale[j] = load_f32(p.z_scale + t);
            }
        }
#pragma unroll
        for (int j = 0; j < kChunk; ++j) v[j] = 0.0f;
        const int end = l.mixed1[half], slot_bytes = kRows * p.R * 2;
#pragma unroll 1
        for (; e < end; ++e, ++b_it) {
            const uint32_t entry = l.mixed[half][e].y, rows = entry >> 16;
            if (int(entry & 0xff) != chunk) break;
            const int slot = b_it % p.slots;
            if (!ptx::mbar_wait_warp(&st.b_full[half][slot], (b_it / p.slots) & 1, &st.abort_flag, p.wait_limit)) return -1;
            const uint8_t* from = b_ring + (half * p.slots + slot) * slot_bytes + ((row - lane + g) * p.R + k_lane) * 2;
            float d[kChunk];
#pragma unroll
            for (int j = 0; j < kChunk; ++j) d[j] = 0.0f;
#pragma unroll
            for (int k = 0; k < kMaxRank / 32; ++k) {
                if (k * 32 >= p.R) break;
                const bool in = k * 32 + k_lane < p.R;
                uint4 b[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) b[j] = in ? *reinterpret_cast<const uint4*>(from + (j * 8 * p.R + k * 32) * 2) : make_uint4(0, 0, 0, 0);
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    if ((rows >> (8 * h)) & 255u) {
#pragma unroll
                        for (int m = 0; m < 2; ++m) {
                            float* c = d + (2 * m + h) * 4;
                            ptx::mma_16x8x16<kHalf>(c, b[2 * m].x, b[2 * m + 1].x, b[2 * m].y, b[2 * m + 1].y, z[k][h].x, z[k][h].y);
                            ptx::mma_16x8x16<kHalf>(c, b[2 * m].z, b[2 * m + 1].z, b[2 * m].w, b[2 * m + 1].w, z[k][h].z, z[k][h].w);
                        }
                    }
            }
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive(&st.b_empty[half][slot]);
#pragma unroll
            for (int j = 0; j < kChunk; ++j) {
                const int column = ((j >> 2) & 1) * 8 + (lane & 3) * 2 + (j & 1);
                if ((rows >> column) & 1u) v[j] = kHalf ? d[j] * scale[((j >> 2) & 1) * 2 + (j & 1)] : d[j];
            }
        }
        return e;
    }
    static __device__ __forceinline__ uint4 load16(const uint16_t* from) {  // past L1: written while this kernel was here already
        uint4 v;
        asm volatile("ld.relaxed.gpu.global.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(from) : "memory");
        return v;
    }

    // The sums of a tile from its parts, in their order: kParts parts of kChunks chunks of this half are loaded at once.
    template <int kParts, int kChunks>
    __device__ __forceinline__ void add_parts(const float* part, int parts, size_t stride, int half, int cols, int t0, int n) {
#pragma unroll 1
        for (int c = half; c * kChunk < cols; c += 2 * kChunks) {
            const float* from = part + c * kChunk * kRows + row * 4;
            float v[kChunks][kChunk];
#pragma unroll
            for (int i = 0; i < kChunks; ++i)
#pragma unroll
                for (int j = 0; j < kChunk; ++j) v[i][j] = 0.0f;
#pragma unroll 1
            for (int o = 0; o < parts; o += kParts) {
                float4 f[kParts][kChunks][kChunk / 4];
#pragma unroll
                for (int k = 0; k < kParts; ++k)
#pragma unroll
                    for (int i = 0; i < kChunks; ++i)
#pragma unroll
                        for (int j = 0; j < kChunk / 4; ++j)
                            f[k][i][j] = o + k < parts && (c + 2 * i) * kChunk + 4 * j < cols
                                             ? streamk::ld_partial4(from + (o + k) * stride + (2 * i * kChunk + 4 * j) * kRows) : make_float4(0, 0, 0, 0);
#pragma unroll
                for (int k = 0; k < kParts; ++k)
#pragma unroll
                    for (int i = 0; i < kChunks; ++i)
#pragma unroll
                        for (int j = 0; j < kChunk / 4; ++j)
                            v[i][4 * j] += f[k][i][j].x, v[i][4 * j + 1] += f[k][i][j].y, v[i][4 * j + 2] += f[k][i][j].z, v[i][4 * j + 3] += f[k][i][j].w;
            }
#pragma unroll
            for (int i = 0; i < kChunks; ++i)
                if ((c + 2 * i) * kChunk < cols) store(v[i], t0 + (c + 2 * i) * kChunk, n);  // behind the tile begin the next one's rows
        }
    }

    __device__ __forceinline__ void run() {
        pdl_wait();  // shrink: the counters, z_scale
        const int group = int(blockIdx.x) >> (kPair ? 1 : 0);
        Pieces pieces(p, group);
        Piece q;
        const int half = warp >> 2;
        for (int acc = 0; pieces.next(&q); ++acc) {
            const int tt = q.tile / p.n_tiles, n = ((q.tile - tt * p.n_tiles) * (kPair ? 2 : 1) + rank) * kRows + row, t0 = tt * p.tok;
            const int buf = acc & 1, parity = (acc >> 1) & 1;
            if (!ptx::mbar_wait_warp(&st.list_full[buf], parity, &st.abort_flag, p.wait_limit)) return;
            const List& l = st.list[buf];
            // columns in use; the two halves of the epilogue take chunks in turn
            const int cols = min(p.tok, p.T - t0), n0 = n - lane;
            // A block's only piece: the mixed products while the tensor core still sums, into the accumulators that nobody needs. Else, and then, the sums.
            const bool ahead = pieces.left() == 0 && acc == 0;
            const uint32_t sums = tmem + buf * p.tok, others = tmem + (buf ^ 1) * p.tok;
            uint32_t mixed_chunks = 0;
            int e = l.mixed0[half];
#pragma unroll 1
            for (int pass = ahead ? 0 : 1; pass < 2; ++pass) {
                if (pass == 1) {
                    if (!ptx::mbar_wait_warp(&st.tmem_full[buf], parity, &st.abort_flag, p.wait_limit)) return;
                    ptx::tc_fence_after();
                }
#pragma unroll 1
                for (int c = half; c * kChunk < cols; c += 2) {
                    float v[kChunk], d[kChunk];
                    const bool now = e < l.mixed1[half] && int(l.mixed[half][e].y & 0xff) == c;
                    if (now && (e = products(l, half, e, c, t0 + c * kChunk, d)) < 0) return;
                    if (pass == 0) {
                        if (now) {
                            ptx::tmem_write_fragments(others + c * kChunk, d);
                            mixed_chunks |= 1u << c;
                        }
                        continue;
                    }
                    float* to = p.part + (size_t(blockIdx.x) * p.tok + c * kChunk) * kRows;
                    if (now || ((mixed_chunks >> c) & 1u) != 0) {
                        if (!now) ptx::tmem_read_fragments(others + c * kChunk, d);
                        ptx::tmem_read_fragments(sums + c * kChunk, v);
#pragma unroll
                        for (int j = 0; j < kChunk; ++j) v[j] += d[j];
                        if (q.of == 1) {
                            store_fragments(v, t0 + c * kChunk, n0);
                            continue;
                        }
#pragma unroll
                        for (int j = 0; j < kChunk; j += 2) {
                            const int r = row - lane + (j >> 3) * 16 + ((j >> 1) & 1) * 8 + (lane >> 2), t = ((j >> 2) & 1) * 8 + (lane & 3) * 2;
                            if (c * kChunk + (t & ~3) < cols) *reinterpret_cast<float2*>(to + (t & ~3) * kRows + r * 4 + (t & 3)) = make_float2(v[j], v[j + 1]);
                        }
                        continue;
                    }
                    ptx::tmem_read(sums + c * kChunk, v);
                    if (q.of == 1) {
                        store(v, t0 + c * kChunk, n);
                        continue;
                    }
#pragma unroll
                    for (int j = 0; j < kChunk; j += 4)
                        if (c * kChunk + j < cols) *reinterpret_cast<float4*>(to + j * kRows + row * 4) = make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]);
                }
            }
            ptx::tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                if constexpr (kPair) ptx::mbar_arrive_cluster(ptx::map_to_cta(&st.tmem_empty[buf], 0));
                else ptx::mbar_arrive(&st.tmem_empty[buf]);
                ptx::mbar_arrive(&st.list_empty[buf]);
            }
            if (q.of == 1) continue;
            // What the warps wrote, the counting thread has seen at `meet`, and its release and acquire at gpu scope hold for all of them: a fence in
            // each thread, before and after, took 1 and 3 to 6 us.
            const int first = kPair ? (group - q.index) * 2 + rank : group - q.index;
            if (!meet()) return;
            if (warp == 0 && lane == 0) {
                int* counter = &p.counters[kPair ? (q.tile - p.whole) * 2 + rank : q.tile - p.whole];
                st.last_part = streamk::atomic_add_acq_rel_gpu(counter, 1) == q.of - 1;
            }
            if (!meet()) return;
            if (*const_cast<volatile int*>(&st.last_part) == 0) continue;
            const size_t stride = size_t(kPair ? 2 : 1) * p.tok * kRows;
            const float* from = p.part + size_t(first) * p.tok * kRows;
            if (q.of == 2) add_parts<2, 2>(from, q.of, stride, half, cols, t0, n);
            else add_parts<5, 1>(from, q.of, stride, half, cols, t0, n);
        }
    }
};

// kPair: two blocks of a cluster have 128 rows of W each of a tile of 256 and half of its rows of x; the first one issues the MMAs for both and owns
// the barriers of the stages.
template <bool kHalf, bool kPair>
__global__ void __launch_bounds__(kThreads, 1)
lora_project_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_z,
                    const __grid_constant__ CUtensorMap map_b, const __grid_constant__ Params p) {
    pdl_launch();
    extern __shared__ uint8_t smem_raw[];
    uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = kPair ? int(ptx::cluster_ctarank()) : 0, group = int(blockIdx.x) >> (kPair ? 1 : 0);
    const int x_rows = kPair ? p.tok / 2 : p.tok;  // of this block
    const int stage = kABytes + x_rows * kKBytes;
    uint8_t* b_ring = ring + p.stages * stage;     // [half of the epilogue][slot]: 128 rows of an adapter's B, as in memory
    const int slot_bytes = kRows * p.R * 2;
    Tail& st = *reinterpret_cast<Tail*>(b_ring + 2 * p.slots * slot_bytes);
    if (threadIdx.x == 0) {
        for (int i = 0; i < p.stages; ++i) {
            ptx::mbar_init(&st.full[i], 1);
            ptx::mbar_init(&st.empty[i], 1);
        }
        for (int i = 0; i < p.slots; ++i)
            for (int h = 0; h < 2; ++h) {
                ptx::mbar_init(&st.b_full[h][i], 1);
                ptx::mbar_init(&st.b_empty[h][i], 4);
            }
        for (int i = 0; i < 2; ++i) {
            ptx::mbar_init(&st.tmem_full[i], 1);
            ptx::mbar_init(&st.tmem_empty[i], kPair ? 16 : 8);
            ptx::mbar_init(&st.list_full[i], 1);
            ptx::mbar_init(&st.list_empty[i], rank == 0 ? 11 : 10);  // TMA thread, B's thread, epilogue warps, the first block's MMA thread
        }
        ptx::mbar_init(&st.meet, 8);
        st.abort_flag = 0;
        ptx::fence_barrier_init();
    }
    if constexpr (kPair) ptx::cluster_sync();  // the other block's barriers exist before anything signals them
    if (warp == 1) {
        if constexpr (kPair) {
            ptx::tmem_alloc_pair(&st.tmem_base, kTmemCols);
            ptx::tmem_relinquish_pair();
        } else {
            ptx::tmem_alloc(&st.tmem_base, kTmemCols);
            ptx::tmem_relinquish();
        }
    }
    ptx::tc_fence_before();
    __syncthreads();
    if constexpr (kPair) ptx::cluster_sync();  // both hold their TMEM before the first MMA
    ptx::tc_fence_after();
    const uint32_t tmem = *const_cast<volatile uint32_t*>(&st.tmem_base);

    if (warp == 0) {
        if (ptx::elect_one()) {
            Pieces pieces(p, group);
            Piece q, held;
            int it = 0;
            bool ok = true, waited = false;
            auto next_stage = [&]() { return ptx::mbar_wait(&st.empty[it % p.stages], ((it / p.stages) & 1) ^ 1, &st.abort_flag, p.wait_limit); };
            // the barrier of stage s, which expects `bytes` from this block, and on pairs as many from the other one
            auto expect = [&](int s, uint32_t bytes) {
                if (rank == 0) ptx::mbar_arrive_expect_tx(&st.full[s], kPair ? 2 * bytes : bytes);
                return kPair ? ptx::map_to_cta(&st.full[s], 0) : ptx::smem_u32(&st.full[s]);
            };
            auto sums = [&](const Piece& q) {  // x W^T
                const int tt = q.tile / p.n_tiles, n0 = ((q.tile - tt * p.n_tiles) * (kPair ? 2 : 1) + rank) * kRows, t0 = tt * p.tok + rank * x_rows;
                for (int kb = q.kb0; kb < q.kb1; ++kb, ++it) {
                    if (!next_stage()) return false;
                    const int s = it % p.stages;
                    const uint32_t bar = expect(s, uint32_t(stage));
                    ptx::tma_load_2d_any<kPair>(ring + s * stage, &map_w, kb * kKElems, n0, bar);
                    ptx::tma_load_2d_any<kPair>(ring + s * stage + kABytes, &map_x, kb * kKElems, t0, bar);
                }
                return true;
            };
            auto products = [&](const Piece& q, int n) {  // z B^T
                const int tt = q.tile / p.n_tiles, n0 = ((q.tile - tt * p.n_tiles) * (kPair ? 2 : 1) + rank) * kRows, t0 = tt * p.tok;
                if (!ptx::mbar_wait(&st.list_full[n & 1], (n >> 1) & 1, &st.abort_flag, p.wait_limit)) return false;
                const List& l = st.list[n & 1];
                if (l.direct0 < l.direct1 && !waited) {
                    pdl_wait();  // shrink: z
                    waited = true;
                }
                for (int i = l.direct0; i < l.direct1; ++i) {
                    const uint2 e = l.direct[i];
                    const int c = int(e.y & 0xff), chunks = int(e.y >> 8);
                    for (int r0 = 0; r0 < p.R; r0 += kKElems, ++it) {
                        if (!next_stage()) return false;
                        const int s = it % p.stages;
                        const int mine = kPair ? chunks / 2 : chunks;  // chunks of z that this block loads
                        const uint32_t bar = expect(s, uint32_t(kABytes + mine * kChunk * kKBytes));
                        ptx::tma_load_3d<kPair>(ring + s * stage, &map_b, r0, n0, int(e.x), bar);
                        for (int j = 0; j < mine; ++j)
                            ptx::tma_load_2d_any<kPair>(ring + s * stage + kABytes + j * kChunk * kKBytes, &map_z, r0, t0 + (c + rank * mine + j) * kChunk, bar);
                    }
                }
                ptx::mbar_arrive(&st.list_empty[n & 1]);
                return true;
            };
            for (int n = 0; ok && pieces.next(&q); ++n) {
                ok = sums(q);
                if (n == 0) held = q;  // shrink may still run: the first piece's products come behind the second one's sums
                else ok = ok && (n > 1 || products(held, 0)) && products(q, n);
                if (n == 0 && pieces.left() == 0) ok = ok && products(q, 0);
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        if (rank == 0 && ptx::elect_one()) {
            Pieces pieces(p, group);
            Piece q;
            int it = 0;
            bool ok = true;
            auto commit = [&](uint64_t* bar) {  // all MMAs so far
                if constexpr (kPair) {
                    ptx::umma_commit_pair(ptx::map_to_cta(bar, 0));
                    ptx::umma_commit_pair(ptx::map_to_cta(bar, 1));
                } else {
                    ptx::umma_commit(bar);
                }
            };
            // one stage into the accumulator at `d`, `cols` columns of the second operand
            auto block = [&](uint32_t d, int cols, int steps, bool more) {
                const uint32_t idesc = ptx::make_idesc(kHalf ? 0 : 1, kPair ? 2 * kRows : kRows, uint32_t(cols));
                const int s = it % p.stages;
                if (!ptx::mbar_wait(&st.full[s], (it / p.stages) & 1, &st.abort_flag, p.wait_limit)) return false;
                ptx::tc_fence_after();
                const uint64_t da = ptx::smem_desc_sw128(ptx::smem_u32(ring + s * stage));
                const uint64_t db = ptx::smem_desc_sw128(ptx::smem_u32(ring + s * stage + kABytes));
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    if (k < steps) {
                        if constexpr (kPair) ptx::umma_pair<1>(d, ptx::smem_desc_advance(da, k * 32), ptx::smem_desc_advance(db, k * 32), idesc, more || k > 0);
                        else ptx::umma<1>(d, ptx::smem_desc_advance(da, k * 32), ptx::smem_desc_advance(db, k * 32), idesc, more || k > 0);
                    }
                commit(&st.empty[s]);
                ++it;
                return true;
            };
            auto sums = [&](const Piece& q, int n) {
                if (!ptx::mbar_wait(&st.tmem_empty[n & 1], ((n >> 1) & 1) ^ 1, &st.abort_flag, p.wait_limit)) return false;
                ptx::tc_fence_after();
                for (int kb = q.kb0; kb < q.kb1; ++kb)
                    if (!block(tmem + (n & 1) * p.tok, p.tok, 4, kb > q.kb0)) return false;
                return true;
            };
            auto products = [&](int n) {
                if (!ptx::mbar_wait(&st.list_full[n & 1], (n >> 1) & 1, &st.abort_flag, p.wait_limit)) return false;
                const List& l = st.list[n & 1];
                for (int e = l.direct0; e < l.direct1; ++e)
                    for (int r0 = 0; r0 < p.R; r0 += kKElems)
                        if (!block(tmem + (n & 1) * p.tok + (l.direct[e].y & 0xff) * kChunk, int(l.direct[e].y >> 8) * kChunk, min(4, (p.R - r0 + 15) / 16), true))
                            return false;
                commit(&st.tmem_full[n & 1]);
                ptx::mbar_arrive(&st.list_empty[n & 1]);
                return true;
            };
            for (int n = 0; ok && pieces.next(&q); ++n) {  // in the order of the copies
                ok = sums(q, n);
                if (n > 0) ok = ok && (n > 1 || products(0)) && products(n);
                if (n == 0 && pieces.left() == 0) ok = ok && products(0);
            }
        }
        __syncwarp();
    } else if (warp == 2) {
        Pieces pieces(p, group);
        Piece q;
        for (int n = 0; pieces.next(&q); ++n) {
            if (!ptx::mbar_wait_warp(&st.list_empty[n & 1], ((n >> 1) & 1) ^ 1, &st.abort_flag, p.wait_limit)) break;
            List& l = st.list[n & 1];
            const int tt = q.tile / p.n_tiles, t0 = tt * p.tok, rows = min(p.tok, p.T - t0);
            int ids[kMaxTok / 32];
#pragma unroll
            for (int c = 0; c < kMaxTok / 32; ++c) ids[c] = c * 32 + lane < rows ? ld_relaxed_gpu(p.ids + t0 + c * 32 + lane) : -2;  // before this kernel's wait, so past L1
            uint32_t scaled_rows = 0;
            // fp16: before shrink is over as if no row had a power of two, which is made good where one has
#pragma unroll 1
            for (bool known = !kHalf;;) {
                make_list<kPair>(p, l, t0, q, lane, ids, scaled_rows);
                __syncwarp();
                if (scaled_rows == 0) {  // the mixed rows' B towards L2 meanwhile: 128 rows of an adapter's follow one another in memory
                    const int n0 = ((q.tile - tt * p.n_tiles) * (kPair ? 2 : 1) + rank) * kRows;
                    const uint32_t bytes = uint32_t(max(0, min(kRows, p.N - n0)) * p.R) * 2u;
#pragma unroll
                    for (int h = 0; h < 2; ++h)
                        for (int e = l.mixed0[h] + lane; bytes > 0 && e < l.mixed1[h]; e += 32)
                            asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(p.lora_b + (size_t(l.mixed[h][e].x) * p.N + n0) * p.R), "r"(bytes));
                }
                if (known) break;
                known = true;
                if (n == 0) pdl_wait();  // shrink: z_scale
                float scale[kMaxTok / 32];  // all loads at once; rows without an adapter have none
#pragma unroll
                for (int c = 0; c < kMaxTok / 32; ++c) scale[c] = c * 32 + lane < rows ? load_f32(p.z_scale + t0 + c * 32 + lane) : 1.0f;
#pragma unroll
                for (int c = 0; c < kMaxTok / 32; ++c)
                    if (ids[c] >= 0 && ids[c] < p.L && scale[c] != 1.0f) scaled_rows |= 1u << c;
                if (!__any_sync(0xffffffffu, scaled_rows != 0)) break;
            }
            if (lane == 0) {
                if (((q.tile - tt * p.n_tiles) * (kPair ? 2 : 1) + rank) * kRows >= p.N) l.mixed1[0] = l.mixed0[0], l.mixed1[1] = l.mixed0[1];  // no rows of W
                ptx::mbar_arrive(&st.list_full[n & 1]);
            }
        }
    } else if (warp == 3) {
        // B of the mixed rows' products: 128 rows of an adapter's follow one another in memory. A lane for each slot of each half: one thread's
        // 300 cycles a copy would set the pace.
        Pieces pieces(p, group);
        Piece q;
        const int h = lane >> 4, slot = lane & 15;
        int before = 0, uses = 0;  // products of this half in earlier pieces; of this slot
        bool ok = true;
        for (int n = 0; ok && pieces.next(&q); ++n) {
            if (!(ok = ptx::mbar_wait_warp(&st.list_full[n & 1], (n >> 1) & 1, &st.abort_flag, p.wait_limit))) break;
            const List& l = st.list[n & 1];
            const int n0 = ((q.tile % p.n_tiles) * (kPair ? 2 : 1) + rank) * kRows;
            const uint32_t bytes = uint32_t(max(0, min(kRows, p.N - n0)) * p.R) * 2u;
            const int first = l.mixed0[h], end = l.mixed1[h];
            int e = slot < p.slots ? first + (slot + p.slots - before % p.slots) % p.slots : end;  // this slot's first
            const long long begin = clock64();
            while (__any_sync(0xffffffffu, e < end)) {
                if (e < end && ptx::mbar_test_wait(&st.b_empty[h][slot], (uses & 1) ^ 1)) {
                    ptx::mbar_arrive_expect_tx(&st.b_full[h][slot], bytes);
                    ptx::bulk_load(b_ring + (h * p.slots + slot) * slot_bytes, p.lora_b + (size_t(l.mixed[h][e].x) * p.N + n0) * p.R, bytes, &st.b_full[h][slot]);
                    ++uses;
                    e += p.slots;
                }
                if (clock64() - begin > p.wait_limit) *const_cast<volatile int*>(&st.abort_flag) = 1;
                if (__any_sync(0xffffffffu, *const_cast<volatile int*>(&st.abort_flag) != 0)) {
                    ok = false;
                    break;
                }
            }
            before += end - first;
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive(&st.list_empty[n & 1]);
        }
        __syncwarp();
    } else if (warp >= 4) {
        Epilogue<kHalf, kPair> ep{p, st, tmem + (uint32_t((warp & 3) * 32) << 16), warp - 4, lane, (warp & 3) * 32 + lane, rank, b_ring};
        ep.run();
    }
    ptx::settle_after_abort(&st.abort_flag);
    ptx::tc_fence_before();
    __syncthreads();
    if constexpr (kPair) ptx::cluster_sync();  // the other block is through with this one's barriers and shared memory
    if (threadIdx.x == 0 && st.abort_flag != 0) *p.status = kStatusProject;
    if (warp == 1) {
        ptx::tc_fence_after();
        if constexpr (kPair) ptx::tmem_dealloc_pair(tmem, kTmemCols);
        else ptx::tmem_dealloc(tmem, kTmemCols);
    }
}

// ---------------------------------------------------------------- host

static int make_map(CUtensorMap* map, const void* base, bool half, int dims, const cuuint64_t* dim, const cuuint64_t* stride, const cuuint32_t* box) {
    gemm::EncodeTiledFn fn = gemm::encode_fn();
    if (fn == nullptr) return fail(DQMOE_ERR_CUDA, __FILE__, __LINE__, "cuTensorMapEncodeTiled", "driver entry point not found");
    const cuuint32_t one[3] = {1, 1, 1};
    const CUresult r = fn(map, half ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, cuuint32_t(dims), const_cast<void*>(base),
                          dim, stride, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(DQMOE_ERR_CUDA, __FILE__, __LINE__, "cuTensorMapEncodeTiled", "CUresult %d", int(r));
    return DQMOE_OK;
}
static int make_map_2d(CUtensorMap* map, const void* base, bool half, int64_t rows, int64_t cols, int64_t ld, int box_rows) {
    const cuuint64_t dim[2] = {cuuint64_t(cols), cuuint64_t(rows)}, stride[1] = {cuuint64_t(ld) * 2};
    const cuuint32_t box[2] = {kKElems, cuuint32_t(box_rows)};
    return make_map(map, base, half, 2, dim, stride, box);
}

struct Layout {
    size_t counters, z, z_scale, part, total;
};
// Tiles of x's rows, blocks or pairs, and parts, by an estimate in clock cycles, whose constants are fits to measurements (all forms, 1 to 8191
// rows, N 2880 to 14336, K 2880 to 7168; the form chosen is within 5 % of the fastest): a K block of a tile takes its MMAs (two cycles a row)
// or its bytes from L2; W and x come from HBM once, and of the two the shorter one costs half of its time beside the longer; a tile's last sums
// leave TMEM behind the last MMA; parts are written, counted and added. N = K = 4096, us per call without adapters: 1 row 1 part of a tile each
// 22, 4 parts 12.8; 128 rows in one tile of 4 parts 18.3, in two of 2 parts 17.7; 512 rows in 4 tiles of 128 27.8, with what had one part
// more or less in each block's share 41.5; 4096 rows on single blocks 110.8, on pairs 103.1.
// Parts add through L2. As clusters that send their sums through distributed shared memory one row took 12.4 instead of 10.5 (4 parts), 64 rows of
// 64 adapters (N 6144, R 16; 3 parts) 22.6 / 20.0: clusters start late and do not fill the chip (of three blocks 45 fit).
constexpr int kL2Bytes[2] = {60, 47};                // per cycle and SM, on single blocks and on pairs
constexpr int kHbmBytes = 3300;                      // per cycle
constexpr int kDrain = 12, kAdd = 8;                 // cycles a column; a column of each part
constexpr int kPairing[2] = {0, 700}, kCount[2] = {3000, 5500};  // a launch; a tile in parts
constexpr int kMixedRows = 512, kMixedBytes = 64 * 1024, kFewMixedBytes = 24 * 1024;
static bool plan_tiles(Params* p) {
    const int sms = sm_count();
    const int64_t hbm = (int64_t(p->N) + p->T) * p->K * 2 / kHbmBytes;
    bool best_pair = false;
    int64_t best = INT64_MAX;
    const int fewest = ceil_div(p->T, kMaxTok);
    for (int pair = 0; pair < 2; ++pair) {
        const int unit = pair ? 32 : kChunk, groups = sms >> pair, n_tiles = ceil_div(p->N, kRows << pair);
        for (int tt = fewest; tt < fewest + 8 && (tt == fewest || tt <= ceil_div(p->T, unit)); ++tt) {
            const int tok = ceil_div(ceil_div(p->T, tt), unit) * unit;
            const int tiles = n_tiles * ceil_div(p->T, tok), rest = tiles % groups;
            const int load = (kABytes + (tok * kKBytes >> pair)) / kL2Bytes[pair], kb = tok * 2 > load ? tok * 2 : load;
            const int most = rest == 0 ? 1 : (groups / rest < kMaxParts ? (groups / rest < p->kbs ? groups / rest : p->kbs) : kMaxParts);
            for (int parts = 1; parts <= most; ++parts) {
                const int64_t kbs = int64_t(tiles / groups) * p->kbs + (rest > 0 ? ceil_div(p->kbs, parts) : 0);
                const int64_t tail = tok * kDrain + (parts > 1 ? kCount[pair] + parts * tok * kAdd : 0) + kPairing[pair], sum = kbs * kb;
                const int64_t cost = (sum > hbm ? sum + hbm / 2 : hbm + sum / 2) + tail;
                if (cost >= best) continue;
                best = cost, best_pair = pair != 0;
                p->tok = tok, p->n_tiles = n_tiles, p->tiles = tiles, p->groups = groups;
                p->whole = parts > 1 ? tiles - rest : tiles, p->parts = parts;
            }
        }
    }
    return best_pair;
}
static Layout plan(Params* p, int T, int N, int K, int R, bool* pair) {
    T = T > 0 ? T : 1;  // an empty batch is asked about like a row
    p->T = T, p->N = N, p->K = K, p->R = R;
    p->kbs = ceil_div(K, kKElems);
    const int sms = sm_count();
    *pair = plan_tiles(p);
    const int stage = kABytes + (*pair ? p->tok / 2 : p->tok) * kKBytes;
    // Few rows may each have an adapter of their own, whose B's come one after the other; of many some chunks where two requests meet
    const int slot = kRows * R * 2, room = (T <= kMixedRows ? kMixedBytes : kFewMixedBytes) / (2 * slot);
    p->slots = room < 1 ? 1 : room < kMaxSlots ? room : kMaxSlots;
    const int left = kRingBytes - 2 * p->slots * slot;
    p->stages = left / stage < kMaxStages ? left / stage : kMaxStages;
    Layout L{};
    size_t off = 0;
    auto add = [&](size_t bytes) {
        const size_t at = off;
        off += align_up(bytes, 256);
        return at;
    };
    // for the most that a call of fewer rows splits, so that a workspace for the longest batch serves all
    const int most = T < kMaxTok ? (T + 31) / 32 * 32 : kMaxTok;
    L.counters = add(size_t(sms) * sizeof(int));
    L.z = add(size_t(T) * R * 2);
    L.z_scale = add(size_t(T) * sizeof(float));
    L.part = add(size_t(sms) * most * kRows * sizeof(float));
    L.total = off;
    return L;
}

static int check_sizes(int64_t T, int N, int K, int L, int R) {
    DQ_CHECK(T >= 0 && N > 0 && K > 0 && L > 0 && R > 0);
    DQ_CHECK_FMT(R % 8 == 0 && R <= kMaxRank, "R=%d: a multiple of 8, at most %d (pad A and B with zeros)", R, kMaxRank);
    DQ_CHECK_FMT(K % 8 == 0, "K=%d: rows must be a multiple of 16 bytes", K);
    // tile numbers, K blocks and the rows of the tensor maps are 32-bit
    DQ_CHECK_FMT(T <= (1 << 24) && N <= (1 << 24) && K <= (1 << 24) && int64_t(L) * R < (int64_t(1) << 31) &&
                     int64_t(ceil_div(N, kRows)) * ((T + 15) / 16) < (int64_t(1) << 31),
                 "T=%lld N=%d K=%d L=%d: too large", (long long) T, N, K, L);
    return DQMOE_OK;
}

template <class K>
static int opt_in(K kern, int which, size_t bytes) {
    static std::mutex mu;
    static size_t configured[5][64] = {};
    int dev = 0;
    DQ_CUDA(cudaGetDevice(&dev));
    DQ_CHECK(dev >= 0 && dev < 64);
    std::lock_guard<std::mutex> lk(mu);
    if (configured[which][dev] < bytes) {
        DQ_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, int(bytes)));
        configured[which][dev] = bytes;
    }
    return DQMOE_OK;
}

// Rows form while what its blocks read of A (each row's adapter, whoever else has it) is a few microseconds' worth of L2.
constexpr int64_t kRowsFormBytes = 32 << 20;
static int launch_shrink(ShrinkParams p, const void* x, cudaStream_t stream) {
    if (p.T <= 256 && int64_t(p.T) * p.R * p.K * 2 <= kRowsFormBytes) {
        const dim3 grid(p.T, p.half ? 1 : ceil_div(p.R, kRowWarps));
        return p.half ? launch_pdl(lora_shrink_rows_kernel<true>, grid, kRowWarps * 32, 0, stream, p)
                      : launch_pdl(lora_shrink_rows_kernel<false>, grid, kRowWarps * 32, 0, stream, p);
    }
    // A tile's K is cut over a cluster, and its groups of adapters over several, as long as two blocks per SM are not reached, less an eighth, as
    // clusters of eight do not fill every part of the chip (288 blocks: the last clusters began after 9 us).
    const int tiles = ceil_div(p.T, kShrinkTok), room = 2 * sm_count() * 7 / 8, kbs = ceil_div(p.K, kKElems);
    int split = kMaxSplit;
    while (split > 1 && (tiles * split > room || split > kbs)) split /= 2;
    p.cap = kRows / 2 / p.R > 1 ? kRows / 2 / p.R : 1;
    const int most = ceil_div(p.L < kShrinkTok ? (p.L < p.T ? p.L : p.T) : (p.T < kShrinkTok ? p.T : kShrinkTok), p.cap);
    const int fit = room / (tiles * split);
    p.slots = fit < 1 ? 1 : fit < most ? fit : most;
    p.stages = kShrinkStages;
    while (p.stages > 2 && shrink_smem(p.R, p.cap, p.stages) > size_t(112) * 1024) --p.stages;  // two blocks per SM
    const size_t smem = shrink_smem(p.R, p.cap, p.stages);
    CUtensorMap xs, a;
    DQ_RC(make_map_2d(&xs, x, p.half != 0, p.T, p.K, p.ldx, kShrinkTok));
    DQ_RC(make_map_2d(&a, p.lora_a, p.half != 0, int64_t(p.L) * p.R, p.K, p.K, p.R));
    DQ_RC(opt_in(lora_shrink_tiles_kernel, 4, size_t(112) * 1024));
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(unsigned(tiles) * p.slots * split, 1, 1);
    cfg.blockDim = dim3(kShrinkThreads, 1, 1);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = unsigned(split);
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    DQ_CUDA(cudaLaunchKernelEx(&cfg, lora_shrink_tiles_kernel, xs, a, p));
    return DQMOE_OK;
}

template <bool kHalf, bool kPair>
static int launch_project(int groups, size_t smem, cudaStream_t stream, const CUtensorMap& x, const CUtensorMap& w, const CUtensorMap& z, const CUtensorMap& b,
                          const Params& p) {
    DQ_RC(opt_in(lora_project_kernel<kHalf, kPair>, (kHalf ? 1 : 0) + (kPair ? 2 : 0), kSmemBytes));
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(unsigned(groups) << (kPair ? 1 : 0), 1, 1);
    cfg.blockDim = dim3(kThreads, 1, 1);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = kPair ? 2 : 1;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = kPair ? 2 : 1;
    DQ_CUDA(cudaLaunchKernelEx(&cfg, lora_project_kernel<kHalf, kPair>, x, w, z, b, p));
    return DQMOE_OK;
}

}  // namespace lora
}  // namespace dq

using namespace dq;

extern "C" {

size_t dqmoe_lora_linear_workspace_bytes(int T, int N, int K, int L, int R) {
    if (lora::check_sizes(T, N, K, L, R) != DQMOE_OK) return 0;
    lora::Params p{};
    bool pair;
    return lora::plan(&p, T, N, K, R, &pair).total;
}

int dqmoe_lora_linear(const void* x, int64_t ldx, const void* w, const void* lora_a, const void* lora_b, const int32_t* ids, const float* scale,
                      const float* bias, void* y, int64_t ldy, void* workspace, size_t workspace_bytes, int T, int N, int K, int L, int R,
                      int type, dqmoe_stream_t stream_) {
    cudaStream_t stream = static_cast<cudaStream_t>(stream_);
    DQ_RC(lora::check_sizes(T, N, K, L, R));
    DQ_CHECK_FMT(type == DQMOE_DT_BF16 || type == DQMOE_DT_HALF, "type=%d: BF16 or HALF", type);
    if (T == 0) return DQMOE_OK;
    DQ_CHECK(x != nullptr && w != nullptr && lora_a != nullptr && lora_b != nullptr && ids != nullptr && y != nullptr);
    DQ_CHECK(is_aligned(x, 16) && is_aligned(w, 16) && is_aligned(lora_a, 16) && is_aligned(lora_b, 16) && is_aligned(y, 2) && is_aligned(ids, 4));
    DQ_CHECK(is_aligned(scale, 4) && is_aligned(bias, 4));
    DQ_CHECK_FMT(ldx >= K && ldx % 8 == 0 && ldx < (int64_t(1) << 36), "ldx=%lld: a multiple of 8, at least K", (long long) ldx);
    DQ_CHECK_FMT(ldy >= N, "ldy=%lld: at least N", (long long) ldy);
    DQ_CHECK_FMT(workspace != nullptr && is_aligned(workspace, 256), "workspace pointer %p is not aligned!", workspace);
    lora::Params p{};
    bool pair;
    const lora::Layout Y = lora::plan(&p, T, N, K, R, &pair);
    if (workspace_bytes != 0 && workspace_bytes < Y.total)
        return fail(DQMOE_ERR_WORKSPACE, __FILE__, __LINE__, "workspace_bytes >= dqmoe_lora_linear_workspace_bytes(...)",
                    "workspace has %zu bytes, the projection needs %zu", workspace_bytes, Y.total);
    const bool half = type == DQMOE_DT_HALF;
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    int* status = device_status_word();
    if (status == nullptr) return DQMOE_ERR_CUDA;

    lora::ShrinkParams sp{};
    sp.x = static_cast<const uint16_t*>(x), sp.ldx = ldx, sp.lora_a = static_cast<const uint16_t*>(lora_a);
    sp.ids = ids, sp.scale = scale;
    sp.z = reinterpret_cast<uint16_t*>(ws + Y.z), sp.z_scale = reinterpret_cast<float*>(ws + Y.z_scale);
    sp.counters = reinterpret_cast<int*>(ws + Y.counters);
    sp.n_counters = (p.tiles - p.whole) << (pair ? 1 : 0);
    sp.T = T, sp.K = K, sp.L = L, sp.R = R, sp.half = half, sp.status = status, sp.wait_limit = wait_limit();

    CUtensorMap xp, wm, zm, bm;
    DQ_RC(lora::make_map_2d(&xp, x, half, T, K, ldx, pair ? p.tok / 2 : p.tok));
    DQ_RC(lora::make_map_2d(&wm, w, half, N, K, K, lora::kRows));
    DQ_RC(lora::make_map_2d(&zm, sp.z, half, T, R, R, lora::kChunk));
    const cuuint64_t dim[3] = {cuuint64_t(R), cuuint64_t(N), cuuint64_t(L)}, stride[2] = {cuuint64_t(R) * 2, cuuint64_t(N) * R * 2};
    const cuuint32_t box[3] = {lora::kKElems, lora::kRows, 1};
    DQ_RC(lora::make_map(&bm, lora_b, half, 3, dim, stride, box));
    DQ_RC(lora::launch_shrink(sp, x, stream));
    p.ids = ids, p.lora_b = static_cast<const uint16_t*>(lora_b), p.z = sp.z, p.z_scale = half ? sp.z_scale : nullptr, p.bias = bias;
    p.y = static_cast<uint16_t*>(y), p.ldy = ldy, p.L = L;
    p.counters = sp.counters, p.part = reinterpret_cast<float*>(ws + Y.part), p.status = status, p.wait_limit = sp.wait_limit;
    const int split = (p.tiles - p.whole) * p.parts, busy = p.whole < p.groups ? (p.whole > split ? p.whole : split) : p.groups;
    const size_t smem = 1024 + size_t(p.stages) * (lora::kABytes + (pair ? p.tok / 2 : p.tok) * lora::kKBytes) + size_t(2) * p.slots * lora::kRows * R * 2 + sizeof(lora::Tail);
    if (half)
        return pair ? lora::launch_project<true, true>(busy, smem, stream, xp, wm, zm, bm, p) : lora::launch_project<true, false>(busy, smem, stream, xp, wm, zm, bm, p);
    return pair ? lora::launch_project<false, true>(busy, smem, stream, xp, wm, zm, bm, p) : lora::launch_project<false, false>(busy, smem, stream, xp, wm, zm, bm, p);
}

}  // extern "C"
