// A list of tiles of equal length, cut into equal shares of their concatenated K steps ("units"): what the kernels with few output
// tiles use to give every SM the same bytes (moe_decode.cu, lora.cu). A tile that several shares take part in is finished by the
// block that completes its part last: each writes its partial sums, counts itself in, and the last one adds all parts in the order of
// the shares, so the result does not depend on which block that was.
#pragma once

#include <stdint.h>

#include "common.cuh"

namespace dq {
namespace streamk {

// first unit of share g of `shares` over `units`; shares [first(g), first(g + 1))
__device__ __forceinline__ int first_unit(int g, int shares, int units) { return int(int64_t(g) * units / shares); }
// the share that unit u lies in: the largest g with first_unit(g) <= u
__device__ __forceinline__ int share_of(int u, int shares, int units) { return int((int64_t(u + 1) * shares - 1) / units); }

__device__ __forceinline__ int ld_acquire_gpu(const int* p) {
    int v;
    asm volatile("ld.acquire.gpu.global.s32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
    return v;
}
__device__ __forceinline__ int atomic_add_acq_rel_gpu(int* p, int v) {
    int old;
    asm volatile("atom.add.acq_rel.gpu.global.s32 %0, [%1], %2;" : "=r"(old) : "l"(p), "r"(v) : "memory");
    return old;
}
__device__ __forceinline__ void red_add_release_gpu(int* p, int v) {
    asm volatile("red.release.gpu.global.add.s32 [%0], %1;" ::"l"(p), "r"(v) : "memory");
}
// Partial sums pass between blocks through L2 only.
__device__ __forceinline__ float4 ld_partial4(const float* p) {
    float4 v;
    asm volatile("ld.relaxed.gpu.global.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "l"(p) : "memory");
    return v;
}

}  // namespace streamk
}  // namespace dq
