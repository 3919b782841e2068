// What the tcgen05 attention kernels over packed sequences and over the block cache share: products issued by a whole warp with one lane
// elected, and a bounded wait.
#pragma once
#include "attention_tile.cuh"

namespace {

// The issuer runs with all its lanes and one of them is elected by a predicate, never by a branch: descriptors then stay in uniform registers,
// where the instruction wants them. Behind a branch each product cost the thread 100 cycles, half as much again as the tensor core.
__device__ __forceinline__ void elected_ss(uint32_t elected, uint32_t tmem_d, uint32_t a, uint32_t a_high, uint32_t b, uint32_t b_high, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n.reg .pred p, e;\n.reg .b64 x, y;\nmov.b64 x, {%1, %2};\nmov.b64 y, {%3, %4};\nsetp.ne.b32 e, %7, 0;\nsetp.ne.b32 p, %6, 0;\n"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %5, p;\n}\n"
        ::"r"(tmem_d), "r"(a), "r"(a_high), "r"(b), "r"(b_high), "r"(idesc), "r"(accumulate), "r"(elected)
        : "memory");
}
__device__ __forceinline__ void elected_ts(uint32_t elected, uint32_t tmem_d, uint32_t tmem_a, uint32_t b, uint32_t b_high, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n.reg .pred p, e;\n.reg .b64 y;\nmov.b64 y, {%2, %3};\nsetp.ne.b32 e, %6, 0;\nsetp.ne.b32 p, %5, 0;\n"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], y, %4, p;\n}\n"
        ::"r"(tmem_d), "r"(tmem_a), "r"(b), "r"(b_high), "r"(idesc), "r"(accumulate), "r"(elected)
        : "memory");
}
__device__ __forceinline__ void elected_commit(uint32_t elected, uint32_t bar) {
    asm volatile("{\n.reg .pred e;\nsetp.ne.b32 e, %1, 0;\n@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}\n" ::"r"(bar), "r"(elected) : "memory");
}
__device__ __forceinline__ uint32_t uniform(uint32_t v) { return __shfl_sync(0xffffffffu, v, 0); }

// A wait of some seconds at most: in these kernels the others may have to wait while a warp does rows again or joins parts.
__device__ __forceinline__ bool long_wait(uint32_t bar, uint32_t parity, volatile uint32_t* abort_flag, uint32_t* status) {
    for (uint32_t it = 0; it < (1u << 25); ++it) {
        if (mbar_try_wait(bar, parity)) return true;
        if (*abort_flag) return false;
        if (it > 64) __nanosleep(64);
    }
    *abort_flag = 1;
    atomicOr(status, 4u);
    return false;
}

}  // namespace
