// Packed fp32 arithmetic (f32x2 instructions), shared by the decay attention and
// beam kernels.
#pragma once

#include "common.cuh"

namespace mb2 {

// two fp32 values in one register pair (packed FMA: half the instructions)
__device__ __forceinline__ uint64_t pair(uint32_t lo, uint32_t hi) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "r"(lo), "r"(hi));
    return r;
}
__device__ __forceinline__ uint64_t pair(float v) {
    return pair(__float_as_uint(v), __float_as_uint(v));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint32_t lo_of(uint64_t v) { return (uint32_t)v; }
__device__ __forceinline__ uint32_t hi_of(uint64_t v) { return (uint32_t)(v >> 32); }

}  // namespace mb2
