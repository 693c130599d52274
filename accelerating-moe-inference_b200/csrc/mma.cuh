// Warp-level pieces of the 4-bit operators: m16n8k16 products with fp32
// accumulation, a transposition between lanes, approximate functions.
//
// Fragments of mma.m16n8k16 (lane = 4 g + j): A holds rows g, g + 8 and, per
// register, the column pairs 2 j, 2 j + 1 (a0 row g, a1 row g + 8) and 2 j + 8,
// 2 j + 9 (a2, a3); B holds column g, the row pairs 2 j.. (b0) and 2 j + 8..
// (b1); C holds rows g (c0, c1) and g + 8 (c2, c3), columns 2 j, 2 j + 1.  The
// order of the inner dimension is free as long as A and B agree on it.
#pragma once

#include <cstdint>
#include <cuda_runtime.h>

#include "ptx.cuh"

namespace moe {

__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// The first product of a sum: c = a b.
__device__ __forceinline__ void mma_f16_first(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%10, %10, %10, %10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
}

// An 8x8 matrix of 16-bit elements, lane 4 g + j holding row g, columns 2 j
// and 2 j + 1, transposed.
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
    uint32_t t;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(t) : "r"(v));
    return t;
}

// 1 / x within one unit in the last place, 2^x within two; subnormals as zero.
__device__ __forceinline__ float rcp_approx(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

}  // namespace moe
