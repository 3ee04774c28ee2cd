// What the kernels that work in 8 bits share: e4m3 conversions, the scale of a block of numbers, and products of e4m3 fragments on
// mma.sync.
//
// A block of numbers (128 neighbours of a row, 128 x 128 of a weight, one head of a key or value) with largest magnitude A is kept as
// q = e4m3(x (1 / s)), s = max(A, 2^-100) / 448, both quotients and the product rounded to float32: the largest becomes +-448, the
// largest e4m3 value, a rounding is off by at most 2^-4 of the number down to 2^-6 s (the smallest normal e4m3) and by 2^-10 s below,
// give or take 2^-22 of the number: where x / s lies that near to the middle of two e4m3 values, either may be taken.  (A division per
// number in place of the product: 2048 x 12288 rows 21.1 us for 14.5, eight rows by 6144 x 4096 13.4 for 9.0; the product and its
// remainder added back, which gives the rounded quotient, 16.1 and 9.6.)  The floor under A keeps s and 1 / s normal, so a block of
// zeros becomes zeros.  An infinity makes the block's s infinite and itself NaN, a NaN becomes NaN: the sums that meet them are NaN.
#pragma once

#include <cuda_fp16.h>

#include "common.cuh"

namespace tllm {

constexpr int kFp8Block = 128;                   // columns (and weight rows) that share a scale
constexpr float kE4m3Max = 448.0f;
constexpr float kFp8Floor = 7.888609052210118e-31f;    // 2^-100

__device__ __forceinline__ float fp8_scale(float largest) { return fmaxf(largest, kFp8Floor) / kE4m3Max; }

// Two float32 numbers as e4m3 (nearest, ties to even, held within +-448), lo in the low byte.
__device__ __forceinline__ uint32_t to_e4m3x2(float lo, float hi) {
    uint16_t d;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;\n" : "=h"(d) : "f"(hi), "f"(lo));
    return d;
}
__device__ __forceinline__ uint32_t to_e4m3x4(float a, float b, float c, float d) {
    return to_e4m3x2(a, b) | (to_e4m3x2(c, d) << 16);
}
// Eight neighbours times `inv`, packed.
__device__ __forceinline__ uint2 to_e4m3x8(const float (&v)[8], float inv) {
    return make_uint2(to_e4m3x4(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv),
                      to_e4m3x4(v[4] * inv, v[5] * inv, v[6] * inv, v[7] * inv));
}
// Two e4m3 numbers (the low or high half of a word) as a pair of float16, which hold every e4m3 value exactly.
__device__ __forceinline__ uint32_t e4m3x2_to_half2(uint32_t pair) {
    uint32_t d;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;\n" : "=r"(d) : "h"((uint16_t)pair));
    return d;
}

// Four at once: the low and the high half of a word.
__device__ __forceinline__ void e4m3x4_to_half2(uint32_t word, uint32_t& lo, uint32_t& hi) {
    asm("{\n\t.reg .b16 l, h;\n\t"
        "mov.b32 {l, h}, %2;\n\t"
        "cvt.rn.f16x2.e4m3x2 %0, l;\n\t"
        "cvt.rn.f16x2.e4m3x2 %1, h;\n\t}\n"
        : "=r"(lo), "=r"(hi)
        : "r"(word));
}

// D[16x8] += A[16x16] . B[16x8], float16 operands, float32 sums.
__device__ __forceinline__ void mma_f16_16816(float (&d)[4], const uint32_t (&a)[4], const uint32_t (&b)[2]) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
        "{%0,%1,%2,%3};\n"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}

// Thread blocks of a cluster.
__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;\n" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;\n" ::: "memory");
}

// Sixteen lanes that hold eight neighbours each: the largest of their 128 (all 32 lanes take part).
__device__ __forceinline__ float half_warp_max(float v) {
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}

__device__ __forceinline__ float largest8(const float (&v)[8]) {
    float a = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) a = fmaxf(a, fabsf(v[i]));
    return a;
}

}  // namespace tllm
