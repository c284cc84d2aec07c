/*
 * ops_quant.cuh -- one block of 128 values to e4m3 with an fp32 scale: scale = max(amax, 2^-100) / 448, q = e4m3(x / scale).
 * Division and conversion are rounded to nearest even, so any implementation of the formula gets the same bits.
 */
#pragma once
#include <cuda_fp8.h>
#include <math.h>
#include <stdint.h>

/* |b| joins the running amax; a NaN stays (max.NaN), so a block that holds one gets a NaN scale */
__device__ __forceinline__ float ops_amax(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(fabsf(b)));
    return r;
}


/* x / scale rounded to nearest, from inv = 1 / scale rounded to nearest: a quotient that is off by a step at most, its exact
 * remainder, and one correction (P. Markstein, "Computation of elementary functions on the IBM RISC System/6000
 * processor", 1990).  Three operations where the division routine takes a dozen and a branch; scales are at least
 * 2^-109, so nothing here leaves the range before the quotient has left e4m3's. */
__device__ __forceinline__ float ops_f8_quot(float x, float scale, float inv) {
    const float q = __fmul_rn(x, inv);
    return __fmaf_rn(__fmaf_rn(-q, scale, x), inv, q);
}

/* max(amax, 2^-100) / 448, rounded to nearest the same way (an infinite amax has no remainder: it stays) */
__device__ __forceinline__ float ops_f8_scale(float amax) {
    const float a = ops_amax(amax, 0x1p-100f), s = ops_f8_quot(a, 448.0f, 1.0f / 448.0f);
    return a < INFINITY ? s : a;
}

/* four numbers as e4m3, the first in the low byte */
__device__ __forceinline__ uint32_t ops_f8_pack4(float a, float b, float c, float d) {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
    return lo | (hi << 16);
}
