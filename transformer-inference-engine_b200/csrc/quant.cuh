// quant.cuh -- levels and scales of values held in few bits, and fp32 values as sums of
// bf16 terms, which the kernels over them share.
#pragma once

#include <cuda_runtime.h>

#include <cstdint>

namespace tie {

// Magnitudes compare as their bits do, infinity above what is finite and NaN above both.
constexpr uint32_t kNotFinite = 0x7f800000u;
__device__ __forceinline__ uint32_t magnitude(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// 1 / s for level_of, 0 where s is so small that its reciprocal may be beyond fp32.
__device__ __forceinline__ float reciprocal_of(float s) { return s < 0x1p-120f ? 0.f : __frcp_rn(s); }

// The level of x at scale s > 0: the integer nearest to the exact quotient, ties to even,
// within +-most. The approximate quotient's nearest integer q is off by one at most; the
// remainder x - q s is exact and tells.
__device__ __forceinline__ int level_of(float x, float s, float inv, float most) {
    const float q0 = fminf(most, fmaxf(-most, rintf(inv > 0.f ? x * inv : __fdiv_rn(x, s))));
    const float r = fmaf(-q0, s, x), r2 = r + r;
    const bool odd = (int)q0 & 1;
    float q = q0;
    if (r2 > s || (r2 == s && odd)) q += 1.f;
    if (r2 < -s || (r2 == -s && odd)) q -= 1.f;
    return (int)fminf(most, fmaxf(-most, q));
}

// An fp32 value is the sum of three bf16 terms, its 24 bits in pieces of 8: the term is
// the value's upper half, the rest is exact. (A value that is not finite has a rest that
// is NaN.)
__device__ __forceinline__ float rest(float x) { return x - __uint_as_float(__float_as_uint(x) & 0xffff0000u); }
// the terms of two values side by side
__device__ __forceinline__ uint32_t terms2(float lo, float hi) {
    return __byte_perm(__float_as_uint(lo), __float_as_uint(hi), 0x7632);
}

// d = c + a b on bf16 (m16n8k16), fp32 sums
__device__ __forceinline__ void mma_bf16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, const float (&c)[4]) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
                 "{%10, %11, %12, %13};"
                 : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
}
__device__ __forceinline__ void mma_bf16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    mma_bf16(d, a, b0, b1, d);
}

}  // namespace tie
