// quant.cuh -- levels and scales of values held in few bits, and fp32 values as sums of
// bf16 terms, which the kernels over them share.
#pragma once

#include <cuda_runtime.h>

#include <cstdint>

namespace tie {

// Magnitudes compare as their bits do, infinity above what is finite and NaN above both.
constexpr uint32_t kNotFinite = 0x7f800000u;
__device__ __forceinline__ uint32_t magnitude(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// the larger magnitude; NaN if either is
__device__ __forceinline__ float max_abs(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(fabsf(a)), "f"(fabsf(b)));
    return r;
}

__device__ __forceinline__ float max_abs3(float a, float b, float c) {
    float r;
    asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

// Two fp32 numbers in one instruction, rounded as each alone would be.
struct Float2x {
    unsigned long long v;
    __device__ __forceinline__ Float2x() {}
    __device__ __forceinline__ explicit Float2x(unsigned long long of) : v(of) {}
    __device__ __forceinline__ Float2x(float lo, float hi) { asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(lo), "f"(hi)); }
    __device__ __forceinline__ void get(float& lo, float& hi) const { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v)); }
};
__device__ __forceinline__ Float2x operator+(Float2x a, Float2x b) {
    Float2x c;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(c.v) : "l"(a.v), "l"(b.v));
    return c;
}
__device__ __forceinline__ Float2x operator*(Float2x a, Float2x b) {
    Float2x c;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(c.v) : "l"(a.v), "l"(b.v));
    return c;
}
__device__ __forceinline__ Float2x fma2(Float2x a, Float2x b, Float2x c) {
    Float2x d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d.v) : "l"(a.v), "l"(b.v), "l"(c.v));
    return d;
}
// 1 / s to one place, 0 where s is so small that its reciprocal may be beyond fp32.
__device__ __forceinline__ float reciprocal_of(float s) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(s));
    return s < 0x1p-100f ? 0.f : r;
}

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

// Levels of N numbers as integers added to kLevelBase (the bits of 1.5 2^23): all of them that are
// clearly nearest to one, which a product with 1 / s tells (its error is below 2^-15 of a level);
// the others, about one of 20,000, by level_of.
constexpr uint32_t kLevelBase = 0x4b400000u;
template <int N>
__device__ __forceinline__ void levels_of(const float (&x)[N], float s, float most, uint32_t (&level)[N]) {
    static_assert(N % 2 == 0, "pairs");
    const float inv = reciprocal_of(s), base = __uint_as_float(kLevelBase);
    const Float2x inv2(inv, inv), base2(base, base), less2(-base, -base), minus2(-1.f, -1.f);
    float far = 0.f;
#pragma unroll
    for (int i = 0; i < N; i += 2) {
        const Float2x t = Float2x(x[i], x[i + 1]) * inv2, y = t + base2;
        float y0, y1, e0, e1;
        y.get(y0, y1);
        fma2(y + less2, minus2, t).get(e0, e1);
        level[i] = __float_as_uint(y0);
        level[i + 1] = __float_as_uint(y1);
        far = max_abs3(far, e0, e1);
    }
    if (far > 0.49996f || inv == 0.f) {
#pragma unroll
        for (int i = 0; i < N; ++i) level[i] = kLevelBase + (uint32_t)level_of(x[i], s, inv, most);
    }
}

// 8 fp32 side by side: 32-byte aligned (VEC 8), 16-byte aligned (4) or anywhere (0)
template <int VEC>
__device__ __forceinline__ void load8(const float* p, float (&x)[8]) {
    if constexpr (VEC == 8) {
        asm volatile("ld.global.nc.L1::no_allocate.v8.f32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                     : "=f"(x[0]), "=f"(x[1]), "=f"(x[2]), "=f"(x[3]), "=f"(x[4]), "=f"(x[5]), "=f"(x[6]), "=f"(x[7])
                     : "l"(p));
    } else if constexpr (VEC == 4) {
        const float4 a = __ldg(reinterpret_cast<const float4*>(p)), b = __ldg(reinterpret_cast<const float4*>(p) + 1);
        x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
        x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = __ldg(p + i);
    }
}
template <int VEC>
__device__ __forceinline__ void store8(float* p, const float (&x)[8]) {
    if constexpr (VEC == 8) {
        asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "f"(x[0]), "f"(x[1]), "f"(x[2]),
                     "f"(x[3]), "f"(x[4]), "f"(x[5]), "f"(x[6]), "f"(x[7])
                     : "memory");
    } else if constexpr (VEC == 4) {
        reinterpret_cast<float4*>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
        reinterpret_cast<float4*>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) p[i] = x[i];
    }
}

// n / d for 0 <= n < 2^31 (the multiplier is 2^(32 + shift) / d, rounded up, less 2^32)
struct Divisor {
    int d, shift;
    unsigned mul;
    __device__ __forceinline__ int operator()(int n) const { return (int)((__umulhi(mul, (unsigned)n) + (unsigned)n) >> shift); }
};
inline Divisor divisor(int d) {
    int shift = 0;
    while ((1LL << shift) < d) ++shift;
    return Divisor{d, shift, (unsigned)(((1ULL << 32) * ((1ULL << shift) - (unsigned long long)d)) / (unsigned long long)d + 1)};
}

// An fp32 value is the sum of three bf16 terms, its 24 bits in pieces of 8: the term is
// the value's upper half, the rest is exact. (A value that is not finite has a rest that
// is NaN.)
__device__ __forceinline__ float rest(float x) { return x - __uint_as_float(__float_as_uint(x) & 0xffff0000u); }
// the terms of two values side by side
__device__ __forceinline__ uint32_t terms2(float lo, float hi) {
    return __byte_perm(__float_as_uint(lo), __float_as_uint(hi), 0x7632);
}

// rest() of two values
__device__ __forceinline__ void rest2(float& lo, float& hi) {
    const Float2x less(__uint_as_float((__float_as_uint(lo) & 0xffff0000u) ^ 0x80000000u),
                       __uint_as_float((__float_as_uint(hi) & 0xffff0000u) ^ 0x80000000u));
    (Float2x(lo, hi) + less).get(lo, hi);
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
