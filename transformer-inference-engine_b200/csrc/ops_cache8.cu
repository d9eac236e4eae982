// ops_cache8.cu -- key and value rows in 8 bits: quantised as they are stored into
// pages, and rows of pages of any format read back as fp32.
//
// A head's 64 elements of a row are kept as levels -127 .. 127 and one scale:
//   scale = max |x| / 127 in fp32,   level = x / scale to the nearest, ties to even,
// so the value that a level stands for is level * scale (the rule of the engine's
// int8 weights, k_quant.cu, with a scale per row and head). The reference keeps its
// one sequence's rows in fp32 only (src/kv_cache.c:150-190).
// Both directions move each byte once and are bound by memory: 16391 rows of 16 heads take 30 us to
// store (172 MB) and 28 to read back, 88 % of the copy rate (B200, 6506 GB/s); 256 rows
// of 12 heads 4 us each, which is a launch.
#include <cuda_bf16.h>

#include <climits>

#include "ops.h"
#include "quant.cuh"

namespace tie {
namespace {

constexpr int kThreads = 256;
constexpr int kLanes = 8;              // of a head's row: eight elements each

// Eight elements of a head's row to levels, by 8 lanes; what the row's scale is.
__device__ __forceinline__ uint2 quantise8(const float (&x)[8], float* scale) {
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, magnitude(x[i]));
#pragma unroll
    for (int o = 1; o < kLanes; o <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (top >= kNotFinite) {           // no value of the row is finite then
        *scale = __uint_as_float(0x7fffffffu);
        return make_uint2(0u, 0u);
    }
    const float s = __fdiv_rn(__uint_as_float(top), 127.f);
    *scale = s;
    if (s == 0.f) return make_uint2(0u, 0u);
    uint32_t q[8];
    levels_of(x, s, 127.f, q);
    return make_uint2(__byte_perm(__byte_perm(q[0], q[1], 0x0040), __byte_perm(q[2], q[3], 0x0040), 0x5410),
                      __byte_perm(__byte_perm(q[4], q[5], 0x0040), __byte_perm(q[6], q[7], 0x0040), 0x5410));
}

// A thread's place: row r, head h and the lane's eight elements.
struct Place {
    int r, h, lane;
    __device__ __forceinline__ Place(long long i, const Divisor& heads) {
        lane = (int)(i % kLanes);
        const int unit = (int)(i / kLanes);
        r = heads(unit);
        h = unit - r * heads.d;
    }
};

// Memory bound: 8 bytes in and 2 out for an element of keys and of values. 8 lanes take
// a head's row of both, eight elements of each a lane; they are in one warp.
template <int VEC>
__global__ void __launch_bounds__(kThreads)
kv_store_q8_kernel(const float* __restrict__ k, const float* __restrict__ v, int ld, const int32_t* __restrict__ slots,
                   long long n, Divisor heads, long long n_slots, int8_t* __restrict__ k_pages,
                   int8_t* __restrict__ v_pages, float* __restrict__ k_scales, float* __restrict__ v_scales) {
    const long long i = (long long)blockIdx.x * kThreads + threadIdx.x;
    const bool live = i < n;           // (all lanes take part in the shuffles)
    const Place at(live ? i : i % kLanes, heads);
    const size_t from = (size_t)at.r * ld + at.h * kHeadDim + 8 * at.lane;
    float x[8], y[8];
    load8<VEC>(k + from, x);
    load8<VEC>(v + from, y);
    const int slot = __ldg(slots + at.r);
    float sk, sv;
    const uint2 a = quantise8(x, &sk), b = quantise8(y, &sv);
    if (!live || slot < 0 || slot >= n_slots) return;
    const size_t to = (size_t)slot * heads.d * kHeadDim + at.h * kHeadDim + 8 * at.lane;
    *reinterpret_cast<uint2*>(k_pages + to) = a;
    *reinterpret_cast<uint2*>(v_pages + to) = b;
    if (at.lane == 0) {
        const size_t s = ((size_t)(slot / kPageRows) * heads.d + at.h) * kPageRows + slot % kPageRows;
        k_scales[s] = sk;
        v_scales[s] = sv;
    }
}

template <int FMT>
__device__ __forceinline__ void row8(const void* pages, const float* scales, size_t at, size_t scale_at, float (&x)[8]) {
    if constexpr (FMT == TIE_KV_F32) {
        load8<4>(static_cast<const float*>(pages) + at, x);
    } else if constexpr (FMT == TIE_KV_BF16) {
        const uint4 u = __ldg(reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(pages) + at));
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[2 * i] = __uint_as_float(w[i] << 16);
            x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
    } else {
        const uint2 u = __ldg(reinterpret_cast<const uint2*>(static_cast<const int8_t*>(pages) + at));
        const float s = __ldg(scales + scale_at);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = (float)(int8_t)((i < 4 ? u.x : u.y) >> (8 * (i & 3))) * s;
    }
}

// The way back, memory bound as well: a lane takes eight elements of a row of keys and
// of its row of values.
template <int FMT, int VEC>
__global__ void __launch_bounds__(kThreads)
kv_load_kernel(const int32_t* __restrict__ slots, long long n, Divisor heads, long long n_slots,
               const void* __restrict__ k_pages, const void* __restrict__ v_pages, const float* __restrict__ k_scales,
               const float* __restrict__ v_scales, float* __restrict__ k, float* __restrict__ v, int ld) {
    const long long i = (long long)blockIdx.x * kThreads + threadIdx.x;
    if (i >= n) return;
    const Place at(i, heads);
    const int slot = __ldg(slots + at.r);
    if (slot < 0 || slot >= n_slots) return;
    const size_t from = (size_t)slot * heads.d * kHeadDim + at.h * kHeadDim + 8 * at.lane;
    const size_t s = ((size_t)(slot / kPageRows) * heads.d + at.h) * kPageRows + slot % kPageRows;
    float x[8], y[8];
    row8<FMT>(k_pages, k_scales, from, s, x);
    row8<FMT>(v_pages, v_scales, from, s, y);
    const size_t to = (size_t)at.r * ld + at.h * kHeadDim + 8 * at.lane;
    store8<VEC>(k + to, x);
    store8<VEC>(v + to, y);
}

// What both entry points ask of the pool and of the rows.
model_status check(const float* k, const float* v, int ld, const int32_t* slots, int rows, const void* k_pages,
                   const void* v_pages, const float* k_scales, const float* v_scales, int n_kv_head) {
    if (!k_pages || !v_pages || rows < 0) return MODEL_ERR_ARG;
    if (rows && (!k || !v || !slots)) return MODEL_ERR_ARG;   // arrays without rows have no address
    if (ld < n_kv_head * kHeadDim || (ld & 3) || !aligned16(k) || !aligned16(v) || !aligned16(k_pages) ||
        !aligned16(v_pages) || !aligned16(k_scales) || !aligned16(v_scales))
        return MODEL_ERR_ARG;
    return MODEL_OK;
}

}  // namespace
}  // namespace tie

using namespace tie;

extern "C" model_status tie_kv_store_q8(const float* k, const float* v, int ld, const int32_t* slots, int rows,
                                        void* k_pages, void* v_pages, float* k_scales, float* v_scales, int n_pages,
                                        int n_kv_head, void* stream) {
    if (!pool_shape_ok(TIE_KV_F32, n_pages, n_kv_head) || !k_scales || !v_scales) return MODEL_ERR_ARG;
    const model_status bad = check(k, v, ld, slots, rows, k_pages, v_pages, k_scales, v_scales, n_kv_head);
    if (bad != MODEL_OK || rows == 0) return bad;
    OnDeviceOf dev(k_pages);
    if (dev.status() != MODEL_OK) return dev.status();
    if ((long long)rows * n_kv_head > INT_MAX) return MODEL_ERR_CAPACITY;
    const long long n = (long long)rows * n_kv_head * kLanes, blocks = (n + kThreads - 1) / kThreads;
    const bool wide = ld % 8 == 0 && aligned(k, 32) && aligned(v, 32);
    (wide ? kv_store_q8_kernel<8> : kv_store_q8_kernel<4>)<<<(unsigned)blocks, kThreads, 0, static_cast<cudaStream_t>(stream)>>>(
        k, v, ld, slots, n, divisor(n_kv_head), (long long)n_pages * kPageRows, static_cast<int8_t*>(k_pages),
        static_cast<int8_t*>(v_pages), k_scales, v_scales);
    TIE_OP_CU(cudaGetLastError());
    ++op_launches;
    return MODEL_OK;
}

extern "C" model_status tie_kv_load(const int32_t* slots, int rows, const void* k_pages, const void* v_pages,
                                    const float* k_scales, const float* v_scales, int kv_format, int n_pages,
                                    int n_kv_head, float* k, float* v, int ld, void* stream) {
    const bool q8 = kv_format == TIE_KV_INT8;
    if (!pool_shape_ok(q8 ? (int)TIE_KV_F32 : kv_format, n_pages, n_kv_head)) return MODEL_ERR_ARG;
    if (q8 ? !k_scales || !v_scales : k_scales || v_scales) return MODEL_ERR_ARG;
    const model_status bad = check(k, v, ld, slots, rows, k_pages, v_pages, k_scales, v_scales, n_kv_head);
    if (bad != MODEL_OK || rows == 0) return bad;
    OnDeviceOf dev(k_pages);
    if (dev.status() != MODEL_OK) return dev.status();
    if ((long long)rows * n_kv_head > INT_MAX) return MODEL_ERR_CAPACITY;
    const long long n = (long long)rows * n_kv_head * kLanes, blocks = (n + kThreads - 1) / kThreads;
    const bool wide = ld % 8 == 0 && aligned(k, 32) && aligned(v, 32);
    auto of = [&](auto* with8, auto* with4) { return wide ? with8 : with4; };
    auto* kernel = q8 ? of(kv_load_kernel<TIE_KV_INT8, 8>, kv_load_kernel<TIE_KV_INT8, 4>)
                      : kv_format == TIE_KV_BF16 ? of(kv_load_kernel<TIE_KV_BF16, 8>, kv_load_kernel<TIE_KV_BF16, 4>)
                                                 : of(kv_load_kernel<TIE_KV_F32, 8>, kv_load_kernel<TIE_KV_F32, 4>);
    kernel<<<(unsigned)blocks, kThreads, 0, static_cast<cudaStream_t>(stream)>>>(
        slots, n, divisor(n_kv_head), (long long)n_pages * kPageRows, k_pages, v_pages, k_scales, v_scales, k, v, ld);
    TIE_OP_CU(cudaGetLastError());
    ++op_launches;
    return MODEL_OK;
}
