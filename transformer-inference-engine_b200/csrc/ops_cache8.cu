// ops_cache8.cu -- key and value rows in 8 bits: quantised as they are stored into
// pages, and rows of pages of any format read back as fp32.
//
// A head's 64 elements of a row are kept as levels -127 .. 127 and one scale:
//   scale = max |x| / 127 in fp32,   level = x / scale to the nearest, ties to even,
// so the value that a level stands for is level * scale (the rule of the engine's
// int8 weights, k_quant.cu, with a scale per row and head). The reference keeps its
// one sequence's rows in fp32 only (src/kv_cache.c:150-190).
#include <cuda_bf16.h>

#include <climits>

#include "ops.h"
#include "quant.cuh"

namespace tie {
namespace {

constexpr int kThreads = 256;
constexpr int kLanes = 16;             // of a head's row: four elements each

// Four elements of a head's row to levels, by 16 lanes; what the row's scale is.
__device__ __forceinline__ uint32_t quantise4(const float4& x, float* scale) {
    const float v[4] = {x.x, x.y, x.z, x.w};
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) top = max(top, magnitude(v[i]));
#pragma unroll
    for (int o = 1; o < kLanes; o <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (top >= kNotFinite) {           // no value of the row is finite then
        *scale = __uint_as_float(0x7fffffffu);
        return 0u;
    }
    const float s = __fdiv_rn(__uint_as_float(top), 127.f);
    *scale = s;
    if (s == 0.f) return 0u;
    const float inv = reciprocal_of(s);
    uint32_t w = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) w |= ((uint32_t)level_of(v[i], s, inv, 127.f) & 255u) << (8 * i);
    return w;
}

// Memory bound: 8 bytes in and 2 out for an element of keys and of values. 16 lanes take
// a head's row of both, four elements of each a lane; they are in one warp.
__global__ void __launch_bounds__(kThreads)
kv_store_q8_kernel(const float* __restrict__ k, const float* __restrict__ v, int ld, const int32_t* __restrict__ slots,
                   long long n, int heads, long long n_slots, int8_t* __restrict__ k_pages,
                   int8_t* __restrict__ v_pages, float* __restrict__ k_scales, float* __restrict__ v_scales) {
    const long long i = (long long)blockIdx.x * kThreads + threadIdx.x;
    const bool live = i < n;           // (all lanes take part in the shuffles)
    const int lane = (int)(i % kLanes);
    const long long unit = live ? i / kLanes : 0;
    const int r = (int)(unit / heads), h = (int)(unit % heads);
    const size_t from = (size_t)r * ld + h * kHeadDim + 4 * lane;
    const float4 x = __ldcs(reinterpret_cast<const float4*>(k + from));
    const float4 y = __ldcs(reinterpret_cast<const float4*>(v + from));
    const int slot = __ldg(slots + r);
    float sk, sv;
    const uint32_t a = quantise4(x, &sk), b = quantise4(y, &sv);
    if (!live || slot < 0 || slot >= n_slots) return;
    const size_t to = (size_t)slot * heads * kHeadDim + h * kHeadDim + 4 * lane;
    *reinterpret_cast<uint32_t*>(k_pages + to) = a;
    *reinterpret_cast<uint32_t*>(v_pages + to) = b;
    if (lane == 0) {
        const size_t at = ((size_t)(slot / kPageRows) * heads + h) * kPageRows + slot % kPageRows;
        k_scales[at] = sk;
        v_scales[at] = sv;
    }
}

template <int FMT>
__device__ __forceinline__ float4 row4(const void* pages, const float* scales, size_t at, size_t scale_at) {
    if constexpr (FMT == TIE_KV_F32) {
        return __ldg(reinterpret_cast<const float4*>(static_cast<const float*>(pages) + at));
    } else if constexpr (FMT == TIE_KV_BF16) {
        const uint2 u = __ldg(reinterpret_cast<const uint2*>(static_cast<const __nv_bfloat16*>(pages) + at));
        return make_float4(__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xffff0000u), __uint_as_float(u.y << 16),
                           __uint_as_float(u.y & 0xffff0000u));
    } else {
        const char4 u = __ldg(reinterpret_cast<const char4*>(static_cast<const int8_t*>(pages) + at));
        const float s = __ldg(scales + scale_at);
        return make_float4(u.x * s, u.y * s, u.z * s, u.w * s);
    }
}

// The way back, memory bound as well: a lane takes four elements of a row of keys and
// of its row of values.
template <int FMT>
__global__ void __launch_bounds__(kThreads)
kv_load_kernel(const int32_t* __restrict__ slots, long long n, int heads, long long n_slots,
               const void* __restrict__ k_pages, const void* __restrict__ v_pages, const float* __restrict__ k_scales,
               const float* __restrict__ v_scales, float* __restrict__ k, float* __restrict__ v, int ld) {
    const long long i = (long long)blockIdx.x * kThreads + threadIdx.x;
    if (i >= n) return;
    const int lane = (int)(i % kLanes);
    const long long unit = i / kLanes;
    const int r = (int)(unit / heads), h = (int)(unit % heads);
    const int slot = __ldg(slots + r);
    if (slot < 0 || slot >= n_slots) return;
    const size_t from = (size_t)slot * heads * kHeadDim + h * kHeadDim + 4 * lane;
    const size_t at = ((size_t)(slot / kPageRows) * heads + h) * kPageRows + slot % kPageRows;
    const float4 x = row4<FMT>(k_pages, k_scales, from, at), y = row4<FMT>(v_pages, v_scales, from, at);
    const size_t to = (size_t)r * ld + h * kHeadDim + 4 * lane;
    __stcs(reinterpret_cast<float4*>(k + to), x);
    __stcs(reinterpret_cast<float4*>(v + to), y);
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
    const long long n = (long long)rows * n_kv_head * kLanes, blocks = (n + kThreads - 1) / kThreads;
    if (blocks > INT_MAX) return MODEL_ERR_CAPACITY;
    kv_store_q8_kernel<<<(unsigned)blocks, kThreads, 0, static_cast<cudaStream_t>(stream)>>>(
        k, v, ld, slots, n, n_kv_head, (long long)n_pages * kPageRows, static_cast<int8_t*>(k_pages),
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
    const long long n = (long long)rows * n_kv_head * kLanes, blocks = (n + kThreads - 1) / kThreads;
    if (blocks > INT_MAX) return MODEL_ERR_CAPACITY;
    auto* kernel = q8 ? kv_load_kernel<TIE_KV_INT8>
                      : kv_format == TIE_KV_BF16 ? kv_load_kernel<TIE_KV_BF16> : kv_load_kernel<TIE_KV_F32>;
    kernel<<<(unsigned)blocks, kThreads, 0, static_cast<cudaStream_t>(stream)>>>(
        slots, n, n_kv_head, (long long)n_pages * kPageRows, k_pages, v_pages, k_scales, v_scales, k, v, ld);
    TIE_OP_CU(cudaGetLastError());
    ++op_launches;
    return MODEL_OK;
}
