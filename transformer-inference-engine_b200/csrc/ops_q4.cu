// ops_q4.cu -- 4-bit weights with group scales: made from fp32, read back, and their
// products with a few rows of activations (decode steps).
//
// A weight matrix W [n, k] (a row per output, as the engine holds its matrices) is cut
// along k into groups of 32, 64 or 128. A group is kept as levels -7 .. 7 and a scale:
//   scale = max |w| / 7 in fp32, rounded to bf16,   level = w / scale to the nearest,
// ties to even. In memory a row is blocks of 128 weights, 64 bytes each, the last one
// filled up with zeros: the 32-bit word 4 t + j of a block holds its weights 32 j + 8 t
// .. + 7, the level + 8 of weight 32 j + 8 t + i in bits 4 i .. 4 i + 3. So one 16-byte
// load gives lane t of four the 8 weights that it has of each 32, whatever the group.
// (The reference has fp32 weights only, src/model.c:331-467.)
#include <cuda_bf16.h>

#include <climits>

#include "ops.h"
#include "quant.cuh"

namespace tie {
namespace {

constexpr int kThreads = 256;
constexpr int kBlock = 128, kBlockBytes = kBlock / 2;
constexpr unsigned kAll = 0xffffffffu;

__host__ __device__ inline int blocks_of(int k) { return (k + kBlock - 1) / kBlock; }

// ------------------------------------------------------------ made, read back --
// Memory bound. 16 lanes take a block, 8 consecutive weights a lane.
template <bool VEC>
__device__ __forceinline__ void load8(const float* row, int c, int k, float (&x)[8]) {
    if (VEC && c + 8 <= k) {
        const float4 a = __ldcs(reinterpret_cast<const float4*>(row + c));
        const float4 b = __ldcs(reinterpret_cast<const float4*>(row + c) + 1);
        x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
        x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = c + i < k ? __ldg(row + c + i) : 0.f;
    }
}

template <bool VEC>
__global__ void __launch_bounds__(kThreads)
quantize_q4_kernel(const float* __restrict__ w, long long ldw, long long units, int k, int blocks, int lanes,
                   uint32_t* __restrict__ packed, __nv_bfloat16* __restrict__ scales, int groups) {
    const long long i = (long long)blockIdx.x * kThreads + threadIdx.x;
    const bool live = i < 16 * units;              // (all lanes take part in the shuffles)
    const long long unit = live ? i / 16 : 0;
    const long long row = unit / blocks;
    const int b = (int)(unit % blocks), l = (int)(i % 16);
    float x[8];
    load8<VEC>(w + row * ldw, b * kBlock + 8 * l, k, x);
    uint32_t top = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) top = max(top, magnitude(x[e]));
    for (int o = 1; o < lanes; o <<= 1) top = max(top, __shfl_xor_sync(kAll, top, o));
    const bool odd = top >= kNotFinite;            // a weight is not finite: no value of the group is
    const __nv_bfloat16 sb = odd ? __ushort_as_bfloat16((unsigned short)0x7fff)
                                 : __float2bfloat16_rn(__fdiv_rn(__uint_as_float(top), 7.f));
    const float s = __bfloat162float(sb);
    const float inv = reciprocal_of(s);
    uint32_t word = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const int q = odd || s == 0.f ? 0 : level_of(x[e], s, inv, 7.f);
        word |= (uint32_t)(q + 8) << (4 * e);
    }
    if (!live) return;
    packed[unit * 16 + 4 * (l % 4) + l / 4] = word;
    if (l % lanes == 0 && b * kBlock + 8 * l < k) scales[row * groups + (b * 16 + l) / lanes] = sb;
}

template <bool VEC>
__global__ void __launch_bounds__(kThreads)
dequantize_q4_kernel(const uint32_t* __restrict__ packed, const __nv_bfloat16* __restrict__ scales, long long units, int k,
                     int blocks, int lanes, int groups, float* __restrict__ w, long long ldw) {
    const long long i = (long long)blockIdx.x * kThreads + threadIdx.x;
    if (i >= 16 * units) return;
    const long long unit = i / 16, row = unit / blocks;
    const int b = (int)(unit % blocks), l = (int)(i % 16), c = b * kBlock + 8 * l;
    if (c >= k) return;
    const uint32_t word = __ldg(packed + unit * 16 + 4 * (l % 4) + l / 4);
    const float s = __bfloat162float(scales[row * groups + (b * 16 + l) / lanes]);
    float x[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = (float)((int)(word >> (4 * e) & 15u) - 8) * s;
    float* out = w + row * ldw + c;
    if (VEC && c + 8 <= k) {
        __stcs(reinterpret_cast<float4*>(out), make_float4(x[0], x[1], x[2], x[3]));
        __stcs(reinterpret_cast<float4*>(out) + 1, make_float4(x[4], x[5], x[6], x[7]));
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (c + e < k) out[e] = x[e];
    }
}

// ------------------------------------------------------------------- products --
// y[r] = act(x[r] W^T + bias) + residual[r] for up to 8 rows of x a CTA, on bf16 MMAs
// (m16n8k16): 16 rows of W are the A operand, the columns of B are rows of x. A level is
// exact in bf16, and an fp32 activation is exactly the sum of three bf16 terms (its 24
// bits in 8-bit pieces), so every product is exact and sums are fp32's: a group's sum of
// level * x in the MMA, times the group's scale, added in fp32. One or two rows of x put
// their terms into six of B's columns, one MMA for 16 weights of each row; up to 8 rows
// take three MMAs into the same sums.
//
// The k blocks of a tile are dealt to the CTA's warps, whose sums are added in order.
struct MatvecArgs {
    const float* x;
    long long ldx;
    int rows;
    const uint8_t* packed;
    const __nv_bfloat16* scales;
    int n, k, blocks, groups;
    const float* bias;
    const float* residual;
    long long ldr;
    int gelu;
    float* y;
    long long ldy;
};

constexpr int kWarps = kThreads / 32;

// Levels i and i + 4 of a word, for i = 0 .. 3, as pairs of bf16: 0x4300 | u is 128 + u.
__device__ __forceinline__ void levels8(uint32_t w, uint32_t (&p)[4]) {
    const __nv_bfloat162 off = __floats2bfloat162_rn(136.f, 136.f);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t u = ((w >> (4 * i)) & 0x000f000fu) | 0x43004300u;
        const __nv_bfloat162 v = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&u), off);
        p[i] = *reinterpret_cast<const uint32_t*>(&v);
    }
}

template <bool FEW, int MT, int G, bool VEC>
__global__ void __launch_bounds__(kThreads) matvec_q4_kernel(MatvecArgs a) {
    constexpr int kTerms = FEW ? 1 : 3;            // MMAs for each 16 weights
    __shared__ float s_sum[kWarps][MT * 16][9];
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5, g = lane >> 2, c = lane & 3;
    const int n0 = blockIdx.x * MT * 16, r0 = blockIdx.y * 8, rows = min(8, a.rows - r0);
    // the row of x that this lane's column of B stands for, and (FEW) which of its terms
    const int xr = FEW ? g / 3 : g, term = FEW ? g % 3 : 0;
    const bool real = xr < rows && (!FEW || g < 6);
    const float* x = a.x + (long long)(r0 + min(xr, rows - 1)) * a.ldx;
    float acc[MT][4] = {};
    for (int kb = warp; kb < a.blocks; kb += kWarps) {
        uint4 w[MT][2];
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int row = min(n0 + 16 * m + 8 * h + g, a.n - 1);
                w[m][h] = __ldg(reinterpret_cast<const uint4*>(a.packed + ((size_t)row * a.blocks + kb) * kBlockBytes) + c);
            }
        uint32_t b[kTerms][4][4];                  // [term][j][pair i, i + 4]
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            float v[8];
            load8<VEC>(x, kb * kBlock + 32 * j + 8 * c, real ? a.k : 0, v);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float lo = v[i], hi = v[i + 4];
                if constexpr (FEW) {
                    if (term) { lo = rest(lo); hi = rest(hi); }
                    if (term == 2) { lo = rest(lo); hi = rest(hi); }
                    b[0][j][i] = terms2(lo, hi);
                } else {
                    b[0][j][i] = terms2(lo, hi);
                    lo = rest(lo); hi = rest(hi);
                    b[1][j][i] = terms2(lo, hi);
                    b[2][j][i] = terms2(rest(lo), rest(hi));
                }
            }
        }
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            const uint32_t w0[4] = {w[m][0].x, w[m][0].y, w[m][0].z, w[m][0].w};
            const uint32_t w1[4] = {w[m][1].x, w[m][1].y, w[m][1].z, w[m][1].w};
#pragma unroll
            for (int j0 = 0; j0 < 4; j0 += G / 32) {
                float d[4] = {};
#pragma unroll
                for (int j = j0; j < j0 + G / 32; ++j) {
                    uint32_t p[4], q[4];
                    levels8(w0[j], p);
                    levels8(w1[j], q);
#pragma unroll
                    for (int i = 0; i < 4; i += 2) {
                        const uint32_t frag[4] = {p[i], q[i], p[i + 1], q[i + 1]};
#pragma unroll
                        for (int e = 0; e < kTerms; ++e) mma_bf16(d, frag, b[e][j][i], b[e][j][i + 1]);
                    }
                }
                const int grp = (kb * kBlock + 32 * j0) / G;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int row = min(n0 + 16 * m + 8 * h + g, a.n - 1);
                    const float s = grp < a.groups ? __bfloat162float(a.scales[(size_t)row * a.groups + grp]) : 0.f;
                    acc[m][2 * h] = fmaf(s, d[2 * h], acc[m][2 * h]);
                    acc[m][2 * h + 1] = fmaf(s, d[2 * h + 1], acc[m][2 * h + 1]);
                }
            }
        }
    }
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int e = 0; e < 4; ++e) s_sum[warp][16 * m + 8 * (e >> 1) + g][2 * c + (e & 1)] = acc[m][e];
    __syncthreads();
    for (int i = t; i < MT * 16 * rows; i += kThreads) {
        const int o = i % (MT * 16), r = i / (MT * 16), j = n0 + o;
        if (j >= a.n) continue;
        float sum = 0.f;
#pragma unroll
        for (int v = 0; v < kWarps; ++v) {
            if constexpr (FEW) sum += s_sum[v][o][3 * r] + (s_sum[v][o][3 * r + 1] + s_sum[v][o][3 * r + 2]);
            else sum += s_sum[v][o][r];
        }
        if (a.bias) sum = __fadd_rn(sum, __ldg(a.bias + j));
        if (a.gelu) sum = gelu_new_ref(sum);
        if (a.residual) sum = __fadd_rn(a.residual[(long long)(r0 + r) * a.ldr + j], sum);
        a.y[(long long)(r0 + r) * a.ldy + j] = sum;
    }
}

template <bool FEW, int MT, bool VEC>
void (*matvec_of(int group))(MatvecArgs) {
    return group == 32 ? matvec_q4_kernel<FEW, MT, 32, VEC>
                       : group == 64 ? matvec_q4_kernel<FEW, MT, 64, VEC> : matvec_q4_kernel<FEW, MT, 128, VEC>;
}
template <bool FEW, bool VEC>
void (*matvec_of(int mt, int group))(MatvecArgs) {
    return mt == 1 ? matvec_of<FEW, 1, VEC>(group) : mt == 2 ? matvec_of<FEW, 2, VEC>(group) : matvec_of<FEW, 4, VEC>(group);
}

// Shapes that the 4-bit entry points share.
bool q4_shape_ok(int n, int k, int group) {
    return n > 0 && k > 0 && (group == 32 || group == 64 || group == 128);
}
constexpr int kMostColumns = 1 << 24;              // a k whose block count and padded width stay far inside int32

}  // namespace
}  // namespace tie

using namespace tie;

extern "C" size_t tie_q4_bytes(int n, int k) {
    return n > 0 && k > 0 ? (size_t)n * ((size_t)(k - 1) / kBlock + 1) * kBlockBytes : 0;
}

extern "C" model_status tie_quantize_q4(const float* w, long long ldw, int n, int k, int group, void* packed, void* scales,
                                        void* stream) {
    if (!w || !packed || !scales || !q4_shape_ok(n, k, group) || ldw < k) return MODEL_ERR_ARG;
    if (!aligned(w, 4) || !aligned16(packed) || !aligned(scales, 2)) return MODEL_ERR_ARG;
    const long long units = (long long)n * blocks_of(k), grid = (16 * units + kThreads - 1) / kThreads;
    if (k > kMostColumns || grid > INT_MAX) return MODEL_ERR_CAPACITY;
    OnDeviceOf dev(packed);
    if (dev.status() != MODEL_OK) return dev.status();
    const bool vec = aligned16(w) && ldw % 4 == 0;
    (vec ? quantize_q4_kernel<true> : quantize_q4_kernel<false>)<<<(unsigned)grid, kThreads, 0, static_cast<cudaStream_t>(stream)>>>(
        w, ldw, units, k, blocks_of(k), group / 8, static_cast<uint32_t*>(packed), static_cast<__nv_bfloat16*>(scales),
        (k + group - 1) / group);
    TIE_OP_CU(cudaGetLastError());
    ++op_launches;
    return MODEL_OK;
}

extern "C" model_status tie_dequantize_q4(const void* packed, const void* scales, int n, int k, int group, float* w,
                                          long long ldw, void* stream) {
    if (!w || !packed || !scales || !q4_shape_ok(n, k, group) || ldw < k) return MODEL_ERR_ARG;
    if (!aligned(w, 4) || !aligned16(packed) || !aligned(scales, 2)) return MODEL_ERR_ARG;
    const long long units = (long long)n * blocks_of(k), grid = (16 * units + kThreads - 1) / kThreads;
    if (k > kMostColumns || grid > INT_MAX) return MODEL_ERR_CAPACITY;
    OnDeviceOf dev(w);
    if (dev.status() != MODEL_OK) return dev.status();
    const bool vec = aligned16(w) && ldw % 4 == 0;
    (vec ? dequantize_q4_kernel<true> : dequantize_q4_kernel<false>)<<<(unsigned)grid, kThreads, 0, static_cast<cudaStream_t>(stream)>>>(
        static_cast<const uint32_t*>(packed), static_cast<const __nv_bfloat16*>(scales), units, k, blocks_of(k), group / 8,
        (k + group - 1) / group, w, ldw);
    TIE_OP_CU(cudaGetLastError());
    ++op_launches;
    return MODEL_OK;
}

extern "C" model_status tie_matvec_q4(const float* x, long long ldx, int rows, const void* packed, const void* scales, int n,
                                      int k, int group, const float* bias, const float* residual, long long ldr, int gelu,
                                      float* y, long long ldy, void* stream) {
    if (!packed || !scales || rows < 0 || !q4_shape_ok(n, k, group)) return MODEL_ERR_ARG;
    if (rows && (!x || !y)) return MODEL_ERR_ARG;             // arrays without rows have no address
    if (ldx < k || ldy < n || (residual && ldr < n) || (gelu != 0 && gelu != 1)) return MODEL_ERR_ARG;
    if (!aligned(x, 4) || !aligned(y, 4) || !aligned(bias, 4) || !aligned(residual, 4) || !aligned16(packed) ||
        !aligned(scales, 2))
        return MODEL_ERR_ARG;
    if (k > kMostColumns || rows > 8 * 65535) return MODEL_ERR_CAPACITY;
    if (rows == 0) return MODEL_OK;
    OnDeviceOf dev(y);
    if (dev.status() != MODEL_OK) return dev.status();
    MatvecArgs a{x, ldx, rows, static_cast<const uint8_t*>(packed), static_cast<const __nv_bfloat16*>(scales), n, k,
                 blocks_of(k), (k + group - 1) / group, bias, residual, ldr, gelu, y, ldy};
    const int tiles = (n - 1) / 16 + 1, sms = sm_count(dev.device());
    const int mt = tiles >= 8 * sms ? 4 : tiles >= 2 * sms ? 2 : 1;
    const bool vec = aligned16(x) && ldx % 4 == 0;
    auto* kernel = rows <= 2 ? (vec ? matvec_of<true, true>(mt, group) : matvec_of<true, false>(mt, group))
                             : (vec ? matvec_of<false, true>(mt, group) : matvec_of<false, false>(mt, group));
    kernel<<<dim3((unsigned)((tiles - 1) / mt + 1), (unsigned)((rows - 1) / 8 + 1)), kThreads, 0,
             static_cast<cudaStream_t>(stream)>>>(a);
    TIE_OP_CU(cudaGetLastError());
    ++op_launches;
    return MODEL_OK;
}
