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
#include <type_traits>

#include "ops.h"
#include "quant.cuh"

namespace tie {
namespace {

constexpr int kThreads = 256;         // of the kernels that make weights and read them back
constexpr int kBlock = 128, kBlockBytes = kBlock / 2;
constexpr unsigned kAll = 0xffffffffu;

__host__ __device__ inline int blocks_of(int k) { return (k + kBlock - 1) / kBlock; }

// ------------------------------------------------------------ made, read back --
// 16 lanes take a block, 8 consecutive weights a lane. 50257 x 1600 (322 MB in fp32, 42 MB packed)
// takes 74 us to make, where finding the levels holds memory to 4.9 TB/s, and 60 to read back (6.1).
// (With IEEE quotients and reciprocals, and levels one by one, making took 90.)
// Weights c .. c + 7 of a row of k, zeros behind it.
template <int VEC>
__device__ __forceinline__ void weights8(const float* row, int c, int k, float (&x)[8]) {
    if (VEC && c + 8 <= k) {
        load8<VEC>(row + c, x);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = c + i < k ? __ldg(row + c + i) : 0.f;
    }
}

// top / 7, rounded to fp32 and then to bf16. The product with 1 / 7 is off by less than two of fp32's last places,
// which matters only next to a tie of bf16.
__device__ __forceinline__ unsigned short seventh(float top) {
    float y = top * (1.f / 7.f);
    if (((__float_as_uint(y) + 0x8004u) & 0xffffu) < 8u || y < 0x1p-100f) y = __fdiv_rn(top, 7.f);
    return __bfloat16_as_ushort(__float2bfloat16_rn(y));
}

// Blocks per 16 lanes: both are loaded before either is used (50257 x 1600 made and read back, a block
// at a time: 140 us, two: 134, four: 143).
constexpr int kUnits = 2;

template <int VEC>
__global__ void __launch_bounds__(kThreads)
quantize_q4_kernel(const float* __restrict__ w, long long ldw, int units, int k, Divisor blocks, int shift,
                   uint32_t* __restrict__ packed, __nv_bfloat16* __restrict__ scales, int groups) {
    const int l = threadIdx.x % 16;
    const unsigned first = blockIdx.x * (kThreads / 16 * kUnits) + threadIdx.x / 16;
    float x[kUnits][8];
    int row[kUnits], c[kUnits];
#pragma unroll
    for (int j = 0; j < kUnits; ++j) {
        // (all lanes take part in the shuffles)
        const int unit = (int)min(first + j * (kThreads / 16), (unsigned)units - 1u);
        row[j] = blocks(unit);
        c[j] = (unit - row[j] * blocks.d) * kBlock + 8 * l;
        weights8<VEC>(w + (long long)row[j] * ldw, c[j], k, x[j]);
    }
#pragma unroll
    for (int j = 0; j < kUnits; ++j) {
        float top = 0.f;
#pragma unroll
        for (int e = 0; e < 8; e += 2) top = max_abs3(top, x[j][e], x[j][e + 1]);
#pragma unroll
        for (int o = 0; o < 4; ++o)
            if (o < shift) top = max_abs(top, __shfl_xor_sync(kAll, top, 1 << o));
        const bool odd = !(top < INFINITY);        // a weight is not finite: no value of the group is
        const unsigned short sb = odd ? (unsigned short)0x7fff : seventh(top);
        const float s = __uint_as_float((uint32_t)sb << 16);
        uint32_t word = 0x88888888u;               // zeros
        if (!odd && s != 0.f) {
            uint32_t q[8];
            levels_of(x[j], s, 7.f, q);
            word = 0u;
#pragma unroll
            for (int e = 7; e >= 0; --e) word = word * 16u + q[e];
            word -= (kLevelBase - 8u) * 0x11111111u;   // what each level was added to, less 8
        }
        const unsigned unit = first + j * (kThreads / 16);
        if (unit >= (unsigned)units) continue;
        packed[unit * 16LL + 4 * (l % 4) + l / 4] = word;
        if ((l & ((1 << shift) - 1)) == 0 && c[j] < k) scales[(long long)row[j] * groups + (c[j] >> (shift + 3))] = __ushort_as_bfloat16(sb);
    }
}

template <int VEC>
__global__ void __launch_bounds__(kThreads)
dequantize_q4_kernel(const uint32_t* __restrict__ packed, const __nv_bfloat16* __restrict__ scales, int units, int k,
                     Divisor blocks, int shift, int groups, float* __restrict__ w, long long ldw) {
    const long long i = (long long)blockIdx.x * kThreads + threadIdx.x;
    if (i >= 16LL * units) return;
    const int unit = (int)(i / 16), row = blocks(unit), b = unit - row * blocks.d, l = (int)(i % 16), c = b * kBlock + 8 * l;
    if (c >= k) return;
    const uint32_t word = __ldg(packed + unit * 16LL + 4 * (l % 4) + l / 4);
    const float s = __bfloat162float(scales[(long long)row * groups + ((b * 16 + l) >> shift)]);
    float x[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = (float)((int)(word >> (4 * e) & 15u) - 8) * s;
    float* out = w + (long long)row * ldw + c;
    if (VEC && c + 8 <= k) {
        store8<VEC>(out, x);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (c + e < k) out[e] = x[e];
    }
}

// ------------------------------------------------------------------- products --
// y[r] = act(x[r] W^T + bias) + residual[r] for up to 8 rows of x a CTA, on integer MMAs
// (m16n8k32): 16 rows of W are the A operand, as the nibbles level + 8 lie in a word (a mask, a
// shift and a mask for eight of them), the columns of B are rows of x. The elements of 128
// columns of x become integers of 31 bits in four signed 8-bit digits: the largest of them is 2^29 to 2^30
// units, so that a rounding is at most 2^-30 of it. A group's sum of each digit is exact; it starts at
// -8 times the digits' own sum, which takes the 8 out of the levels, and at the bits of an fp32 number
// (quant.cuh), so that it ends as fp32 and needs no conversion. Then come the group's scale and the sum over groups, in fp32. One or
// two rows of x put their digits into B's eight columns, one MMA for 32 weights of each
// row; up to 8 rows take four. (On bf16 terms of x the levels had to be converted, 11 instructions for eight
// weights instead of 3: 50257 x 1600 took 24.7 us for 2 rows and 28.8 for 8.)
//
// Bound by the reading of W where that is large, by the chain of a strip's steps where it is
// small. A CTA takes an equal share of the strips of 16 rows of W and turns x into digits once, in shared
// memory, in the order that the lanes read them. The share's steps (a strip's blocks of 128
// columns) form a line that its 16 warps cut into equal stretches; a warp has the weights of
// kAhead steps on their way in registers, over the ends of strips. A strip that one warp has all of
// goes out at once, the others' sums, in order, through shared memory, where the digits were. 50257 x 1600, 42 MB, takes 17 us for 2 rows and 20 for 8; the loads alone, in this order, take 10.
struct MatvecArgs {
    const float* x;
    long long ldx;
    int rows;
    const uint8_t* packed;
    const __nv_bfloat16* scales;
    int n, k, blocks, groups, strips;
    const float* bias;
    const float* residual;
    long long ldr;
    int gelu;
    float* y;
    long long ldy;
};

constexpr int kWarps = 16, kAhead = 3;

// d = c + a b on levels (unsigned) and digits (signed), m16n8k32
__device__ __forceinline__ void mma_u8s8(int (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, const int (&c)[4]) {
    asm("mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %11, %12, %13};"
        : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "r"(c[0]), "r"(c[1]), "r"(c[2]), "r"(c[3]));
}
// where a digit's sum starts: 1.5 2^23, 2^31, 2^39, 2^47, whose last places are worth 1, 256, ...
__host__ __device__ constexpr int start_of(int digit) { return 0x4b400000 + (digit << 26); }

// A block of x in shared memory: digits [j][digit pair][lane] (few: [j][lane]), where sums start
// [group][digit][column], what 1 is worth [column].
template <bool FEW, int G>
struct XBlock {
    static constexpr int kDigits = FEW ? 1 : 4, kGroups = kBlock / G;
    static constexpr int kDigitBytes = 4 * kDigits * 32 * 8, kStartBytes = kGroups * kDigits * 8 * 4;
    static constexpr int kBytes = kDigitBytes + kStartBytes + 8 * 4;
};
constexpr int kSumBytes = 16 * 8 * 4;              // a warp's sums of a strip

// acc + y s unit, rounded once, for a group's sum y (an integer below 2^40, of one digit below 2^17), its scale s and
// a unit, which is a power of two. y times the unit is exact (it is a multiple of 2^-127) and fits in fp32 below
// kFarUnit, whatever s is; s times the unit need not: with s first, small products lost bits and
// 0 times infinity was NaN. From kFarUnit on, s (a bf16 number) times the unit is exact or infinite, and infinite only
// where the product with any y but 0 is.
constexpr float kFarUnit = 0x1p80f;
template <bool FAR>
__device__ __forceinline__ float add_group(float y, float s, float unit, float acc) {
    if (FAR && unit >= kFarUnit) return fmaf(y, y == 0.f ? s : s * unit, acc);
    return fmaf(y * unit, s, acc);
}

// y of row r0 + r, output j, from the sum of its products
__device__ __forceinline__ void put(const MatvecArgs& a, int r, int j, float sum) {
    if (j >= a.n) return;
    if (a.bias) sum = __fadd_rn(sum, __ldg(a.bias + j));
    if (a.gelu) sum = gelu_new_ref(sum);
    if (a.residual) sum = __fadd_rn(a.residual[(long long)r * a.ldr + j], sum);
    a.y[(long long)r * a.ldy + j] = sum;
}

template <bool FEW, int G, bool VEC>
__global__ void __launch_bounds__(kWarps * 32, 1) matvec_q4_kernel(const __grid_constant__ MatvecArgs a) {
    using X = XBlock<FEW, G>;
    constexpr int kDigits = X::kDigits, kGroups = X::kGroups, kRows = FEW ? 2 : 8;
    extern __shared__ __align__(16) uint8_t smem[];
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5, g = lane >> 2, c = lane & 3;
    const int r0 = blockIdx.y * kRows, rows = min(kRows, a.rows - r0);
    const int strip0 = (int)((long long)a.strips * blockIdx.x / gridDim.x);
    const int strip1 = (int)((long long)a.strips * (blockIdx.x + 1) / gridDim.x);
    const int steps = (strip1 - strip0) * a.blocks;          // (fits: 2^27 strips of at most 128 blocks over the SMs)
    auto from_step = [&](int w) { return (int)((unsigned long long)(unsigned)steps * (unsigned)w / kWarps); };
    const int q0 = from_step(warp), q1 = from_step(warp + 1);
    pdl_wait();

    // weights and scales (of group c of the block; the others have theirs from lane c) on their way
    uint4 w[kAhead][2];
    unsigned short sc[kAhead][2];
    const uint8_t* w_at[2];
    const unsigned short* s_at[2];
    int left = q1 - q0, next_strip = strip0 + q0 / a.blocks, next_kb = q0 % a.blocks;
    auto rows_of = [&]() {                         // of next_strip
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const long long row = min(next_strip * 16 + 8 * h + g, a.n - 1);
            w_at[h] = a.packed + (row * a.blocks + next_kb) * kBlockBytes + 16 * c;
            s_at[h] = reinterpret_cast<const unsigned short*>(a.scales) + row * a.groups;
        }
    };
    rows_of();
    auto load = [&](uint4 (&to)[2], unsigned short (&s)[2]) {
        if (left <= 0) return;
        --left;
        const int grp = min(next_kb * kGroups + (c & (kGroups - 1)), a.groups - 1);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            asm volatile("ld.global.nc.L1::no_allocate.v4.b32 {%0, %1, %2, %3}, [%4];"
                         : "=r"(to[h].x), "=r"(to[h].y), "=r"(to[h].z), "=r"(to[h].w)
                         : "l"(w_at[h]));
            s[h] = __ldg(s_at[h] + grp);
            w_at[h] += kBlockBytes;
        }
        if (++next_kb == a.blocks) {
            next_kb = 0;
            ++next_strip;
            rows_of();
        }
    };
#pragma unroll
    for (int d = 0; d < kAhead; ++d) load(w[d], sc[d]);

    // the row of x that this lane's column g of B stands for, and (FEW) which of its digits
    const int xr = FEW ? g >> 2 : g;
    const bool real = xr < rows;
    const float* x = a.x + (long long)(r0 + min(xr, rows - 1)) * a.ldx;
    bool far = false;                              // a unit of x is above kFarUnit
    // block kb of x, by one warp
    auto x_of = [&](int kb) {
        uint8_t* const to = smem + (size_t)kb * X::kBytes;
        float top = 0.f, v[4][8];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            weights8<VEC ? 4 : 0>(x, kb * kBlock + 32 * j + 8 * c, real ? a.k : 0, v[j]);
#pragma unroll
            for (int i = 0; i < 8; ++i) top = max_abs(top, v[j][i]);
        }
        top = max_abs(top, __shfl_xor_sync(kAll, top, 1));
        top = max_abs(top, __shfl_xor_sync(kAll, top, 2));
        // the largest is below 2^(e - 126): times 2^(156 - e), it is at most 2^30
        const int e = max((int)(__float_as_uint(top) >> 23), 29);
        const float up = __uint_as_float((uint32_t)(283 - e) << 23);
        // (2^-127 is the smallest unit; a row with an element that is not finite gets NaN)
        float one = e >= 255 ? top * 0.f : __uint_as_float(e == 29 ? 0x00400000u : (uint32_t)(e - 29) << 23);
        if constexpr (FEW) one *= (float)(1 << (8 * (g & 3)));
        far |= one >= kFarUnit;
        int sum[kDigits][kGroups] = {};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            uint32_t b[kDigits][2];
#pragma unroll
            for (int o = 0; o < 2; ++o) {
                uint32_t w[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) w[i] = ((uint32_t)__float2int_rn(v[j][2 * i + o] * up) + 0x00808080u) ^ 0x00808080u;
                uint32_t d[4];                     // digit by digit
                const uint32_t lo0 = __byte_perm(w[0], w[1], 0x5140), lo1 = __byte_perm(w[2], w[3], 0x5140);
                const uint32_t hi0 = __byte_perm(w[0], w[1], 0x7362), hi1 = __byte_perm(w[2], w[3], 0x7362);
                d[0] = __byte_perm(lo0, lo1, 0x5410);
                d[1] = __byte_perm(lo0, lo1, 0x7632);
                d[2] = __byte_perm(hi0, hi1, 0x5410);
                d[3] = __byte_perm(hi0, hi1, 0x7632);
#pragma unroll
                for (int z = 0; z < kDigits; ++z) {
                    b[z][o] = FEW ? ((g & 2) ? (g & 1 ? d[3] : d[2]) : (g & 1 ? d[1] : d[0])) : d[z];
                    sum[z][j / (G / 32)] = __dp4a((int)b[z][o], 0x01010101, sum[z][j / (G / 32)]);
                }
            }
            if constexpr (FEW) {
                reinterpret_cast<uint2*>(to)[j * 32 + lane] = make_uint2(b[0][0], b[0][1]);
            } else {
                reinterpret_cast<uint4*>(to)[(2 * j) * 32 + lane] = make_uint4(b[0][0], b[0][1], b[1 % kDigits][0], b[1 % kDigits][1]);
                reinterpret_cast<uint4*>(to)[(2 * j + 1) * 32 + lane] =
                    make_uint4(b[2 % kDigits][0], b[2 % kDigits][1], b[3 % kDigits][0], b[3 % kDigits][1]);
            }
        }
        int* const starts = reinterpret_cast<int*>(to + X::kDigitBytes);
#pragma unroll
        for (int z = 0; z < kDigits; ++z)
#pragma unroll
            for (int i = 0; i < kGroups; ++i) {
                int y = sum[z][i];
                y += __shfl_xor_sync(kAll, y, 1);
                y += __shfl_xor_sync(kAll, y, 2);
                if (c == 0) starts[(i * kDigits + z) * 8 + g] = start_of(z) - 8 * y;
            }
        if (c == 0) reinterpret_cast<float*>(to + X::kDigitBytes + X::kStartBytes)[g] = one;
    };
    for (int kb = warp; kb < a.blocks; kb += kWarps) x_of(kb);
    far = __syncthreads_or(far);                   // (a row's sums are the same either way, if its own units are below)

    float acc[4] = {}, ended[4];                   // ended: of the strip that the warp goes on with
    bool went_on = false;
    int strip = strip0 + q0 / a.blocks, kb = q0 % a.blocks, first = kb;
    auto add = [&](auto far_units, uint4 (&wd)[2], unsigned short (&sd)[2]) {
        constexpr bool kFar = decltype(far_units)::value;
        const uint32_t w0[4] = {wd[0].x, wd[0].y, wd[0].z, wd[0].w}, w1[4] = {wd[1].x, wd[1].y, wd[1].z, wd[1].w};
        const float s[2] = {__uint_as_float((uint32_t)sd[0] << 16), __uint_as_float((uint32_t)sd[1] << 16)};
        load(wd, sd);
        const uint8_t* const xb = smem + (size_t)kb * X::kBytes;
        const int* const starts = reinterpret_cast<const int*>(xb + X::kDigitBytes) + 2 * c;
        const float2 unit = *reinterpret_cast<const float2*>(xb + X::kDigitBytes + X::kStartBytes + 8 * c);
#pragma unroll
        for (int i = 0; i < kGroups; ++i) {
            int d[kDigits][4];
#pragma unroll
            for (int z = 0; z < kDigits; ++z) {
                const int2 from = *reinterpret_cast<const int2*>(starts + (i * kDigits + z) * 8);
                d[z][0] = d[z][2] = from.x;
                d[z][1] = d[z][3] = from.y;
            }
#pragma unroll
            for (int j = i * (G / 32); j < (i + 1) * (G / 32); ++j) {
                const uint32_t frag[4] = {w0[j] & 0x0f0f0f0fu, w1[j] & 0x0f0f0f0fu, (w0[j] >> 4) & 0x0f0f0f0fu,
                                          (w1[j] >> 4) & 0x0f0f0f0fu};
                if constexpr (FEW) {
                    const uint2 u = reinterpret_cast<const uint2*>(xb)[j * 32 + lane];
                    mma_u8s8(d[0], frag, u.x, u.y, d[0]);
                } else {
                    const uint4 u = reinterpret_cast<const uint4*>(xb)[(2 * j) * 32 + lane];
                    const uint4 v = reinterpret_cast<const uint4*>(xb)[(2 * j + 1) * 32 + lane];
                    mma_u8s8(d[0], frag, u.x, u.y, d[0]);
                    mma_u8s8(d[1 % kDigits], frag, u.z, u.w, d[1 % kDigits]);
                    mma_u8s8(d[2 % kDigits], frag, v.x, v.y, d[2 % kDigits]);
                    mma_u8s8(d[3 % kDigits], frag, v.z, v.w, d[3 % kDigits]);
                }
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const float f = kGroups == 1 ? s[h] : __shfl_sync(kAll, s[h], (lane & ~3) | i);
#pragma unroll
                for (int e = 2 * h; e < 2 * h + 2; ++e) {
                    float y;
                    if constexpr (FEW) {
                        y = __int_as_float(d[0][e]) - __int_as_float(start_of(0));
                    } else {
                        const float high = (__int_as_float(d[3 % kDigits][e]) - __int_as_float(start_of(3))) +
                                           (__int_as_float(d[2 % kDigits][e]) - __int_as_float(start_of(2)));
                        const float low = __int_as_float(d[1 % kDigits][e]) - (__int_as_float(start_of(1)) + __int_as_float(start_of(0)));
                        y = high + (low + __int_as_float(d[0][e]));
                    }
                    acc[e] = add_group<kFar>(y, f, e & 1 ? unit.y : unit.x, acc[e]);
                }
            }
        }
        if (++kb < a.blocks) return;
        // the strip's end
        if (first == 0) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int j = strip * 16 + 8 * h + g;
                if constexpr (FEW) {               // columns 4 r .. 4 r + 3 are row r's digits
                    float y = acc[2 * h] + acc[2 * h + 1];
                    y += __shfl_xor_sync(kAll, y, 1);
                    if ((c & 1) == 0 && (c >> 1) < rows) put(a, r0 + (c >> 1), j, y);
                } else {
#pragma unroll
                    for (int e = 0; e < 2; ++e)
                        if (2 * c + e < rows) put(a, r0 + 2 * c + e, j, acc[2 * h + e]);
                }
            }
        } else {
            went_on = true;
#pragma unroll
            for (int e = 0; e < 4; ++e) ended[e] = acc[e];
        }
        acc[0] = acc[1] = acc[2] = acc[3] = 0.f;
        kb = first = 0;
        ++strip;
    };
    // (two loops: with the choice inside, five rows of 6400 x 1600 in groups of 32 took 8.4 us instead of 7.9)
    auto run = [&](auto far_units) {
        for (int q = q0; q < q1; q += kAhead) {
#pragma unroll
            for (int d = 0; d < kAhead; ++d)
                if (q + d < q1) add(far_units, w[d], sc[d]);
        }
    };
    if (far) run(std::true_type{});
    else run(std::false_type{});
    // (a strip that is not at its end here: begun by this warp, or, within the stretch, gone on with)
    const bool open = q0 < q1 && kb > 0, begun = open && first == 0;
    // Sums of a warp's cut strips, where x was: of the one that it goes on with, of the one that it begins.
    float* const sums = reinterpret_cast<float*>(smem);
    auto keep = [&](int slot, const float (&y)[4]) {
        float* const to = sums + (size_t)(2 * warp + slot) * (kSumBytes / 4);
#pragma unroll
        for (int h = 0; h < 2; ++h) *reinterpret_cast<float2*>(to + (8 * h + g) * 8 + 2 * c) = make_float2(y[2 * h], y[2 * h + 1]);
    };
    __syncthreads();
    if (went_on) keep(0, ended);
    if (open) keep(begun, acc);
    __syncthreads();
    if (!begun) return;
    // the warp that began a cut strip adds the sums of those that went on with it, in order
    int last = warp + 1;
    while (from_step(last + 1) < (strip - strip0 + 1) * a.blocks) ++last;
    const int o = lane & 15;
    float sum[kRows / 2] = {};
    for (int v = warp; v <= last; ++v) {
        if (v > warp && from_step(v) == from_step(v + 1)) continue;          // a warp without steps
        const float* z = sums + (size_t)(2 * v + (v == warp)) * (kSumBytes / 4) + o * 8;
#pragma unroll
        for (int i = 0; i < kRows / 2; ++i) {
            const int r = 2 * i + (lane >> 4);
            if constexpr (FEW) {
                const float4 d = *reinterpret_cast<const float4*>(z + 4 * r);
                sum[i] += (d.x + d.y) + (d.z + d.w);
            } else {
                sum[i] += z[r];
            }
        }
    }
#pragma unroll
    for (int i = 0; i < kRows / 2; ++i) {
        const int r = 2 * i + (lane >> 4);
        if (r < rows) put(a, r0 + r, strip * 16 + o, sum[i]);
    }
}

template <bool FEW, bool VEC>
void (*matvec_of(int group))(MatvecArgs) {
    return group == 32 ? matvec_q4_kernel<FEW, 32, VEC> : group == 64 ? matvec_q4_kernel<FEW, 64, VEC> : matvec_q4_kernel<FEW, 128, VEC>;
}
template <bool FEW>
size_t x_block_bytes(int group) {
    return group == 32 ? XBlock<FEW, 32>::kBytes : group == 64 ? XBlock<FEW, 64>::kBytes : XBlock<FEW, 128>::kBytes;
}

// Shapes that the 4-bit entry points share.
bool q4_shape_ok(int n, int k, int group) {
    return n > 0 && k > 0 && (group == 32 || group == 64 || group == 128);
}
// the lanes that share a group: 2 to this
int shift_of(int group) { return group == 32 ? 2 : group == 64 ? 3 : 4; }
constexpr int kMostInputs = 16384;                 // of a product: two rows of x fit in shared memory
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
    const long long units = (long long)n * blocks_of(k), per = kThreads / 16 * kUnits, grid = (units + per - 1) / per;
    if (k > kMostColumns || units > INT_MAX) return MODEL_ERR_CAPACITY;
    OnDeviceOf dev(packed);
    if (dev.status() != MODEL_OK) return dev.status();
    const bool vec8 = aligned(w, 32) && ldw % 8 == 0, vec4 = aligned16(w) && ldw % 4 == 0;
    (vec8 ? quantize_q4_kernel<8> : vec4 ? quantize_q4_kernel<4> : quantize_q4_kernel<0>)<<<(unsigned)grid, kThreads, 0, static_cast<cudaStream_t>(stream)>>>(
        w, ldw, (int)units, k, divisor(blocks_of(k)), shift_of(group), static_cast<uint32_t*>(packed), static_cast<__nv_bfloat16*>(scales),
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
    if (k > kMostColumns || units > INT_MAX) return MODEL_ERR_CAPACITY;
    OnDeviceOf dev(w);
    if (dev.status() != MODEL_OK) return dev.status();
    const bool vec8 = aligned(w, 32) && ldw % 8 == 0, vec4 = aligned16(w) && ldw % 4 == 0;
    (vec8 ? dequantize_q4_kernel<8> : vec4 ? dequantize_q4_kernel<4> : dequantize_q4_kernel<0>)<<<(unsigned)grid, kThreads, 0, static_cast<cudaStream_t>(stream)>>>(
        static_cast<const uint32_t*>(packed), static_cast<const __nv_bfloat16*>(scales), (int)units, k, divisor(blocks_of(k)), shift_of(group),
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
    if (k > kMostInputs || rows > 2 * 65535) return MODEL_ERR_CAPACITY;
    if (rows == 0) return MODEL_OK;
    OnDeviceOf dev(y);
    if (dev.status() != MODEL_OK) return dev.status();
    const int strips = (n - 1) / 16 + 1, sms = sm_count(dev.device()), blocks = blocks_of(k);
    const size_t sums = (size_t)kWarps * 2 * kSumBytes, most = 227 * 1024;
    // two rows at a time also where 8 rows of x do not fit
    const bool few = rows <= 2 || blocks * x_block_bytes<false>(group) > most;
    const size_t x_bytes = few ? x_block_bytes<true>(group) : x_block_bytes<false>(group);
    const int passes = (rows - 1) / (few ? 2 : 8) + 1;
    MatvecArgs a{x, ldx, rows, static_cast<const uint8_t*>(packed), static_cast<const __nv_bfloat16*>(scales), n, k,
                 blocks, (k + group - 1) / group, strips, bias, residual, ldr, gelu, y, ldy};
    const bool vec = aligned16(x) && ldx % 4 == 0;
    auto* kernel = few ? (vec ? matvec_of<true, true>(group) : matvec_of<true, false>(group))
                       : (vec ? matvec_of<false, true>(group) : matvec_of<false, false>(group));
    // (always the most that any call wants: calls on other threads set it too)
    TIE_OP_CU(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)most));
    const size_t smem = blocks * x_bytes > sums ? blocks * x_bytes : sums;
    TIE_OP_CU(launch_pdl(kernel, dim3((unsigned)(strips < sms ? strips : sms), (unsigned)passes), dim3(32 * kWarps), smem,
                         static_cast<cudaStream_t>(stream), a));
    ++op_launches;
    return MODEL_OK;
}
