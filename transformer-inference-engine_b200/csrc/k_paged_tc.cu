// k_paged_tc.cu -- attention of many new rows over a paged cache on the tensor
// cores (head_dim 64), for the sequences that ops_attn.cu's streaming kernel
// leaves to it.
//
// One CTA per SM takes an equal stretch of the batch's jobs (paged_attn.cuh): a
// job is one step over the keys of 128 rows,
//
//   S  = Q . K^T    M = 128 rows, N = 128 keys, K = 64 dims
//   O += P . V      M = 128 rows, N = 64 dims,  K = 128 keys
//
// with an online softmax. Two streams of jobs run side by side in a CTA, each
// with its own O, maximum and sum: the two halves of a tile of more than 128
// rows, over the same steps (keys and values are converted once for both), or
// else the even and the odd steps of its one half, joined at the end. Three
// buffers of S go round, so the next S is there when a stream has written its
// P, and nothing stops between tiles: every role runs ahead as far as its
// buffers let it.
//
// Arithmetic. Results are fp32's. A 16-bit MMA runs at twice the rate of a
// tf32 one and fp16 has tf32's 11 significant bits, so every operand is split
// into two fp16 terms, x = hi + lo, and a product is hi.hi + hi.lo + lo.hi in
// three MMAs with fp32 accumulation (what is left out is below 2^-22 of it).
// bf16 pages need no lo term: 8 significant bits fit one fp16. What fp16 lacks
// is range, so operands are scaled by powers of two that are undone exactly:
//   - a query row by its largest element, a key row by its own: to [2^14, 2^15).
//     Down to 2^-17 of the largest element of its row an element keeps all 22
//     bits, below that an absolute error of 2^-40 of the largest. S is
//     multiplied by both rows' scales when the softmax reads it.
//   - a value row by 2^-e, its largest element again: the probability of key
//     j takes up 2^e_j, that is, the softmax runs on t_j = s_j + e_j and O sums
//     2^(t_j - m) (v_j 2^-e_j) = 2^(s_j - m) v_j. The row sum is
//     sum 2^(t_j - m) 2^-e_j. With m at most 8 below the largest t so far, the
//     probabilities lie in [0, 2^15] around 2^7 and their small ones keep an
//     absolute error of 2^-32 of the largest. What falls below 2^-126 is nothing
//     to O, but in the row sum it may be the largest weight there is (a row of
//     zeros beside values of 2^70). A sum that could miss such weights is small
//     (kLeastSum), and the epilogue forms it anew from the scores alone.
// A scale belongs to one row where rows may be masked (steps that cross the
// diagonal), so a masked row's range costs no visible one bits; elsewhere the 16
// rows of a page, which every query row sees, share theirs.
//
// Sums. The MMA adds to its fp32 accumulator by cutting off: each one loses
// about 1.5e-8 of the sum, always towards zero, 3e-5 over 16,384 keys (the row
// sum, added in registers, is rounded and does not). So an O takes kFlush steps
// (at most 64 MMAs, 1e-6) and is then added, rounded, to a running O that the L2
// cache holds for the tile (red, so that nobody waits for it), and lo products
// come before hi . hi. Error of 2048 rows over 14,336 cached positions, bf16:
// 3.1e-5 -> 1.5e-6; the additions cost 5 % of the time.
//
// Masks. Keys behind the unit's last visible one and keys of unmapped pages
// are loaded as zero with e = -inf: no comparison is needed except in the
// steps that cross the diagonal, where a masked t is set to -inf. A value that
// is not finite would reach every row of the tile (0 * inf): the loaders put 0
// in its place and raise a flag, and the epilogue adds it to the rows that see
// it.
//
// Warps (640 threads, five warpgroups that share the registers by need):
//   0-7   softmax: stream warp / 4, TMEM lanes 32 (warp % 4) .. + 31, a row per
//         thread. S is read twice, for the maximum and for the probabilities,
//         32 columns at a time; P takes the columns of S as they are read.
//         The running maximum m moves only when it has grown by more than 8
//         (powers of two), so O is rescaled rarely.
//   8-15  loaders: warp w takes keys 16 w .. 16 w + 15 of a step, one page, 32
//         bytes per lane and row; scales, splits and stores them in the
//         128-byte-swizzled layout of the MMA's operands (K: K-major; V as it
//         lies, MN-major). The next step's rows are in registers by then. A
//         tile's Q goes the same way, 16 rows a warp.
//   16    allocates TMEM and issues the MMAs: whatever is ready, S up to three jobs
//         ahead of P . V, each kind in the order of the jobs.
//   17    walks the CTA's stretch and leaves each tile's description in a ring.
//   18    leaves the join its record; 19 only completes the warpgroup.
// The roles' loops together outgrow the instruction cache, so loops that would be
// unrolled elsewhere are not and waits are kept short: 16 % -> 7 % of the fetches
// missed, 1,050 -> 955 us for the chunk above, 357 -> 335 us for 48 mixed sequences.
// In all, with the join: the chunk (32 query heads on 8) 881 us, of which 311 are its
// MMAs at the measured rate; 48 sequences of up to 117 new rows and 900 cached, 25
// heads, fp32: 245 us, bound by the loaders' chain of a step (convert keys, convert
// values, wait for their buffers) and by a tile's start, not by memory (51 us).
// TMEM (512 columns): three S / P (384), two O (128).
// Every wait is bounded (2 s; longer only for the place of a tile of more than 16,384
// steps in the ring): on expiry it raises the abort flag, which ends every other wait;
// the roles run out without storing, the MMAs issued are drained and TMEM is freed.
#include <cuda.h>

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <atomic>
#include <type_traits>

#include "paged_attn.cuh"

namespace tie {
namespace {

#include "tc_ptx.cuh"

constexpr int kThreads = 640;
// Registers a thread: at launch, and after the warpgroups have shared them out (softmax
// 2 x 128 threads, loaders 2 x 128, MMA 128); the sum must not pass what the block was
// launched with, and a share that is taken with .inc (or .dec) not be below (above) it.
// fp32 rows take the loaders twice the registers of bf16 ones. Both splits with both types
// (us, 112 / 104 / 48 and 112 / 112 / 32): 48 sequences of 60 new rows behind 450, 25 heads,
// fp32 274 and 232, bf16 184 and 200; 8 of 256 behind 512, 12 heads, fp32 88 and 84, bf16 68
// and 72; the chunk, bf16 864 and 995, but fp32 1,264 and 1,452: there the shape would want
// the other split. (120 / 96 / 48 and 104 / 112 / 48 were slower for one or the other.)
constexpr int kRegsLaunch = 96;
template <bool BF16>
constexpr int kRegsSoftmax = 112;
template <bool BF16>
constexpr int kRegsLoad = BF16 ? 104 : 112;
template <bool BF16>
constexpr int kRegsMma = BF16 ? 48 : 32;
template <bool BF16>
constexpr bool kRegsFit = 256 * kRegsSoftmax<BF16> + 256 * kRegsLoad<BF16> + 128 * kRegsMma<BF16> <= kThreads * kRegsLaunch &&
                          kRegsSoftmax<BF16> >= kRegsLaunch && kRegsLoad<BF16> >= kRegsLaunch && kRegsMma<BF16> <= kRegsLaunch;
static_assert(kRegsFit<true> && kRegsFit<false>, "register split");
constexpr int kSoftmaxWarps = 8, kLoadWarps = 8, kMmaWarp = 16, kUnitWarp = 17;
constexpr uint32_t kWaitLimitNs = 2000000000u;  // 2 s
constexpr unsigned kAll = 0xffffffffu;
constexpr float kBase = 7.f;        // the largest probability is 2^7 when m is the maximum
constexpr float kSlack = 8.f;       // m may lag the maximum by this (probabilities up to 2^15)

// shared memory (bytes from the 1024-aligned base)
constexpr uint32_t kTermBytes = kTileKeys * 128;          // 128 rows of 64 fp16
constexpr int kKeyRing = 8, kUnitRing = 8, kQsRing = kUnitRing;
constexpr uint32_t kOffK = 0;                             // two buffers of hi, lo
constexpr uint32_t kOffV = kOffK + 4 * kTermBytes;
constexpr uint32_t kOffQ = kOffV + 4 * kTermBytes;        // two halves of hi, lo
constexpr uint32_t kOffKeys = kOffQ + 4 * kTermBytes;     // [8][3][128] per key (or page): scale, e, 2^-e
constexpr uint32_t kOffQs = kOffKeys + kKeyRing * 3 * kTileKeys * 4;   // [8][256] per row
constexpr uint32_t kOffXch = kOffQs + kQsRing * kTileRows * 4;         // [2][4][128] the streams' maxima and sums
constexpr uint32_t kOffRun = kOffXch + 8 * kHalfRows * 4;              // [256] maxima that running O's are relative to
constexpr uint32_t kOffUnits = kOffRun + kTileRows * 4;
constexpr uint32_t kOffBars = kOffUnits + kUnitRing * 80;
constexpr uint32_t kSmemBytes = kOffBars + 512;
static_assert(kSmemBytes + 1024 <= 227 * 1024, "shared memory");
// the line of jobs lies in the buffers that nothing uses yet
static_assert((kOpsMaxSeqs + 1) * 8 <= (int)kOffKeys, "line of jobs");
// steps of a stream that one O takes before it is added to the running O: 64 or 48 MMAs
// (twice the steps: 3 % faster, twice the error)
template <bool BF16>
constexpr int kFlush = BF16 ? 4 : 2;
constexpr float kFarUp = 40.f;     // the running O is rescaled when the maximum has grown by this
// A key whose 2^(s + e - m) flushed weighs less than 2^(81 - 126) in the row sum (e >= -81).
// A sum of this for each of its keys has lost less than 2^-24 of itself.
constexpr float kLeastSum = 0x1p-21f;

// TMEM columns: S / P of buffer b at 128 b, O of stream st at kColO + 64 st
constexpr uint32_t kTmemCols = 512, kColO = 384;

// kind::f16 with f16 operands, fp32 accumulation, M = 128
constexpr uint32_t kIdescS = (1u << 4) | ((uint32_t)(kTileKeys >> 3) << 17) | ((uint32_t)(kHalfRows >> 4) << 24);
constexpr uint32_t kIdescO = (1u << 4) | (1u << 16) /* B is MN-major */ | ((uint32_t)(kHeadDim >> 3) << 17) |
                             ((uint32_t)(kHalfRows >> 4) << 24);

__device__ __forceinline__ bool mbar_test(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(bar), "r"(parity)
        : "memory");
    return ok != 0;
}

__device__ __forceinline__ void mbar_arrive_n(uint32_t bar, uint32_t n) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(n) : "memory");
}

__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}

// two floats in one register pair, and the packed fp32 operations on them
// (each lane rounds as the scalar operation does)
typedef unsigned long long f32x2;
__device__ __forceinline__ f32x2 pair(float a, float b) {
    f32x2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float2 unpair(f32x2 v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
    f32x2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) {
    f32x2 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) {
    f32x2 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

// (a, b) as two fp16 terms each: hi and lo, packed. x - hi is exact in fp32.
__device__ __forceinline__ void split2(float a, float b, uint32_t& hi, uint32_t& lo) {
    hi = pack2(a, b);
    float ra, rb;
    asm("{\n\t.reg .b16 h0, h1, one;\n\t"
        "mov.b32 {h0, h1}, %2;\n\t"
        "mov.b16 one, 0xBC00;\n\t"              // -1
        "fma.rn.f32.f16 %0, h0, one, %3;\n\t"
        "fma.rn.f32.f16 %1, h1, one, %4;\n\t}"
        : "=f"(ra), "=f"(rb)
        : "r"(hi), "f"(a), "f"(b));
    lo = pack2(ra, rb);
}

// 32 columns of the warp's 32 lanes, on their way until tmem_arrived(r)
__device__ __forceinline__ void tmem_ld32_start(uint32_t taddr, uint32_t (&r)[32]) {
    __syncwarp();
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
          "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
          "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr));
}
template <int N>
__device__ __forceinline__ void tmem_arrived(uint32_t (&r)[N]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
    // no use of a register is moved ahead of the wait
#pragma unroll
    for (int i = 0; i < N; ++i) asm volatile("" : "+r"(r[i]));
}
// the same columns written; tmem_stored() waits for all of the warp's stores
__device__ __forceinline__ void tmem_st32_start(uint32_t taddr, const uint32_t (&r)[32]) {
    __syncwarp();
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
        "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
        "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};"
        ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
          "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]),
          "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]),
          "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
        : "memory");
}
// *to += v, rounded to nearest, without waiting for it; a thread's own additions to one
// place are made in their order
__device__ __forceinline__ void add_global4(float4* to, float4 v) {
    asm volatile("red.relaxed.gpu.global.add.v4.f32 [%0], {%1, %2, %3, %4};"
                 ::"l"(to), "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w) : "memory");
}
__device__ __forceinline__ void tmem_stored() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// What a job rarely does to its O, out of the way of the softmax loop, whose registers
// it would take. All: this thread's row of the 64 columns at col_o; the row's running O
// is dims 4 k .. 4 k + 3 at running(run_o) + k * kHalfRows, and nobody else touches it.
__device__ __forceinline__ float4* running(float* run_o) {
    return reinterpret_cast<float4*>(run_o) + ((size_t)2 * blockIdx.x + (threadIdx.x >> 7)) * (kHeadDim / 4) * kHalfRows +
           (threadIdx.x & 127);
}
__device__ __noinline__ void scale_o(uint32_t col_o, float f) {
#pragma unroll 1
    for (int h = 0; h < 2; ++h) {
        uint32_t x[32];
        tmem_ld32_start(col_o + 32u * h, x);
        tmem_arrived(x);
#pragma unroll
        for (int d = 0; d < 32; ++d) x[d] = __float_as_uint(__uint_as_float(x[d]) * f);
        tmem_st32_start(col_o + 32u * h, x);
    }
}
// O, relative to the maximum m_o, added to the running O, which is relative to *m_run;
// first: there is none yet.
__device__ __noinline__ void add_to_running(uint32_t col_o, float* run_o, float* m_run, float m_o, bool first) {
    float4* const run = running(run_o);
    float mr = first ? -INFINITY : *m_run;
    if (mr == -INFINITY) {                    // (nothing, or nothing but zeros)
        mr = m_o;
    } else if (m_o > mr + kFarUp) {
        const float f = ex2_ftz(mr - m_o);
#pragma unroll 1
        for (int k = 0; k < kHeadDim / 4; ++k) {
            const float4 v = __ldcg(run + k * kHalfRows);
            __stcg(run + k * kHalfRows, make_float4(v.x * f, v.y * f, v.z * f, v.w * f));
        }
        mr = m_o;
    }
    *m_run = mr;
    const float f = m_o == -INFINITY ? 0.f : ex2_ftz(m_o - mr);
#pragma unroll 1
    for (int h = 0; h < 2; ++h) {
        uint32_t x[32];
        tmem_ld32_start(col_o + 32u * h, x);
        tmem_arrived(x);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const float4 v = make_float4(__uint_as_float(x[4 * k]) * f, __uint_as_float(x[4 * k + 1]) * f,
                                         __uint_as_float(x[4 * k + 2]) * f, __uint_as_float(x[4 * k + 3]) * f);
            if (first) __stcg(run + (8 * h + k) * kHalfRows, v);
            else add_global4(run + (8 * h + k) * kHalfRows, v);
        }
    }
}
// at a tile's end: the running O, scaled by f, goes back into O
__device__ __noinline__ void add_running(uint32_t col_o, float* run_o, float f) {
    const float4* const run = running(run_o);
#pragma unroll 1
    for (int h = 0; h < 2; ++h) {
        uint32_t x[32];
        float4 v[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = __ldcg(run + (8 * h + k) * kHalfRows);
        tmem_ld32_start(col_o + 32u * h, x);
        tmem_arrived(x);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            x[4 * k] = __float_as_uint(fmaf(v[k].x, f, __uint_as_float(x[4 * k])));
            x[4 * k + 1] = __float_as_uint(fmaf(v[k].y, f, __uint_as_float(x[4 * k + 1])));
            x[4 * k + 2] = __float_as_uint(fmaf(v[k].z, f, __uint_as_float(x[4 * k + 2])));
            x[4 * k + 3] = __float_as_uint(fmaf(v[k].w, f, __uint_as_float(x[4 * k + 3])));
        }
        tmem_st32_start(col_o + 32u * h, x);
    }
    tmem_stored();
}

// the larger magnitude; NaN if either is
__device__ __forceinline__ float max_abs(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(fabsf(a)), "f"(fabsf(b)));
    return r;
}

// the biased exponent of a row's largest magnitude, within [lo, 254]; what is
// not finite counts as 2^14 (scale 1)
__device__ __forceinline__ int row_exponent(float mx, int lo) {
    const int e = (int)(__float_as_uint(mx) >> 23);
    return e == 255 ? 141 : max(e, lo);
}
__device__ __forceinline__ float pow2_biased(int e) { return __uint_as_float((uint32_t)e << 23); }

// 8 elements of one row, by one load that stays where it is written
template <bool BF16>
struct Row8;
template <>
struct Row8<false> {
    float x[8];
    __device__ __forceinline__ void load(const void* base, size_t at) {
        asm volatile("ld.global.nc.L1::no_allocate.v8.f32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                     : "=f"(x[0]), "=f"(x[1]), "=f"(x[2]), "=f"(x[3]), "=f"(x[4]), "=f"(x[5]), "=f"(x[6]), "=f"(x[7])
                     : "l"(static_cast<const float*>(base) + at));
    }
    // the same from a row that is only 16-byte aligned
    __device__ __forceinline__ void load_any(const float* from) {
        const float4 u = __ldg(reinterpret_cast<const float4*>(from)), v = __ldg(reinterpret_cast<const float4*>(from) + 1);
        x[0] = u.x; x[1] = u.y; x[2] = u.z; x[3] = u.w;
        x[4] = v.x; x[5] = v.y; x[6] = v.z; x[7] = v.w;
    }
    __device__ __forceinline__ void negate() {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = -x[i];
    }
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = 0.f;
    }
    __device__ __forceinline__ void get(float (&y)[8]) const {
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = x[i];
    }
    // zero for every element that is not finite; whether there was one
    __device__ __forceinline__ bool clear_odd() {
        bool odd = false;
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (!(fabsf(x[i]) < INFINITY)) { x[i] = 0.f; odd = true; }
        return odd;
    }
};
template <>
struct Row8<true> {
    uint32_t x[4];
    __device__ __forceinline__ void load(const void* base, size_t at) {
        asm volatile("ld.global.nc.L1::no_allocate.v4.b32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3])
                     : "l"(static_cast<const __nv_bfloat16*>(base) + at));
    }
    __device__ __forceinline__ void zero() { x[0] = x[1] = x[2] = x[3] = 0u; }
    __device__ __forceinline__ void get(float (&y)[8]) const {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            y[2 * i] = __uint_as_float(x[i] << 16);
            y[2 * i + 1] = __uint_as_float(x[i] & 0xffff0000u);
        }
    }
    __device__ __forceinline__ bool clear_odd() {
        bool odd = false;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if ((x[i] & 0x7f80u) == 0x7f80u) { x[i] &= 0xffff0000u; odd = true; }
            if ((x[i] & 0x7f800000u) == 0x7f800000u) { x[i] &= 0xffffu; odd = true; }
        }
        return odd;
    }
};

// the largest of 8 lanes (a row's) or of the warp (a page's)
__device__ __forceinline__ float lanes_max(float m, int lanes) {
#pragma unroll
    for (int o = 1; o < lanes; o <<= 1) m = max_abs(m, __shfl_xor_sync(kAll, m, o));
    return m;
}

// Scales 8 elements, splits them, and stores the terms at the row's 16-byte
// chunk `off` of a 128-byte-swizzled operand.
template <bool BF16>
__device__ __forceinline__ void store_terms(uint8_t* hi, uint32_t off, const float (&y)[8], float scale) {
    uint32_t h[4], l[4];
    const f32x2 sc = pair(scale, scale);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 v = unpair(mul2(pair(y[2 * i], y[2 * i + 1]), sc));
        if constexpr (BF16) h[i] = pack2(v.x, v.y);
        else split2(v.x, v.y, h[i], l[i]);
    }
    *reinterpret_cast<uint4*>(hi + off) = make_uint4(h[0], h[1], h[2], h[3]);
    if constexpr (!BF16) *reinterpret_cast<uint4*>(hi + kTermBytes + off) = make_uint4(l[0], l[1], l[2], l[3]);
}

__device__ __forceinline__ float max_abs8(const float (&y)[8]) {
    return max_abs(max_abs(max_abs(y[0], y[1]), max_abs(y[2], y[3])), max_abs(max_abs(y[4], y[5]), max_abs(y[6], y[7])));
}

// A tile of the CTA's stretch, as warp 17 describes it to the others.
struct Unit {
    int steps;            // over keys [key0, key1); negative: no more tiles
    int both;             // the streams are the tile's two halves; else its even and odd steps
    int g, token0;        // K/V head; the sequence's first row of q and out
    int row0, n_rows;     // rows of the sequence
    int key0, key1;
    int first_last;       // the least last visible position of the rows
    int ctx, part;        // where the result goes: partial 2 * CTA + part, or -1: out
    int fill0, job0;      // steps and jobs of the tiles before it
    int half0;            // Q halves used before it
    int s;
    int odd;              // a value is not finite (set by the loaders)
    int used0, used1;     // tiles before it that have jobs of each stream
    int pad[2];
};
static_assert(sizeof(Unit) == 80, "ring entry");

// Adds the values of keys [key0, key1) that are not finite to 32 elements at `to`
// (whatever their probabilities: what sees them is not finite). Rare: out of line.
template <bool BF16>
__device__ __noinline__ void add_odd(const void* values, const int32_t* table, size_t w, int n_pages, float* to, int dim,
                                     int key0, int key1) {
    for (int key = key0; key < key1; ++key) {
        const int e = __ldg(table + key / kPageRows);
        if (e < 0 || e >= n_pages) continue;
        const size_t at = ((size_t)e * kPageRows + key % kPageRows) * w + dim;
#pragma unroll 1
        for (int d = 0; d < 32; ++d) {
            float v;
            if constexpr (BF16) v = __bfloat162float(static_cast<const __nv_bfloat16*>(values)[at + d]);
            else v = static_cast<const float*>(values)[at + d];
            if (!(fabsf(v) < INFINITY)) to[d] += v;
        }
    }
}

// four elements of a row of the pool
template <bool BF16>
__device__ __forceinline__ float4 four_of(const void* pool, size_t at) {
    if constexpr (BF16) {
        const uint2 u = __ldg(reinterpret_cast<const uint2*>(static_cast<const __nv_bfloat16*>(pool) + at));
        return make_float4(__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xffff0000u), __uint_as_float(u.y << 16),
                           __uint_as_float(u.y & 0xffff0000u));
    } else {
        return __ldg(reinterpret_cast<const float4*>(static_cast<const float*>(pool) + at));
    }
}

// The row sum, relative to the maximum m, of row i of the unit's sequence over those of the unit's
// keys that it sees, from the scores alone. Rare, hence simple: four keys at a time, which a warp's
// rows share (0.6 us a key and tile: the waits of the other roles bound a tile to 3 million keys).
template <bool BF16>
__device__ __noinline__ float row_sum(const PagedAttnArgs& a, const volatile Unit& n, int i, float m) {
    const size_t w = (size_t)a.n_kv_head * kHeadDim;
    const float* q = a.q + (size_t)(n.token0 + i / a.group) * a.ldq + (n.g * a.group + i % a.group) * kHeadDim;
    const int32_t* table = a.table + (size_t)n.s * a.width;
    const int key1 = min(n.key1, n.ctx + i / a.group + 1);
    float sum = 0.f;
    constexpr int kKeys = 4;
#pragma unroll 1
    for (int key = n.key0; key < key1; key += kKeys) {     // (key0 is a multiple of a page)
        const int page = __ldg(table + key / kPageRows);
        if (page < 0 || page >= a.n_pages) continue;
        const size_t from = ((size_t)page * kPageRows + key % kPageRows) * w + (size_t)n.g * kHeadDim;
        float s[kKeys] = {};
#pragma unroll 2
        for (int d = 0; d < kHeadDim; d += 4) {
            const float4 x = __ldg(reinterpret_cast<const float4*>(q + d));
#pragma unroll
            for (int r = 0; r < kKeys; ++r) {
                const float4 y = four_of<BF16>(a.k, from + r * w + d);
                s[r] = fmaf(x.w, y.w, fmaf(x.z, y.z, fmaf(x.y, y.y, fmaf(x.x, y.x, s[r]))));
            }
        }
        float part = 0.f;
#pragma unroll
        for (int r = 0; r < kKeys; ++r)
            if (key + r < key1) part += ex2_ftz(fmaf(s[r], a.scale2, kBase - m));
        sum += part;
    }
    return sum;
}

template <bool BF16>
__global__ void __launch_bounds__(kThreads, 1) paged_tc_kernel(const __grid_constant__ PagedAttnArgs a) {
    pdl_trigger();                     // few_rows_kernel takes the SMs that are done
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    float* s_keys = reinterpret_cast<float*>(smem + kOffKeys);
    float* s_qs = reinterpret_cast<float*>(smem + kOffQs);
    float* s_run = reinterpret_cast<float*>(smem + kOffRun);
    float* s_xch = reinterpret_cast<float*>(smem + kOffXch);
    volatile Unit* units = reinterpret_cast<volatile Unit*>(smem + kOffUnits);
    // Barriers; a phase of each is one use of what it guards, in order.
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + kOffBars);
    uint64_t* k_full = bars + 0;     // [step % 2] keys written (loader warps)
    uint64_t* v_full = bars + 2;     // [step % 2] values and per-key numbers written (loader warps)
    uint64_t* k_free = bars + 4;     // [step % 2] keys read by all their MMAs (two commits)
    uint64_t* v_free = bars + 6;     // [step % 2] values likewise
    uint64_t* q_full = bars + 8;     // [half % 2] Q half written (loader warps)
    uint64_t* q_free = bars + 10;    // [half % 2] read by all its MMAs (commit)
    uint64_t* s_full = bars + 12;    // [job % 3] S computed (commit)
    uint64_t* p_full = bars + 15;    // [job % 3] P written, O rescaled (the stream's softmax warps)
    uint64_t* o_done = bars + 18;    // [job % 3] P . V done (commit)
    uint64_t* o_last = bars + 21;    // [stream] the tile's last P . V of the stream done (commit)
    uint64_t* o_free = bars + 23;    // [stream] O read by the epilogue (softmax warps), a phase for each tile
                                     // that has jobs of the stream: arrivals for one without could come
                                     // before those of the tile before it
    uint64_t* pair_in = bars + 25;   // [lane quarter] both streams' maxima and sums written
    uint64_t* unit_full = bars + 29; // [tile % 8] description written
    uint64_t* unit_free = bars + 37; // [tile % 8] read for good (softmax, loader and MMA warps)
    uint64_t* drained = bars + 45;   // every MMA done (commit)
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 46);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    const int t = threadIdx.x, warp = t >> 5, lane = t & 31;

    if (t == 0) {
        for (int b = 0; b < 2; ++b) {
            mbar_init(smem_u32(&k_full[b]), kLoadWarps);
            mbar_init(smem_u32(&v_full[b]), kLoadWarps);
            mbar_init(smem_u32(&k_free[b]), 2);
            mbar_init(smem_u32(&v_free[b]), 2);
            mbar_init(smem_u32(&q_full[b]), kLoadWarps);
            mbar_init(smem_u32(&q_free[b]), 1);
            mbar_init(smem_u32(&o_last[b]), 1);
            mbar_init(smem_u32(&o_free[b]), kSoftmaxWarps);
        }
        for (int b = 0; b < 3; ++b) {
            mbar_init(smem_u32(&s_full[b]), 1);
            mbar_init(smem_u32(&p_full[b]), kSoftmaxWarps / 2);
            mbar_init(smem_u32(&o_done[b]), 1);
        }
        for (int b = 0; b < 4; ++b) mbar_init(smem_u32(&pair_in[b]), 2);
        for (int b = 0; b < kUnitRing; ++b) {
            mbar_init(smem_u32(&unit_full[b]), 1);
            mbar_init(smem_u32(&unit_free[b]), kSoftmaxWarps + kLoadWarps + 1);
        }
        mbar_init(smem_u32(drained), 1);
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == kMmaWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                     ::"r"(smem_u32(tmem_slot)), "r"(kTmemCols));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    __shared__ ScheduleScratch<kThreads> scratch;
    JobLine line;
    build_line<kThreads>(a, reinterpret_cast<long long*>(smem), &scratch, t, &line);
    const long long all = line.base[a.n_seq], g0 = blockIdx.x * line.share, g1 = min(g0 + line.share, all);
    LineUnit here;                   // the stretch's first tile (warp 17's own)
    if (warp == kUnitWarp && g0 < g1) here = unit_at(a, line, g0);
    if (warp == kUnitWarp + 1 && lane == 0) {
        // the tile that this CTA begins and does not finish, for the join: it lies in the
        // CTA's second part and the first parts of the CTAs after it (while the line is
        // still there: the loaders write over it)
        JoinRecord rec{};
        if (g0 < g1 && g1 < all) {
            const LineUnit u = unit_at(a, line, g1 - 1);
            if (u.jobs >= g0 && u.jobs < g1 && u.end > g1) {
                rec.parts = (int)((u.end - 1) / line.share) - (int)blockIdx.x + 1;
                rec.n_rows = tile_n_rows(u.q, u.tile);
                rec.token0 = u.q.row0;
                rec.i0 = u.tile * kTileRows;
                rec.g = u.g;
            }
        }
        a.record[1][blockIdx.x] = rec;
    }
    asm volatile("tcgen05.fence::before_thread_sync;");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;");
    const uint32_t tmem = *tmem_slot;

    // (there are many of these: each is kept short)
    auto wait = [&](const uint64_t* bar, uint32_t parity) -> bool {
        const uint32_t b = smem_u32(bar), t0 = nanoseconds();
        for (uint32_t i = 1; !mbar_try_wait(b, parity); ++i)
            if ((i & 255u) == 0 && (*abort_flag || nanoseconds() - t0 > kWaitLimitNs)) {
                *abort_flag = 1;
                return false;
            }
        return true;
    };
    auto wait_all = [&](const uint64_t* bar, uint32_t parity) -> bool { return __all_sync(kAll, wait(bar, parity)); };
    // tile number n of the stretch is described
    auto unit_there = [&](uint32_t n) -> bool { return wait_all(&unit_full[n % kUnitRing], n / kUnitRing & 1u); };
    auto unit_read = [&](uint32_t n) {
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&unit_free[n % kUnitRing]));
    };
    const size_t w = (size_t)a.n_kv_head * kHeadDim;

    if (warp < kSoftmaxWarps) {
        // ------------------------------------------------------------ softmax
        // tcgen05.ld / .st are warp-collective: every condition around them is
        // the warp's.
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsSoftmax<BF16>));
        const int st = warp >> 2, qq = warp & 3, r = qq * 32 + lane;
        const uint32_t lanes = tmem + ((uint32_t)(qq * 32) << 16);
        uint32_t lasts = 0, pairs = 0;      // o_last and pair_in phases so far
        for (uint32_t un = 0;; ++un) {
            if (!unit_there(un)) break;
            const volatile Unit& n = units[un % kUnitRing];
            const int steps = n.steps, both = n.both;
            if (steps < 0) break;
            const int row = (both ? st * kHalfRows : 0) + r, n_rows = n.n_rows;   // of the tile
            const int i = n.row0 + min(row, n_rows - 1), last = n.ctx + i / a.group;
            const int key0 = n.key0, first_last = n.first_last;
            const uint32_t fill0 = (uint32_t)n.fill0, job0 = (uint32_t)n.job0;
            float m = -INFINITY, l = 0.f, qs = 0.f;
            bool ok = true;
            const int j0 = both ? 0 : st, dj = both ? 1 : 2;
            // none of the warp's 32 rows exists: what P holds there reaches only rows of
            // O that nobody reads
            const bool idle = (both ? st * kHalfRows : 0) + qq * 32 >= n_rows;
#pragma unroll 1
            for (int j = j0; j < steps; j += dj) {
                const uint32_t f = fill0 + (uint32_t)j, job = job0 + (both ? 2u * j + st : (uint32_t)j), buf = job % 3u;
                const uint32_t col_s = lanes + buf * kTileKeys;
                if (idle) {
                    if (!(ok = wait_all(&s_full[buf], job / 3u & 1u))) break;
                    if (lane == 0) mbar_arrive(smem_u32(&p_full[buf]));
                    continue;
                }
                ok = ok && wait_all(&v_full[f & 1u], f >> 1 & 1u);
                ok = ok && wait_all(&s_full[buf], job / 3u & 1u);
                if (!ok) break;
                asm volatile("tcgen05.fence::after_thread_sync;");
                if (j == j0) qs = s_qs[(un % kQsRing) * kTileRows + row];   // written before the tile's first v_full
                const float* keys = s_keys + (f % kKeyRing) * 3 * kTileKeys;
                const int pos = key0 + j * kTileKeys;
                const bool diagonal = pos + kTileKeys - 1 > first_last;
                uint32_t x[32];
                // t of four columns 4 k .. 4 k + 3 of a step on the diagonal: a scale per key
                auto t_of4 = [&](const uint32_t* s4, int k, float (&tt)[4]) {
                    const float4 ks = reinterpret_cast<const float4*>(keys)[k];
                    const float4 ee = reinterpret_cast<const float4*>(keys + kTileKeys)[k];
                    const float fk[4] = {ks.x, ks.y, ks.z, ks.w}, e[4] = {ee.x, ee.y, ee.z, ee.w};
#pragma unroll
                    for (int d = 0; d < 4; ++d) {
                        // (the scales first: S times one of them may be beyond fp32)
                        tt[d] = fmaf(__uint_as_float(s4[d]), qs * fk[d], e[d]);
                        if (pos + 4 * k + d > last) tt[d] = -INFINITY;
                    }
                };
                float mt = -INFINITY;
                // one body per pass for the four chunks of 32 columns: unrolled, the
                // roles' code together outgrows the instruction cache
                tmem_ld32_start(col_s, x);
#pragma unroll 1
                for (int c = 0; c < 4; ++c) {
                    tmem_arrived(x);
                    if (diagonal) {
#pragma unroll
                        for (int k = 0; k < 8; ++k) {
                            float tt[4];
                            t_of4(x + 4 * k, 8 * c + k, tt);
                            mt = fmaxf(fmaxf(fmaxf(mt, tt[0]), tt[1]), fmaxf(tt[2], tt[3]));
                        }
                    } else {
                        // a scale per page: the largest t is the largest S's
#pragma unroll
                        for (int g = 0; g < 2; ++g) {
                            float s0 = __uint_as_float(x[16 * g]), s1 = __uint_as_float(x[16 * g + 1]);
#pragma unroll
                            for (int d = 2; d < 16; d += 2) {
                                s0 = fmaxf(s0, __uint_as_float(x[16 * g + d]));
                                s1 = fmaxf(s1, __uint_as_float(x[16 * g + d + 1]));
                            }
                            mt = fmaxf(mt, fmaf(fmaxf(s0, s1), qs * keys[2 * c + g], keys[kTileKeys + 2 * c + g]));
                        }
                    }
                    tmem_ld32_start(col_s + 32u * ((c + 1) & 3), x);   // the last one begins the second pass
                }
                float alpha = 1.f, sum = 0.f;
                const float m_o = m;           // what O is relative to
                if (mt > m + kSlack || m == -INFINITY) {      // also the first finite maximum
                    alpha = ex2_ftz(m - mt);                  // m = -inf: 0 (or, mt = -inf too, unused)
                    if (alpha == 0.f) sum = weigh(l, m - mt); // the row sum may outweigh it
                    if (mt == -INFINITY) alpha = 1.f;
                    m = mt;
                }
                const float lift = m == -INFINITY ? 0.f : kBase - m;
#pragma unroll 1
                for (int c = 0; c < 4; ++c) {
                    tmem_arrived(x);
                    uint32_t p[32];                           // hi terms of columns 2 k, 2 k + 1 in p[k], lo in p[16 + k]
                    if (diagonal) {
#pragma unroll
                        for (int k = 0; k < 8; ++k) {
                            float tt[4];
                            t_of4(x + 4 * k, 8 * c + k, tt);
                            const float4 iv = reinterpret_cast<const float4*>(keys + 2 * kTileKeys)[8 * c + k];
#pragma unroll
                            for (int d = 0; d < 4; ++d) tt[d] = ex2_ftz(tt[d] + lift);
                            sum = fmaf(tt[3], iv.w, fmaf(tt[2], iv.z, fmaf(tt[1], iv.y, fmaf(tt[0], iv.x, sum))));
                            split2(tt[0], tt[1], p[2 * k], p[16 + 2 * k]);
                            split2(tt[2], tt[3], p[2 * k + 1], p[16 + 2 * k + 1]);
                        }
                    } else {
#pragma unroll
                        for (int g = 0; g < 2; ++g) {
                            const float fk = qs * keys[2 * c + g], e = keys[kTileKeys + 2 * c + g] + lift;
                            const f32x2 ff = pair(fk, fk), ee = pair(e, e);
                            f32x2 part = pair(0.f, 0.f);
#pragma unroll
                            for (int d = 0; d < 8; ++d) {
                                const int k = 8 * g + d;
                                const float2 y = unpair(fma2(pair(__uint_as_float(x[2 * k]), __uint_as_float(x[2 * k + 1])), ff, ee));
                                const float p0 = ex2_ftz(y.x), p1 = ex2_ftz(y.y);
                                part = add2(part, pair(p0, p1));
                                split2(p0, p1, p[k], p[16 + k]);
                            }
                            const float2 ps = unpair(part);
                            sum = fmaf(ps.x + ps.y, keys[2 * kTileKeys + 2 * c + g], sum);
                        }
                    }
                    if (c < 3) tmem_ld32_start(col_s + 32u * (c + 1), x);
                    tmem_st32_start(col_s + 32u * c, p);      // over the columns of S it was made from
                }
                l = fmaf(l, alpha, sum);
                const int nth = both ? j : j >> 1;                        // of the stream's jobs in this tile
                const bool flush = nth && nth % kFlush<BF16> == 0;
                if (__any_sync(kAll, flush || (alpha != 1.f && nth))) {
                    // O of the stream's job before, once its P . V is done
                    const uint32_t before = job - 2u;
                    ok = ok && wait_all(&o_done[before % 3u], before / 3u & 1u);
                    if (!ok) break;
                    asm volatile("tcgen05.fence::after_thread_sync;");
                    const uint32_t col_o = lanes + kColO + 64u * st;
                    if (flush) {
                        add_to_running(col_o, a.run_o, &s_run[threadIdx.x], m_o, nth == kFlush<BF16>);
                    } else {
                        scale_o(col_o, alpha);
                    }
                }
                tmem_stored();
                asm volatile("tcgen05.fence::before_thread_sync;");
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&p_full[buf]));
            }
            if (j0 < steps) {
                ok = ok && wait_all(&o_last[st], lasts & 1u);
                ++lasts;
            }
            if (!ok) break;
            if ((both ? steps : (steps - st + 1) >> 1) > kFlush<BF16> && !idle) {
                asm volatile("tcgen05.fence::after_thread_sync;");
                add_running(lanes + kColO + 64u * st, a.run_o, m == -INFINITY ? 0.f : ex2_ftz(s_run[threadIdx.x] - m));
            }
            // this thread's results: row `row`, dims [dim0, dim0 + 32), from o
            auto put = [&](uint32_t (&o)[32], int dim0, float mm, float ll) {
                float4* to;
                float f = 1.f;
                if (n.part < 0) {
                    f = ll == 0.f ? 0.f : 1.f / ll;
                    to = reinterpret_cast<float4*>(a.out + (size_t)(n.token0 + i / a.group) * a.ldo +
                                                   (n.g * a.group + i % a.group) * kHeadDim + dim0);
                } else {
                    const size_t at = (2 * (size_t)blockIdx.x + n.part) * kTileRows + row;
                    to = reinterpret_cast<float4*>(a.part_o[1] + at * kHeadDim + dim0);
                    if (dim0 == 0) {
                        a.part_ml[1][2 * at] = mm == -INFINITY ? mm : mm - kBase;
                        a.part_ml[1][2 * at + 1] = ll;
                    }
                }
#pragma unroll
                for (int c = 0; c < 8; ++c)
                    to[c] = f == 0.f ? make_float4(0.f, 0.f, 0.f, 0.f)
                                     : make_float4(__uint_as_float(o[4 * c]) * f, __uint_as_float(o[4 * c + 1]) * f,
                                                   __uint_as_float(o[4 * c + 2]) * f, __uint_as_float(o[4 * c + 3]) * f);
                if (n.odd && f != 0.f)
                    add_odd<BF16>(a.v, a.table + (size_t)n.s * a.width, w, a.n_pages, reinterpret_cast<float*>(to),
                                  n.g * kHeadDim + dim0, key0, min(n.key1, last + 1));
            };
            uint32_t o[32];
            if (both) {
                if (l < (float)steps * (kTileKeys * kLeastSum) && m != -INFINITY && row < n_rows) l = row_sum<BF16>(a, n, i, m);
                asm volatile("tcgen05.fence::after_thread_sync;");
#pragma unroll 1
                for (int h = 0; h < 2; ++h) {
                    tmem_ld32_start(lanes + kColO + 64u * st + 32u * h, o);
                    tmem_arrived(o);
                    if (steps == 0) {
                        // the stretch has the second half of a step that belongs to the CTA
                        // before: a part with nothing in it
#pragma unroll
                        for (int d = 0; d < 32; ++d) o[d] = 0u;
                    }
                    if (row < n_rows) put(o, 32 * h, m, l);
                }
                asm volatile("tcgen05.fence::before_thread_sync;");
                __syncwarp();
                if (lane == 0 && steps) mbar_arrive_n(smem_u32(&o_free[st]), 2);
            } else {
                // the streams' results joined: each stream's warps do 32 dims
                float* xch = s_xch + (pairs & 1u) * 4 * kHalfRows;
                xch[(2 * st) * kHalfRows + r] = m;
                xch[(2 * st + 1) * kHalfRows + r] = l;
                asm volatile("tcgen05.fence::before_thread_sync;");
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&pair_in[qq]));
                if (!wait_all(&pair_in[qq], pairs & 1u)) break;
                ++pairs;
                asm volatile("tcgen05.fence::after_thread_sync;");
                const float m0 = xch[r], l0 = xch[kHalfRows + r], m1 = xch[2 * kHalfRows + r], l1 = xch[3 * kHalfRows + r];
                const float mm = fmaxf(m0, m1), base = mm == -INFINITY ? 0.f : mm;
                const float f0 = ex2_ftz(m0 - base), f1 = ex2_ftz(m1 - base);
                float ll = fmaf(l1, f1, l0 * f0);
                const float far = fminf(m0, m1) - base;
                if ((ll < (float)steps * (kTileKeys * kLeastSum) || (far < -126.f && far > -INFINITY)) && mm != -INFINITY && row < n_rows)
                    ll = row_sum<BF16>(a, n, i, mm);
                uint32_t v1[32];
                tmem_ld32_start(lanes + kColO + 32u * st, o);
                tmem_arrived(o);
                tmem_ld32_start(lanes + kColO + 64u + 32u * st, v1);
                tmem_arrived(v1);
                asm volatile("tcgen05.fence::before_thread_sync;");
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(smem_u32(&o_free[0]));
                    if (steps > 1) mbar_arrive(smem_u32(&o_free[1]));
                }
#pragma unroll
                for (int d = 0; d < 32; ++d) {
                    float v = f0 > 0.f ? __uint_as_float(o[d]) * f0 : 0.f;
                    // a stream without steps has left nothing in its O
                    if (f1 > 0.f) v = fmaf(__uint_as_float(v1[d]), f1, v);
                    o[d] = __float_as_uint(v);
                }
                if (row < n_rows) put(o, 32 * st, mm, ll);
            }
            unit_read(un);
        }
    } else if (warp < kSoftmaxWarps + kLoadWarps) {
        // ------------------------------------------------------------ loaders
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsLoad<BF16>));
        const int lw = warp - kSoftmaxWarps, sub = lane >> 3, dl = lane & 7;
        Row8<BF16> kr[4], vr[4];
        // the rows of step j of a tile that this warp has: its page (or -1), and their
        // loads. All 16 rows of a page are read (page 0's for none) and what is not
        // there is cleared afterwards: a branch at each load costs more than the rest.
        auto page_of = [&](const volatile Unit& n, int j) {
            const int p = (n.key0 + j * kTileKeys) / kPageRows + lw;
            if (j >= n.steps || (long long)p * kPageRows >= n.key1) return -1;
            const int e = __ldg(a.table + (size_t)n.s * a.width + p);
            return e >= 0 && e < a.n_pages ? e : -1;
        };
        const size_t lane_at = (size_t)sub * w + 8 * dl;
        auto load = [&](Row8<BF16>(&rows)[4], const void* from, int g, int page) {
            const size_t at = (size_t)max(page, 0) * (kPageRows * w) + g * kHeadDim + lane_at;
#pragma unroll
            for (int i = 0; i < 4; ++i) rows[i].load(from, at + (size_t)(4 * i) * w);
        };
        // there: positions of the page that are (all of them: 16 or more)
        auto clear = [&](Row8<BF16>(&rows)[4], int there) {
            if (there >= kPageRows) return;
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (4 * i + sub >= there) rows[i].zero();
        };
        // stores this warp's 16 rows as terms; mx: what each row (in all its lanes) is scaled by
        auto store = [&](uint8_t* to, const auto (&rows)[4], const float (&mx)[4], int lo, auto is_bf16) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int row = lw * 16 + 4 * i + sub;
                float y[8];
                rows[i].get(y);
                store_terms<decltype(is_bf16)::value>(to, (uint32_t)(row * 128 + ((dl ^ (row & 7)) << 4)), y,
                                                      pow2_biased(268 - row_exponent(mx[i], lo)));
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        };
        auto row_max = [&](const auto (&rows)[4], float (&mx)[4]) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float y[8];
                rows[i].get(y);
                mx[i] = max_abs8(y);
            }
        };
        auto arrive = [&](uint64_t* bar) {
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(bar));
        };
        bool ok = unit_there(0);
        int page = -1, page_next = -1;
        if (ok && units[0].steps > 0) {
            page = page_of(units[0], 0);
            load(kr, a.k, units[0].g, page);
            load(vr, a.v, units[0].g, page);
        }
        for (uint32_t un = 0; ok; ++un) {
            volatile Unit& n = units[un % kUnitRing];
            const int steps = n.steps;
            if (steps < 0) break;
            if (steps > 0) {
                // Q: rows of 64 floats, a scale per row
                const uint32_t half0 = (uint32_t)n.half0;
                page_next = page_of(n, 1);
#pragma unroll 1
                for (int h = 0; h <= n.both && ok; ++h) {
                    const uint32_t half = half0 + (uint32_t)h;
                    Row8<false> qr[4];
                    float mx[4];
                    const int n_rows = n.n_rows, row0 = n.row0, token0 = n.token0, g = n.g;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int row = h * kHalfRows + lw * 16 + 4 * i + sub, at = row0 + row;
                        if (row < n_rows)
                            qr[i].load_any(a.q + (size_t)(token0 + at / a.group) * a.ldq +
                                           (g * a.group + at % a.group) * kHeadDim + 8 * dl);
                        else
                            qr[i].zero();
                    }
                    row_max(qr, mx);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        mx[i] = lanes_max(mx[i], 8);
                        if (a.scale2 < 0.f) qr[i].negate();   // the scale's sign goes to Q: s_qs >= 0
                        if (dl == 0)
                            s_qs[(un % kQsRing) * kTileRows + h * kHalfRows + lw * 16 + 4 * i + sub] =
                                pow2_biased(row_exponent(mx[i], 15) - 14) * fabsf(a.scale2);
                    }
                    if (half >= 2) ok = wait_all(&q_free[half & 1u], ((half >> 1) - 1) & 1u);
                    if (!ok) break;
                    store(smem + kOffQ + (half & 1u) * 2 * kTermBytes, qr, mx, 15, std::false_type{});
                    arrive(&q_full[half & 1u]);
                }
            }
#pragma unroll 1
            for (int j = 0; j < steps && ok; ++j) {
                const uint32_t f = (uint32_t)n.fill0 + (uint32_t)j, b = f & 1u, before = ((f >> 1) - 1) & 1u;
                const int there = page < 0 ? 0 : n.key1 - (n.key0 + j * kTileKeys + lw * kPageRows);
                const bool diagonal = n.key0 + j * kTileKeys + kTileKeys - 1 > n.first_last;
                float* keys = s_keys + (f % kKeyRing) * 3 * kTileKeys;
                // largest magnitudes: of each row, or of the page in every entry
                auto spread = [&](float (&mx)[4]) {
                    if (diagonal) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) mx[i] = lanes_max(mx[i], 8);
                    } else {
                        mx[0] = mx[1] = mx[2] = mx[3] = lanes_max(max_abs(max_abs(mx[0], mx[1]), max_abs(mx[2], mx[3])), 32);
                    }
                };
                float mx[4];
                clear(kr, there);
                row_max(kr, mx);
                spread(mx);
                // key buffer b is free once the S of the step before last are computed
                if (f >= 2 && !(ok = wait_all(&k_free[b], before))) break;
                store(smem + kOffK + b * 2 * kTermBytes, kr, mx, 15, std::integral_constant<bool, BF16>{});
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (diagonal ? dl == 0 : i == 0 && lane == 0)
                        keys[diagonal ? lw * kPageRows + 4 * i + sub : lw] = pow2_biased(row_exponent(mx[i], 15) - 14);
                arrive(&k_full[b]);
                // the next step's rows, of this tile or the next one
                const bool over = j + 1 == steps;
                const volatile Unit* nn = &n;
                if (over) {
                    if (!(ok = unit_there(un + 1))) break;
                    nn = &units[(un + 1) % kUnitRing];
                    page_next = nn->steps > 0 ? page_of(*nn, 0) : -1;
                }
                const int gn = nn->steps > 0 ? nn->g : -1;
                if (gn >= 0) load(kr, a.k, gn, page_next);
                clear(vr, there);
                row_max(vr, mx);
                spread(mx);
                if (__any_sync(kAll, !(mx[0] < INFINITY && mx[1] < INFINITY && mx[2] < INFINITY && mx[3] < INFINITY))) {
                    // rare: elements that are not finite are left to the epilogue
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (vr[i].clear_odd()) n.odd = 1;
                    row_max(vr, mx);
                    spread(mx);
                }
                // value buffer b is free once the P . V of the step before last are done
                if (f >= 2 && !(ok = wait_all(&v_free[b], before))) break;
                store(smem + kOffV + b * 2 * kTermBytes, vr, mx, 60, std::integral_constant<bool, BF16>{});
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (diagonal ? dl == 0 : i == 0 && lane == 0) {
                        const int at = diagonal ? lw * kPageRows + 4 * i + sub : lw, e = row_exponent(mx[i], 60);
                        keys[kTileKeys + at] = (diagonal ? 4 * i + sub : 0) < there ? (float)(e - 141) : -INFINITY;
                        keys[2 * kTileKeys + at] = pow2_biased(268 - e);
                    }
                arrive(&v_full[b]);
                if (gn >= 0) load(vr, a.v, gn, page_next);
                page = page_next;
                page_next = over ? -1 : page_of(n, j + 2);
            }
            if (!ok) break;
            unit_read(un);
            if (steps == 0) {
                // nothing was prefetched for the tile after an empty one
                if (!(ok = unit_there(un + 1))) break;
                const volatile Unit& x = units[(un + 1) % kUnitRing];
                if (x.steps > 0) {
                    page = page_of(x, 0);
                    load(kr, a.k, x.g, page);
                    load(vr, a.v, x.g, page);
                }
            }
        }
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsMma<BF16>));
        if (warp == kMmaWarp) {
            // ------------------------------------------------------------ MMA
            const uint32_t sb = smem_u32(smem), tm = __shfl_sync(kAll, tmem, 0);
            // a place in the line of jobs: job k of tile un
            struct Cursor {
                uint32_t un, job;
                int k, jobs, both, steps;
            };
            // (values of the ring are the same in all lanes, and known to the compiler to be)
            auto uniform = [&](int v) { return __shfl_sync(kAll, v, 0); };
            // to the next tile with jobs from c.un on; false: there is none
            auto settle = [&](Cursor& c) -> bool {
                for (;; ++c.un) {
                    if (!unit_there(c.un)) return false;
                    const volatile Unit& n = units[c.un % kUnitRing];
                    c.steps = uniform(n.steps);
                    if (c.steps < 0) return false;
                    c.both = uniform(n.both);
                    c.k = 0;
                    c.jobs = c.steps << c.both;
                    if (c.jobs) return true;
                }
            };
            // Whether all of the phases have completed, without waiting: the warp issues
            // whatever is ready, the S of a later job or the P . V of an earlier one. (In
            // a fixed order a P . V whose P has long been there waits behind an S whose
            // keys are still on their way, and the loaders behind both.)
            auto there = [&](const uint64_t* bar, uint32_t phase) { return mbar_test(smem_u32(bar), phase & 1u); };
            Cursor sc{}, pc{};
            bool s_more = settle(sc), p_more = s_more && settle(pc);
            // S of the next job, into the buffer that the job three before has left
            auto issue_s = [&]() -> bool {
                const volatile Unit& n = units[sc.un % kUnitRing];
                const int j = sc.k >> sc.both, st = sc.k & 1;
                const uint32_t f = (uint32_t)uniform(n.fill0) + (uint32_t)j, b = f & 1u, buf = sc.job % 3u;
                const uint32_t half = (uint32_t)uniform(n.half0) + (sc.both ? (uint32_t)st : 0u);
                const bool first = sc.both ? j == 0 : sc.k == 0, last = sc.both ? j == sc.steps - 1 : sc.k == sc.jobs - 1;
                if (!__all_sync(kAll, there(&k_full[b], f >> 1) && (!first || there(&q_full[half & 1u], half >> 1)) &&
                                          (sc.job < 3 || there(&o_done[buf], sc.job / 3u - 1))))
                    return false;
                asm volatile("tcgen05.fence::after_thread_sync;");
                const uint32_t kb = sb + kOffK + b * 2 * kTermBytes, qb = sb + kOffQ + (half & 1u) * 2 * kTermBytes;
                const uint32_t d = tm + buf * kTileKeys;
                // the small terms first: q_lo . k_hi (2), q_hi . k_lo (1), q_hi . k_hi (0)
#pragma unroll 1
                for (int term = 2; term >= 0; term -= BF16 ? 2 : 1) {
                    const uint32_t qt = qb + (term == 2 ? kTermBytes : 0u), kt = kb + (term == 1 ? kTermBytes : 0u);
#pragma unroll (BF16 ? 4 : 1)
                    for (int ks = 0; ks < kHeadDim / 16; ++ks)
                        mma_f16(d, sw128_desc(qt + 32u * ks), sw128_desc(kt + 32u * ks), kIdescS, ks || term < 2 ? 1u : 0u);
                }
                commit_elected(smem_u32(&s_full[buf]));
                commit_elected(smem_u32(&k_free[b]));
                if (!sc.both) commit_elected(smem_u32(&k_free[b]));   // no other job reads the buffer
                if (last) commit_elected(smem_u32(&q_free[half & 1u]));
                ++sc.job;
                if (++sc.k == sc.jobs) {
                    ++sc.un;
                    s_more = settle(sc);
                }
                return true;
            };
            uint32_t freed = 0;         // tiles whose description is no longer needed
            auto issue_pv = [&]() -> bool {
                const volatile Unit& n = units[pc.un % kUnitRing];
                const int j = pc.k >> pc.both, st = pc.k & 1;
                const uint32_t f = (uint32_t)uniform(n.fill0) + (uint32_t)j, b = f & 1u, buf = pc.job % 3u;
                const bool first = pc.both ? j == 0 : pc.k < 2;
                const bool last = pc.both ? j == pc.steps - 1 : pc.k + 2 >= pc.jobs;
                // (at the stream's first job of a tile, the tile before has left O)
                const int used = first ? uniform(st ? n.used1 : n.used0) : 0;
                if (!__all_sync(kAll, there(&p_full[buf], pc.job / 3u) && there(&v_full[b], f >> 1) &&
                                          (!used || there(&o_free[st], (uint32_t)used - 1))))
                    return false;
                asm volatile("tcgen05.fence::after_thread_sync;");
                const uint32_t vb = sb + kOffV + b * 2 * kTermBytes, p_col = tm + buf * kTileKeys, d = tm + kColO + 64u * st;
                const uint32_t more = (pc.both ? j : j >> 1) % kFlush<BF16> ? 1u : 0u;   // O goes on
                // 32 columns of P: the hi terms of 32 keys, then their lo terms
                auto p_at = [&](int ks) { return p_col + 32u * (ks >> 1) + 8u * (ks & 1); };
                // (bf16 in pairs that share their V: with all of lo first 1,110 instead of 990 us;
                // fp32 all of lo first, for the sum's sake, at no cost)
                if constexpr (BF16) {
#pragma unroll 2
                    for (int ks = 0; ks < kTileKeys / 16; ++ks) {
                        const uint64_t v = sw128_desc(vb + 2048u * ks);
                        mma_f16_ta(d, p_at(ks) + 16u, v, kIdescO, ks ? 1u : more);
                        mma_f16_ta(d, p_at(ks), v, kIdescO, 1u);
                    }
                } else {
#pragma unroll 1
                    for (int term = 2; term >= 0; --term) {
                        const uint32_t pt = term == 2 ? 16u : 0u, vt = vb + (term == 1 ? kTermBytes : 0u);
#pragma unroll 2
                        for (int ks = 0; ks < kTileKeys / 16; ++ks)
                            mma_f16_ta(d, p_at(ks) + pt, sw128_desc(vt + 2048u * ks), kIdescO, ks || term < 2 ? 1u : more);
                    }
                }
                commit_elected(smem_u32(&o_done[buf]));
                commit_elected(smem_u32(&v_free[b]));
                if (!pc.both) commit_elected(smem_u32(&v_free[b]));
                if (last) commit_elected(smem_u32(&o_last[st]));
                ++pc.job;
                if (++pc.k == pc.jobs) {
                    ++pc.un;
                    p_more = settle(pc);
                    for (; freed < pc.un; ++freed) unit_read(freed);
                }
                return true;
            };
            uint32_t since = nanoseconds();
            for (uint32_t idle = 0; p_more;) {
                bool some = false;
                // (an S is at most three jobs ahead: the buffer's P . V has been issued)
                if (s_more && sc.job < pc.job + 3u) some = issue_s();
                if (sc.job > pc.job && issue_pv()) some = true;
                if (some) {
                    idle = 0;
                } else if ((++idle & 63u) == 0) {
                    if (__any_sync(kAll, *abort_flag != 0)) break;
                    if (idle == 64) since = nanoseconds();
                    if (__any_sync(kAll, nanoseconds() - since > kWaitLimitNs)) {
                        *abort_flag = 1;
                        break;
                    }
                }
            }
            for (; freed < pc.un; ++freed) unit_read(freed);
            // every MMA issued completes before TMEM is freed, also when cut short
            commit_elected(smem_u32(drained));
            const uint32_t t0 = nanoseconds();
            while (!mbar_try_wait(smem_u32(drained), 0))
                if (nanoseconds() - t0 > kWaitLimitNs) {
                    *abort_flag = 1;
                    break;
                }
        } else if (warp == kUnitWarp) {
            // ---------------------------------------------------------- tiles
            uint32_t un = 0;
            int fills = 0, jobs = 0, halves = 0, used0 = 0, used1 = 0;
            // a place in the ring: its tile may be a long one, so the steps that it takes (2 to 4 us
            // each, 65 ms for 16,384) extend the wait, which the other roles cut short when they stall
            auto place_free = [&]() -> bool {
                if (un < kUnitRing) return true;
                const uint32_t b = smem_u32(&unit_free[un % kUnitRing]), parity = (un / kUnitRing - 1) & 1u;
                int more = units[un % kUnitRing].steps / 16384;
                for (uint32_t i = 1, t0 = nanoseconds(); !mbar_try_wait(b, parity); ++i) {
                    if ((i & 255u) != 0) continue;
                    if (*abort_flag) return false;
                    if (nanoseconds() - t0 <= kWaitLimitNs) continue;
                    if (--more < 0) {
                        *abort_flag = 1;
                        return false;
                    }
                    t0 = nanoseconds();
                }
                return true;
            };
            for (long long x = g0; x < g1; unit_next(a, here)) {
                const long long from = max(x, here.jobs), to = min(here.end, g1);
                x = here.end;
                if (from >= to) {                       // only places before its jobs are in the stretch
                    if (x >= g1) break;
                    continue;
                }
                if (!__all_sync(kAll, place_free())) break;
                if (lane == 0) {
                    volatile Unit& n = units[un % kUnitRing];
                    const int n_rows = tile_n_rows(here.q, here.tile), both = n_rows > kHalfRows;
                    // a step belongs to the CTA that has its first job
                    const int step0 = (int)((from - here.jobs + both) >> both), step1 = (int)((to - here.jobs + both) >> both);
                    n.steps = step1 - step0;
                    n.both = both;
                    n.g = here.g;
                    n.token0 = here.q.row0;
                    n.row0 = here.tile * kTileRows;
                    n.n_rows = n_rows;
                    n.key0 = step0 * kTileKeys;
                    n.key1 = min(step1 * kTileKeys, tile_keys(a, here.q, here.tile));
                    n.first_last = here.q.ctx + here.tile * kTileRows / a.group;
                    n.ctx = here.q.ctx;
                    n.part = here.jobs < g0 ? 0 : here.end > g1 ? 1 : -1;
                    n.fill0 = fills;
                    n.job0 = jobs;
                    n.half0 = halves;
                    n.s = here.s;
                    n.odd = 0;
                    n.used0 = used0;
                    n.used1 = used1;
                    fills += step1 - step0;
                    jobs += (step1 - step0) << both;
                    if (step1 > step0) {
                        halves += 1 + both;
                        ++used0;
                        if (both || step1 > step0 + 1) ++used1;
                    }
                    mbar_arrive(smem_u32(&unit_full[un % kUnitRing]));
                }
                __syncwarp();
                ++un;
                if (x >= g1) break;
            }
            if (__all_sync(kAll, place_free())) {
                if (lane == 0) {
                    units[un % kUnitRing].steps = -1;
                    mbar_arrive(smem_u32(&unit_full[un % kUnitRing]));
                }
            }
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;");
    __syncthreads();
    if (t == 0 && *abort_flag && a.status) atomicExch(a.status, (int)MODEL_ERR_DEVICE);
    if (warp == kMmaWarp) {
        asm volatile("tcgen05.fence::after_thread_sync;");
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols));
    }
}

}  // namespace

cudaError_t launch_paged_attn_tc(const PagedAttnArgs& a, bool bf16, cudaStream_t st) {
    auto* kernel = bf16 ? paged_tc_kernel<true> : paged_tc_kernel<false>;
    const size_t smem = 1024 + kSmemBytes;
    // once per device and format: the shared memory, and that the register split
    // finds the registers it will wait for
    static std::atomic<bool> ready[64][2];
    int device = 0;
    cudaError_t e = cudaGetDevice(&device);
    if (e != cudaSuccess) return e;
    if (device >= 64 || !ready[device][bf16]) {
        if ((e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem)) != cudaSuccess) return e;
        cudaFuncAttributes f;
        if ((e = cudaFuncGetAttributes(&f, kernel)) != cudaSuccess) return e;
        if (f.numRegs != kRegsLaunch) return cudaErrorInvalidConfiguration;
        if (device < 64) ready[device][bf16] = true;
    }
    kernel<<<(unsigned)a.ctas, kThreads, smem, st>>>(a);
    return cudaGetLastError();
}

}  // namespace tie
