// k_paged_tc.cu -- attention of many new rows over a paged cache on the tensor
// cores (head_dim 64), for the sequences that ops_attn.cu's streaming kernel
// leaves to it.
//
// One CTA per SM takes units (paged_attn.cuh): 128 rows -- new tokens times the
// query heads of one K/V head -- against a range of keys in steps of 128, with
// an online softmax:
//
//   S  = Q . K^T    M = 128 rows, N = 128 keys, K = 64 dims
//   O += P . V      M = 128 rows, N = 64 dims,  K = 128 keys
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
//     absolute error of 2^-32 of the largest.
// A scale belongs to one row, so no row's range costs another row bits.
//
// Masks. Keys behind the unit's last visible one and keys of unmapped pages
// are loaded as zero with e = -inf: no comparison is needed except in the
// steps that cross the diagonal, where a masked t is set to -inf. A value that
// is not finite would reach every row of the tile (0 * inf): the loaders put 0
// in its place and raise a flag, and the epilogue adds it to the rows that see
// it.
//
// Warps (640 threads, five warpgroups that share the registers by need):
//   0-7   softmax: warp (q, hf) = (warp % 4, warp / 4) owns TMEM lanes
//         32 q .. 32 q + 31 (a row per thread) and half hf of the columns.
//         The running maximum m moves only when it has grown by more than 8
//         (powers of two), so O is rescaled rarely. Warps 0-3 also bring Q.
//   8-15  loaders: warp w takes keys 16 w .. 16 w + 15 of a step, one page, 32
//         bytes per lane and row; scales, splits and stores them in the
//         128-byte-swizzled layout of the MMA's B operand (K: K-major; V as it
//         lies, MN-major). The next step's rows are in registers by then.
//   16    allocates TMEM, issues the MMAs (17-19 only complete the warpgroup).
// TMEM (512 columns): S of two steps (256), O (64), P hi/lo (128), Q hi/lo (64).
// Barriers as in k_tc_attn.cu; every wait is bounded.
#include <cuda.h>

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <atomic>

#include "paged_attn.cuh"

namespace tie {
namespace {

#include "tc_ptx.cuh"

constexpr int kThreads = 640;
// registers a thread: at launch, and after the warpgroups have shared them out
// (softmax 2 x 128 threads, loaders 2 x 128, MMA 128); the sum must not pass
// what the block was launched with
constexpr int kRegsLaunch = 96, kRegsSoftmax = 120, kRegsLoad = 96, kRegsMma = 40;
static_assert(256 * kRegsSoftmax + 256 * kRegsLoad + 128 * kRegsMma <= kThreads * kRegsLaunch, "register split");
constexpr int kSoftmaxWarps = 8, kLoadWarps = 8;
constexpr unsigned long long kWaitLimitNs = 2000000000ull;  // 2 s
constexpr unsigned kAll = 0xffffffffu;
constexpr float kBase = 7.f;        // the largest probability is 2^7 when m is the maximum
constexpr float kSlack = 8.f;       // m may lag the maximum by this (probabilities up to 2^15)

// shared memory (bytes from the 1024-aligned base)
constexpr uint32_t kTermBytes = kTileKeys * 128;          // 128 rows of 64 fp16
constexpr uint32_t kOffK = 0;                             // two buffers of hi, lo
constexpr uint32_t kOffV = kOffK + 4 * kTermBytes;
constexpr uint32_t kOffKeys = kOffV + 4 * kTermBytes;     // [4][3][128] per key: scale, e, 2^-e
constexpr uint32_t kOffQs = kOffKeys + 4 * 3 * kTileKeys * 4;   // [128] per row
constexpr uint32_t kOffXch = kOffQs + kTileRows * 4;      // [2][2][128] partial maxima / sums
constexpr uint32_t kOffBars = kOffXch + 4 * kTileRows * 4;
constexpr uint32_t kOffSched = kOffBars + 128;
// TMEM columns
constexpr uint32_t kTmemCols = 512, kColO = 256, kColP = 320, kColQ = 448;

// kind::f16 with f16 operands, fp32 accumulation, M = 128
constexpr uint32_t kIdescS = (1u << 4) | ((uint32_t)(kTileKeys >> 3) << 17) | ((uint32_t)(kTileRows >> 4) << 24);
constexpr uint32_t kIdescO = (1u << 4) | (1u << 16) /* B is MN-major */ | ((uint32_t)(kHeadDim >> 3) << 17) |
                             ((uint32_t)(kTileRows >> 4) << 24);

// D += A . B with A in tensor memory (two fp16 of consecutive k per 32-bit
// column). Called by a whole, converged warp, of which one lane issues: with
// one lane in a branch of its own every operand of every MMA would be moved to
// a uniform register there and then, and the MMAs would wait for the moves.
__device__ __forceinline__ void mma_f16_ta(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p, one;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "elect.sync _|one, 0xffffffff;\n\t"
        "@one tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
        ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate));
}

__device__ __forceinline__ void commit_elected(uint32_t bar) {
    asm volatile(
        "{\n\t.reg .pred one;\n\t"
        "elect.sync _|one, 0xffffffff;\n\t"
        "@one tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}"
        ::"r"(bar)
        : "memory");
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

// 64 columns of the warp's 32 lanes, by two loads and one wait
__device__ __forceinline__ void tmem_ld64(uint32_t taddr, uint32_t (&r)[64]) {
    __syncwarp();
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        uint32_t* x = r + 32 * h;
        asm volatile(
            "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
            "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
            "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
            : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3]), "=r"(x[4]), "=r"(x[5]), "=r"(x[6]), "=r"(x[7]),
              "=r"(x[8]), "=r"(x[9]), "=r"(x[10]), "=r"(x[11]), "=r"(x[12]), "=r"(x[13]), "=r"(x[14]), "=r"(x[15]),
              "=r"(x[16]), "=r"(x[17]), "=r"(x[18]), "=r"(x[19]), "=r"(x[20]), "=r"(x[21]), "=r"(x[22]), "=r"(x[23]),
              "=r"(x[24]), "=r"(x[25]), "=r"(x[26]), "=r"(x[27]), "=r"(x[28]), "=r"(x[29]), "=r"(x[30]), "=r"(x[31])
            : "r"(taddr + 32u * h));
    }
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
    // no use of a register is moved ahead of the wait
#pragma unroll
    for (int i = 0; i < 64; ++i) asm volatile("" : "+r"(r[i]));
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
        asm volatile("ld.global.nc.v8.f32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                     : "=f"(x[0]), "=f"(x[1]), "=f"(x[2]), "=f"(x[3]), "=f"(x[4]), "=f"(x[5]), "=f"(x[6]), "=f"(x[7])
                     : "l"(static_cast<const float*>(base) + at));
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
        asm volatile("ld.global.nc.v4.b32 {%0, %1, %2, %3}, [%4];"
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

template <bool BF16>
__global__ void __launch_bounds__(kThreads, 1) paged_tc_kernel(PagedAttnArgs a) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    float* s_keys = reinterpret_cast<float*>(smem + kOffKeys);
    float* s_qs = reinterpret_cast<float*>(smem + kOffQs);
    float* s_xch = reinterpret_cast<float*>(smem + kOffXch);
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + kOffBars);
    uint64_t* k_full = bars + 0;    // [2] keys of the step in buffer b written (loader warps)
    uint64_t* v_full = bars + 2;    // [2] values and per-key numbers written (loader warps)
    uint64_t* s_full = bars + 4;    // [2] S computed: key buffer b free (MMA commit)
    uint64_t* v_free = bars + 6;    // [2] P . V of value buffer b done (MMA commit)
    uint64_t* p_full = bars + 8;    // P written, O rescaled (softmax warps)
    uint64_t* o_full = bars + 9;    // P . V done: P free (MMA commit)
    uint64_t* drained = bars + 10;  // every MMA of the unit done (MMA commit)
    uint64_t* q_full = bars + 11;   // Q of the unit in TMEM (softmax warps 0-3)
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 12);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    volatile int* odd_values = reinterpret_cast<volatile int*>(tmem_slot + 2);   // a value of the unit is not finite
    const int t = threadIdx.x, warp = t >> 5, lane = t & 31;

    if (t == 0) {
        for (int b = 0; b < 2; ++b) {
            mbar_init(smem_u32(&k_full[b]), kLoadWarps);
            mbar_init(smem_u32(&v_full[b]), kLoadWarps);
            mbar_init(smem_u32(&s_full[b]), 1);
            mbar_init(smem_u32(&v_free[b]), 1);
        }
        mbar_init(smem_u32(p_full), kSoftmaxWarps);
        mbar_init(smem_u32(o_full), 1);
        mbar_init(smem_u32(drained), 1);
        mbar_init(smem_u32(q_full), 4);
        *abort_flag = 0;
        *odd_values = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == kSoftmaxWarps + kLoadWarps) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                     ::"r"(smem_u32(tmem_slot)), "r"(kTmemCols));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    __shared__ ScheduleScratch<kThreads> scratch;
    Schedule sch;
    build_schedule<kThreads>(a, 1, reinterpret_cast<int*>(smem + kOffSched), &scratch, t, &sch);
    asm volatile("tcgen05.fence::before_thread_sync;");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;");
    const uint32_t tmem = *tmem_slot;
    const uint32_t lane_addr = tmem + ((uint32_t)((warp & 3) * 32) << 16);

    auto wait = [&](const uint64_t* bar, uint32_t parity) -> bool {
        const uint32_t b = smem_u32(bar);
        if (mbar_try_wait(b, parity)) return true;
        const unsigned long long t0 = globaltimer_ns();
        for (uint32_t i = 1;; ++i) {
            if (mbar_try_wait(b, parity)) return true;
            if ((i & 255u) == 0) {
                if (*abort_flag) return false;
                if (globaltimer_ns() - t0 > kWaitLimitNs) break;
            }
        }
        *abort_flag = 1;
        if (a.status) atomicExch(a.status, (int)MODEL_ERR_DEVICE);
        return false;
    };

    auto wait_all = [&](const uint64_t* bar, uint32_t parity) -> bool { return __all_sync(kAll, wait(bar, parity)); };

    const int units = sch.unit[a.n_seq];
    const size_t w = (size_t)a.n_kv_head * kHeadDim;

    // Each role runs its own loop over the CTA's units (a register count per
    // role needs code of its own), all in the same order; `base` counts the
    // steps of the units before, so buffers and parities run on.
    struct Unit {
        SeqShape q;
        int s, in, sp, g, row0, n_rows, key0, key1, steps;
        int first_last;   // the least last visible position of the rows
        const int32_t* table;
    };
    auto unit_of = [&](int u) {
        Unit x;
        x.s = owner_of(sch.unit, a.n_seq, u);
        x.q = seq_shape(a, x.s);
        x.sp = splits_of(x.q, sch.chunk);
        x.in = u - sch.unit[x.s];
        x.g = x.in % a.n_kv_head;
        const int split = x.in / a.n_kv_head % x.sp, tile = x.in / a.n_kv_head / x.sp;
        x.row0 = tile * kTileRows;
        x.n_rows = min(kTileRows, x.q.rows - x.row0);
        // keys [key0, key1): the split's, up to the tile's last visible one
        x.key0 = split * sch.chunk * kTileKeys;
        const int seen = x.q.ctx + (x.row0 + x.n_rows - 1) / a.group + 1;
        x.key1 = (int)min((long long)seen, (long long)x.key0 + (long long)sch.chunk * kTileKeys);
        x.steps = x.key1 > x.key0 ? (x.key1 - x.key0 + kTileKeys - 1) / kTileKeys : 0;
        x.table = a.table + (size_t)x.s * a.width;
        x.first_last = x.q.ctx + x.row0 / a.group;
        return x;
    };
    // the end of a unit, for all threads: nothing of it is in flight; false ends the loop
    auto unit_end = [&]() -> bool {
        asm volatile("tcgen05.fence::before_thread_sync;");
        asm volatile("bar.sync 0;" ::: "memory");
        asm volatile("tcgen05.fence::after_thread_sync;");
        const bool go = !*abort_flag;
        if (t == 0) *odd_values = 0;
        asm volatile("bar.sync 0;" ::: "memory");
        return go;
    };

    if (warp < kSoftmaxWarps) {
        // ------------------------------------------------------------ softmax
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsSoftmax));
        uint32_t base = 0, unit_no = 0;
        for (int u = blockIdx.x; u < units; u += gridDim.x) {
            const Unit n = unit_of(u);
            // tcgen05.ld / .st and the named barriers are warp-collective: a
            // failed wait clears `ok` and the n.steps run on, storing nothing.
            const int qq = warp & 3, hf = warp >> 2, r = qq * 32 + lane;
            const int i = min(n.row0 + r, n.q.rows - 1), last = n.q.ctx + i / a.group;
            auto pair_sync = [&]() { asm volatile("bar.sync %0, 64;" ::"r"(1 + qq) : "memory"); };
            float m = -INFINITY, l = 0.f;
            bool ok = true;
            if (hf == 0 && n.steps > 0) {
                // Q: TMEM lane = row, a thread's 64 dims
                float x[64], mx = 0.f;
                const float* from = a.q + (size_t)(n.q.row0 + i / a.group) * a.ldq + (n.g * a.group + i % a.group) * kHeadDim;
#pragma unroll
                for (int c = 0; c < 16; ++c) {
                    const float4 v = r < n.n_rows ? __ldg(reinterpret_cast<const float4*>(from) + c)
                                                : make_float4(0.f, 0.f, 0.f, 0.f);
                    x[4 * c] = v.x; x[4 * c + 1] = v.y; x[4 * c + 2] = v.z; x[4 * c + 3] = v.w;
                }
#pragma unroll
                for (int c = 0; c < 64; ++c) mx = max_abs(mx, x[c]);
                const int e = row_exponent(mx, 15);
                const float sc = copysignf(pow2_biased(268 - e), a.scale2);   // the scale's sign goes to Q: s_qs >= 0
                s_qs[r] = pow2_biased(e - 14) * fabsf(a.scale2);
                uint32_t h[32], lo[32];
#pragma unroll
                for (int c = 0; c < 32; ++c) split2(x[2 * c] * sc, x[2 * c + 1] * sc, h[c], lo[c]);
                tmem_st32(lane_addr + kColQ, h);
                tmem_st32(lane_addr + kColQ + 32u, lo);
                asm volatile("tcgen05.fence::before_thread_sync;");
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(q_full));
            }
            pair_sync();     // the partner warp's s_qs
            const float qs = s_qs[r];
            for (int j = 0; j < n.steps; ++j) {
                const uint32_t jj = base + (uint32_t)j, b = jj & 1u;
                ok = wait_all(&v_full[b], (jj >> 1) & 1u) && ok;
                ok = wait_all(&s_full[b], (jj >> 1) & 1u) && ok;
                asm volatile("tcgen05.fence::after_thread_sync;");
                const float* keys = s_keys + (jj & 3u) * 3 * kTileKeys;
                const int pos = n.key0 + j * kTileKeys;
                const bool diagonal = pos + kTileKeys - 1 > n.first_last;
                uint32_t x[64];
                tmem_ld64(lane_addr + b * kTileKeys + 64u * hf, x);
                float mt = -INFINITY;
                f32x2 c[4];        // a page's factor of S, and what its exponent adds
                float ev[4];
                if (diagonal) {
                    // a scale per key; t in place of S
#pragma unroll
                    for (int k = 0; k < 16; ++k) {
                        const float4 ks = reinterpret_cast<const float4*>(keys + 64 * hf)[k];
                        const float4 ee = reinterpret_cast<const float4*>(keys + kTileKeys + 64 * hf)[k];
                        const int p0 = pos + 64 * hf + 4 * k;
                        auto t_of = [&](int d, float f, float e) {
                            float v = fmaf(__uint_as_float(x[4 * k + d]) * qs, f, e);
                            if (p0 + d > last) v = -INFINITY;
                            x[4 * k + d] = __float_as_uint(v);
                            mt = fmaxf(mt, v);
                        };
                        t_of(0, ks.x, ee.x);
                        t_of(1, ks.y, ee.y);
                        t_of(2, ks.z, ee.z);
                        t_of(3, ks.w, ee.w);
                    }
                } else {
                    // a scale per page: the largest t is the largest S's
#pragma unroll
                    for (int g = 0; g < 4; ++g) {
                        const float f = qs * keys[4 * hf + g];
                        ev[g] = keys[kTileKeys + 4 * hf + g];
                        float sm = __uint_as_float(x[16 * g]);
#pragma unroll
                        for (int d = 1; d < 16; ++d) sm = fmaxf(sm, __uint_as_float(x[16 * g + d]));
                        mt = fmaxf(mt, fmaf(sm, f, ev[g]));
                        c[g] = pair(f, f);
                    }
                }
                s_xch[(b * 2 + hf) * kTileRows + r] = mt;
                pair_sync();
                mt = fmaxf(mt, s_xch[(b * 2 + (hf ^ 1)) * kTileRows + r]);
                float alpha = 1.f;
                if (mt > m + kSlack || m == -INFINITY) {      // also the first finite maximum
                    alpha = ex2_ftz(m - mt);                  // m = -inf: 0 (or, mt = -inf too, unused)
                    if (mt == -INFINITY) alpha = 1.f;
                    m = mt;
                }
                const float lift = m == -INFINITY ? 0.f : kBase - m;
                // probabilities, their sum, and their two terms: hi[k] packs columns
                // 2 k and 2 k + 1, x[k] then holds their lo terms
                uint32_t hi[32];
                float sum = 0.f;
                if (diagonal) {
#pragma unroll
                    for (int k = 0; k < 16; ++k) {
                        const float4 iv = reinterpret_cast<const float4*>(keys + 2 * kTileKeys + 64 * hf)[k];
                        const float p0 = ex2_ftz(__uint_as_float(x[4 * k]) + lift);
                        const float p1 = ex2_ftz(__uint_as_float(x[4 * k + 1]) + lift);
                        const float p2 = ex2_ftz(__uint_as_float(x[4 * k + 2]) + lift);
                        const float p3 = ex2_ftz(__uint_as_float(x[4 * k + 3]) + lift);
                        sum = fmaf(p3, iv.w, fmaf(p2, iv.z, fmaf(p1, iv.y, fmaf(p0, iv.x, sum))));
                        split2(p0, p1, hi[2 * k], x[2 * k]);
                        split2(p2, p3, hi[2 * k + 1], x[2 * k + 1]);
                    }
                } else {
#pragma unroll
                    for (int g = 0; g < 4; ++g) {
                        const f32x2 add = pair(ev[g] + lift, ev[g] + lift);
                        f32x2 part = pair(0.f, 0.f);
#pragma unroll
                        for (int d = 0; d < 8; ++d) {
                            const int k = 8 * g + d;
                            const float2 e = unpair(fma2(pair(__uint_as_float(x[2 * k]), __uint_as_float(x[2 * k + 1])), c[g], add));
                            const float p0 = ex2_ftz(e.x), p1 = ex2_ftz(e.y);
                            part = add2(part, pair(p0, p1));
                            split2(p0, p1, hi[k], x[k]);
                        }
                        const float2 ps = unpair(part);
                        sum = fmaf(ps.x + ps.y, keys[2 * kTileKeys + 4 * hf + g], sum);
                    }
                }
                l = fmaf(l, alpha, sum);
                if (j > 0) {
                    // P . V of step j - 1 is done: P is free, and O can be rescaled
                    ok = wait_all(o_full, (jj - 1) & 1u) && ok;
                    asm volatile("tcgen05.fence::after_thread_sync;");
                    if (__any_sync(kAll, alpha != 1.f)) {
                        uint32_t v[32];
                        tmem_ld32(lane_addr + kColO + 32u * hf, v);
#pragma unroll
                        for (int d = 0; d < 32; ++d) v[d] = __float_as_uint(__uint_as_float(v[d]) * alpha);
                        tmem_st32(lane_addr + kColO + 32u * hf, v);
                    }
                }
                tmem_st32(lane_addr + kColP + 32u * hf, hi);
#pragma unroll
                for (int k = 0; k < 32; ++k) hi[k] = x[k];
                tmem_st32(lane_addr + kColP + 64u + 32u * hf, hi);
                asm volatile("tcgen05.fence::before_thread_sync;");
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(p_full));
            }
            float o[32];
            if (n.steps > 0) {
                ok = wait_all(o_full, (base + (uint32_t)n.steps - 1) & 1u) && ok;
                asm volatile("tcgen05.fence::after_thread_sync;");
                pair_sync();     // both halves have read the last maxima
                s_xch[hf * kTileRows + r] = l;
                pair_sync();
                l = s_xch[r] + s_xch[kTileRows + r];
                uint32_t v[32];
                tmem_ld32(lane_addr + kColO + 32u * hf, v);
#pragma unroll
                for (int d = 0; d < 32; ++d) o[d] = __uint_as_float(v[d]);
            } else {
#pragma unroll
                for (int d = 0; d < 32; ++d) o[d] = 0.f;
            }
            if (ok && r < n.n_rows) {
                if (*odd_values) {
                    // values that are not finite, for the rows that see them
                    for (int key = n.key0; key < min(n.key1, last + 1); ++key) {
                        const int e = __ldg(n.table + key / kPageRows);
                        if (e < 0 || e >= a.n_pages) continue;
                        const size_t at = ((size_t)e * kPageRows + key % kPageRows) * w + n.g * kHeadDim + 32 * hf;
#pragma unroll
                        for (int d = 0; d < 32; ++d) {
                            float x;
                            if constexpr (BF16) x = __bfloat162float(static_cast<const __nv_bfloat16*>(a.v)[at + d]);
                            else x = static_cast<const float*>(a.v)[at + d];
                            if (!(fabsf(x) < INFINITY)) o[d] += x;
                        }
                    }
                }
                if (n.sp == 1) {
                    const float inv = l == 0.f ? 0.f : 1.f / l;
                    float4* to = reinterpret_cast<float4*>(a.out + (size_t)(n.q.row0 + i / a.group) * a.ldo +
                                                           (n.g * a.group + i % a.group) * kHeadDim + 32 * hf);
#pragma unroll
                    for (int c = 0; c < 8; ++c)
                        to[c] = l == 0.f ? make_float4(0.f, 0.f, 0.f, 0.f)
                                         : make_float4(o[4 * c] * inv, o[4 * c + 1] * inv, o[4 * c + 2] * inv, o[4 * c + 3] * inv);
                } else {
                    const size_t pu = (size_t)(sch.part[n.s] + n.in) * kTileRows + r;
                    float4* to = reinterpret_cast<float4*>(a.part_o[1] + pu * kHeadDim + 32 * hf);
#pragma unroll
                    for (int c = 0; c < 8; ++c) to[c] = make_float4(o[4 * c], o[4 * c + 1], o[4 * c + 2], o[4 * c + 3]);
                    if (hf == 0) {
                        a.part_ml[1][2 * pu] = m == -INFINITY ? m : m - kBase;
                        a.part_ml[1][2 * pu + 1] = l;
                    }
                }
            }
            base += (uint32_t)n.steps;
            unit_no += n.steps > 0;
            if (!unit_end()) break;
        }
    } else if (warp < kSoftmaxWarps + kLoadWarps) {
        // ------------------------------------------------------------ loaders
        uint32_t base = 0, unit_no = 0;
        for (int u = blockIdx.x; u < units; u += gridDim.x) {
            const Unit n = unit_of(u);
            const int lw = warp - kSoftmaxWarps, sub = lane >> 3, dl = lane & 7;
            Row8<BF16> kr[4], vr[4];
            // this warp's page of step j: its 16 positions, or -1
            auto page_of = [&](int j) {
                const int p = (n.key0 + j * kTileKeys) / kPageRows + lw;
                if (j >= n.steps || (long long)p * kPageRows >= n.key1) return -1;
                const int e = __ldg(n.table + p);
                return e >= 0 && e < a.n_pages ? e : -1;
            };
            auto load = [&](Row8<BF16>(&r)[4], const void* from, int j, int page) {
                const int pos = n.key0 + j * kTileKeys + lw * kPageRows;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int row = 4 * i + sub;
                    if (page >= 0 && pos + row < n.key1)
                        r[i].load(from, ((size_t)page * kPageRows + row) * w + n.g * kHeadDim + 8 * dl);
                    else
                        r[i].zero();
                }
            };
            int page = page_of(0), page_next = page_of(1);
            load(kr, a.k, 0, page);
            load(vr, a.v, 0, page);
            for (int j = 0; j < n.steps; ++j) {
                const uint32_t jj = base + (uint32_t)j, b = jj & 1u, use = jj >> 1;
                const int pos = n.key0 + j * kTileKeys + lw * kPageRows;
                float* keys = s_keys + (jj & 3u) * 3 * kTileKeys;
                // key buffer b is free once S of step j - 2 is computed
                if (jj >= 2 && !wait(&s_full[b], (use - 1) & 1u)) break;
                uint8_t* kb = smem + kOffK + b * 2 * kTermBytes;
                const bool diagonal = n.key0 + j * kTileKeys + kTileKeys - 1 > n.first_last;
                // largest magnitudes: of each row, or of the page in every entry
                auto magnitudes = [&](const Row8<BF16>(&r)[4], float (&mx)[4]) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        float y[8];
                        r[i].get(y);
                        mx[i] = max_abs8(y);
                    }
                    if (diagonal) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) mx[i] = lanes_max(mx[i], 8);
                    } else {
                        mx[0] = mx[1] = mx[2] = mx[3] = lanes_max(max_abs(max_abs(mx[0], mx[1]), max_abs(mx[2], mx[3])), 32);
                    }
                };
                float mx[4];
                magnitudes(kr, mx);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int row = lw * kPageRows + 4 * i + sub, e = row_exponent(mx[i], 15);
                    float y[8];
                    kr[i].get(y);
                    store_terms<BF16>(kb, (uint32_t)(row * 128 + ((dl ^ (row & 7)) << 4)), y, pow2_biased(268 - e));
                    if (diagonal ? dl == 0 : i == 0 && lane == 0) keys[diagonal ? lw * kPageRows + 4 * i + sub : lw] = pow2_biased(e - 14);
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&k_full[b]));
                load(kr, a.k, j + 1, page_next);
                // value buffer b is free once P . V of step j - 2 is done
                if (jj >= 2 && !wait(&v_free[b], (use - 1) & 1u)) break;
                uint8_t* vb = smem + kOffV + b * 2 * kTermBytes;
                magnitudes(vr, mx);
                if (__any_sync(kAll, !(fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) < INFINITY) ||
                                         mx[0] != mx[0] || mx[1] != mx[1] || mx[2] != mx[2] || mx[3] != mx[3])) {
                    // rare: elements that are not finite are left to the epilogue
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (vr[i].clear_odd()) *odd_values = 1;
                    magnitudes(vr, mx);
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int row = lw * kPageRows + 4 * i + sub, e = row_exponent(mx[i], 60);
                    float y[8];
                    vr[i].get(y);
                    store_terms<BF16>(vb, (uint32_t)(row * 128 + ((dl ^ (row & 7)) << 4)), y, pow2_biased(268 - e));
                    if (diagonal ? dl == 0 : i == 0 && lane == 0) {
                        const int at = diagonal ? row : lw;
                        const bool there = page >= 0 && pos + 4 * i + sub < n.key1;
                        keys[kTileKeys + at] = there ? (float)(e - 141) : -INFINITY;
                        keys[2 * kTileKeys + at] = pow2_biased(268 - e);
                    }
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&v_full[b]));
                load(vr, a.v, j + 1, page_next);
                page = page_next;
                page_next = page_of(j + 2);
            }
            base += (uint32_t)n.steps;
            unit_no += n.steps > 0;
            if (!unit_end()) break;
        }
    } else {
        // ---------------------------------------------------------------- MMA
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsMma));
        uint32_t base = 0, unit_no = 0;
        for (int u = blockIdx.x; u < units; u += gridDim.x) {
            const Unit n = unit_of(u);
            const int steps = __shfl_sync(kAll, n.steps, 0);   // the same in all lanes, and known to be
            if (warp == kSoftmaxWarps + kLoadWarps && steps > 0) {
                const uint32_t sb = smem_u32(smem), tm = __shfl_sync(kAll, tmem, 0);
                auto issue_s = [&](int j) -> bool {
                    const uint32_t jj = base + (uint32_t)j, b = jj & 1u;
                    if (!wait_all(&k_full[b], (jj >> 1) & 1u)) return false;
                    asm volatile("tcgen05.fence::after_thread_sync;");
                    const uint32_t kb = sb + kOffK + b * 2 * kTermBytes, d = tm + b * kTileKeys;
#pragma unroll
                    for (int ks = 0; ks < kHeadDim / 16; ++ks) {
                        const uint32_t q_hi = tm + kColQ + 8u * ks, q_lo = q_hi + 32u;
                        const uint64_t k_hi = sw128_desc(kb + 32u * ks);
                        mma_f16_ta(d, q_lo, k_hi, kIdescS, ks ? 1u : 0u);
                        if constexpr (!BF16) mma_f16_ta(d, q_hi, sw128_desc(kb + kTermBytes + 32u * ks), kIdescS, 1u);
                        mma_f16_ta(d, q_hi, k_hi, kIdescS, 1u);
                    }
                    commit_elected(smem_u32(&s_full[b]));
                    return true;
                };
                bool go = wait_all(q_full, unit_no & 1u) && issue_s(0) && (steps < 2 || issue_s(1));
                for (int j = 0; go && j < steps; ++j) {
                    const uint32_t jj = base + (uint32_t)j, b = jj & 1u;
                    if (!wait_all(p_full, jj & 1u) || !wait_all(&v_full[b], (jj >> 1) & 1u)) break;
                    asm volatile("tcgen05.fence::after_thread_sync;");
                    const uint32_t vb = sb + kOffV + b * 2 * kTermBytes, d = tm + kColO;
#pragma unroll
                    for (int ks = 0; ks < kTileKeys / 16; ++ks) {
                        const uint32_t p_hi = tm + kColP + 8u * ks, p_lo = p_hi + 64u;
                        const uint64_t v_hi = sw128_desc(vb + 2048u * ks);
                        mma_f16_ta(d, p_lo, v_hi, kIdescO, (j | ks) ? 1u : 0u);
                        if constexpr (!BF16) mma_f16_ta(d, p_hi, sw128_desc(vb + kTermBytes + 2048u * ks), kIdescO, 1u);
                        mma_f16_ta(d, p_hi, v_hi, kIdescO, 1u);
                    }
                    commit_elected(smem_u32(o_full));
                    commit_elected(smem_u32(&v_free[b]));
                    // S of step j + 2 into the buffer that step j's softmax has read
                    if (j + 2 < steps && !issue_s(j + 2)) break;
                }
                // arrives once every MMA issued above has completed, also when cut short
                commit_elected(smem_u32(drained));
                const unsigned long long t0 = globaltimer_ns();
                while (!mbar_try_wait(smem_u32(drained), unit_no & 1u))
                    if (globaltimer_ns() - t0 > kWaitLimitNs) {
                        *abort_flag = 1;
                        if (a.status) atomicExch(a.status, (int)MODEL_ERR_DEVICE);
                        break;
                    }
            }
            base += (uint32_t)n.steps;
            unit_no += n.steps > 0;
            if (!unit_end()) break;
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;");
    __syncthreads();
    if (warp == kSoftmaxWarps + kLoadWarps) {
        asm volatile("tcgen05.fence::after_thread_sync;");
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols));
    }
}

}  // namespace

cudaError_t launch_paged_attn_tc(const PagedAttnArgs& a, bool bf16, int sms, cudaStream_t st) {
    auto* kernel = bf16 ? paged_tc_kernel<true> : paged_tc_kernel<false>;
    const size_t smem = 1024 + kOffSched + 2 * (size_t)(a.n_seq + 1) * sizeof(int);
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return e;
    // the register split waits for registers that a smaller launch would not have
    static std::atomic<int> checked[2] = {{0}, {0}};
    if (!checked[bf16]) {
        cudaFuncAttributes f;
        if ((e = cudaFuncGetAttributes(&f, kernel)) != cudaSuccess) return e;
        if (f.numRegs != kRegsLaunch) return cudaErrorInvalidConfiguration;
        checked[bf16] = 1;
    }
    kernel<<<(unsigned)sms, kThreads, smem, st>>>(a);
    return cudaGetLastError();
}

}  // namespace tie
