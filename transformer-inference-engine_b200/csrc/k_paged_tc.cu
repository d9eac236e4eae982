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

// D += A . B with A in tensor memory (two fp16 of consecutive k per 32-bit column)
__device__ __forceinline__ void mma_f16_ta(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
        ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate));
}

__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float2 unpack2(uint32_t u) { return __half22float2(*reinterpret_cast<const __half2*>(&u)); }

// (a, b) as two packed fp16 terms each: hi, and lo in a float's bits
__device__ __forceinline__ void split2(float a, float b, uint32_t& hi, float& lo) {
    hi = pack2(a, b);
    const float2 f = unpack2(hi);
    lo = __uint_as_float(pack2(a - f.x, b - f.y));
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
};

__device__ __forceinline__ float group8_max(float m) {
#pragma unroll
    for (int o = 4; o; o >>= 1) m = max_abs(m, __shfl_xor_sync(kAll, m, o));
    return m;
}

// Scales 8 elements by 2^(268 - e - 127), splits them, and stores the terms at
// the row's 16-byte chunk c of a 128-byte-swizzled operand.
template <bool BF16>
__device__ __forceinline__ void store_terms(uint8_t* hi, uint32_t off, float (&y)[8], float scale) {
    uint32_t h[4], l[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float a = y[2 * i] * scale, b = y[2 * i + 1] * scale;
        h[i] = pack2(a, b);
        if constexpr (!BF16) {
            const float2 f = unpack2(h[i]);
            l[i] = pack2(a - f.x, b - f.y);
        }
    }
    *reinterpret_cast<uint4*>(hi + off) = make_uint4(h[0], h[1], h[2], h[3]);
    if constexpr (!BF16) *reinterpret_cast<uint4*>(hi + kTermBytes + off) = make_uint4(l[0], l[1], l[2], l[3]);
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

    const int units = sch.unit[a.n_seq];
    const size_t w = (size_t)a.n_kv_head * kHeadDim;

    // Each role runs its own loop over the CTA's units (a register count per
    // role needs code of its own), all in the same order; `base` counts the
    // steps of the units before, so buffers and parities run on.
    struct Unit {
        SeqShape q;
        int s, in, sp, g, row0, n_rows, key0, key1, steps;
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
            const int first_last = n.q.ctx + n.row0 / a.group;   // the least last visible position of the tile
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
                const float sc = pow2_biased(268 - e);
                s_qs[r] = pow2_biased(e - 14) * a.scale2;
                uint32_t h[32];
#pragma unroll
                for (int c = 0; c < 32; ++c) split2(x[2 * c] * sc, x[2 * c + 1] * sc, h[c], x[c]);
                tmem_st32(lane_addr + kColQ, h);
#pragma unroll
                for (int c = 0; c < 32; ++c) h[c] = __float_as_uint(x[c]);
                tmem_st32(lane_addr + kColQ + 32u, h);
                asm volatile("tcgen05.fence::before_thread_sync;");
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(q_full));
            }
            pair_sync();     // the partner warp's s_qs
            const float qs = s_qs[r];
            for (int j = 0; j < n.steps; ++j) {
                const uint32_t jj = base + (uint32_t)j, b = jj & 1u;
                ok = __all_sync(kAll, wait(&v_full[b], (jj >> 1) & 1u)) && ok;
                ok = __all_sync(kAll, wait(&s_full[b], (jj >> 1) & 1u)) && ok;
                asm volatile("tcgen05.fence::after_thread_sync;");
                const float4* keys = reinterpret_cast<const float4*>(s_keys + (jj & 3u) * 3 * kTileKeys + 64 * hf);
                float x[64];
                {
                    uint32_t v[32];
                    tmem_ld32(lane_addr + b * kTileKeys + 64u * hf, v);
#pragma unroll
                    for (int c = 0; c < 32; ++c) x[c] = __uint_as_float(v[c]);
                    tmem_ld32(lane_addr + b * kTileKeys + 64u * hf + 32u, v);
#pragma unroll
                    for (int c = 0; c < 32; ++c) x[32 + c] = __uint_as_float(v[c]);
                }
#pragma unroll
                for (int c = 0; c < 16; ++c) {
                    const float4 ks = keys[c], ev = keys[kTileKeys / 4 + c];
                    x[4 * c] = fmaf(x[4 * c] * qs, ks.x, ev.x);
                    x[4 * c + 1] = fmaf(x[4 * c + 1] * qs, ks.y, ev.y);
                    x[4 * c + 2] = fmaf(x[4 * c + 2] * qs, ks.z, ev.z);
                    x[4 * c + 3] = fmaf(x[4 * c + 3] * qs, ks.w, ev.w);
                }
                const int pos = n.key0 + j * kTileKeys;
                if (pos + kTileKeys - 1 > first_last) {       // the step crosses the diagonal
#pragma unroll
                    for (int c = 0; c < 64; ++c)
                        if (pos + 64 * hf + c > last) x[c] = -INFINITY;
                }
                float mt = x[0];
#pragma unroll
                for (int c = 1; c < 64; ++c) mt = fmaxf(mt, x[c]);
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
                // probabilities, their sum, and their two terms: hi[c] packs columns
                // 2 c and 2 c + 1, x[c] then holds the bits of their lo terms
                uint32_t hi[32];
                float sum = 0.f;
#pragma unroll
                for (int c = 0; c < 16; ++c) {
                    const float4 iv = keys[2 * (kTileKeys / 4) + c];
                    const float p0 = ex2_ftz(x[4 * c] + lift), p1 = ex2_ftz(x[4 * c + 1] + lift);
                    const float p2 = ex2_ftz(x[4 * c + 2] + lift), p3 = ex2_ftz(x[4 * c + 3] + lift);
                    sum = fmaf(p0, iv.x, sum);
                    sum = fmaf(p1, iv.y, sum);
                    sum = fmaf(p2, iv.z, sum);
                    sum = fmaf(p3, iv.w, sum);
                    split2(p0, p1, hi[2 * c], x[2 * c]);
                    split2(p2, p3, hi[2 * c + 1], x[2 * c + 1]);
                }
                l = fmaf(l, alpha, sum);
                if (j > 0) {
                    // P . V of step j - 1 is done: P is free, and O can be rescaled
                    ok = __all_sync(kAll, wait(o_full, (jj - 1) & 1u)) && ok;
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
                for (int c = 0; c < 32; ++c) hi[c] = __float_as_uint(x[c]);
                tmem_st32(lane_addr + kColP + 64u + 32u * hf, hi);
                asm volatile("tcgen05.fence::before_thread_sync;");
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(p_full));
            }
            float o[32];
            if (n.steps > 0) {
                ok = __all_sync(kAll, wait(o_full, (base + (uint32_t)n.steps - 1) & 1u)) && ok;
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
                float* keys = s_keys + (jj & 3u) * 3 * kTileKeys + lw * kPageRows;
                // key buffer b is free once S of step j - 2 is computed
                if (jj >= 2 && !wait(&s_full[b], (use - 1) & 1u)) break;
                uint8_t* kb = smem + kOffK + b * 2 * kTermBytes;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int row = lw * kPageRows + 4 * i + sub;
                    float y[8];
                    kr[i].get(y);
                    float mx = 0.f;
#pragma unroll
                    for (int c = 0; c < 8; ++c) mx = max_abs(mx, y[c]);
                    const int e = row_exponent(group8_max(mx), 15);
                    store_terms<BF16>(kb, (uint32_t)(row * 128 + ((dl ^ (row & 7)) << 4)), y, pow2_biased(268 - e));
                    if (dl == 0) keys[4 * i + sub] = pow2_biased(e - 14);
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&k_full[b]));
                load(kr, a.k, j + 1, page_next);
                // value buffer b is free once P . V of step j - 2 is done
                if (jj >= 2 && !wait(&v_free[b], (use - 1) & 1u)) break;
                uint8_t* vb = smem + kOffV + b * 2 * kTermBytes;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int row = lw * kPageRows + 4 * i + sub;
                    float y[8];
                    vr[i].get(y);
                    float mx = 0.f;
#pragma unroll
                    for (int c = 0; c < 8; ++c) mx = max_abs(mx, y[c]);
                    mx = group8_max(mx);
                    if (__any_sync(kAll, !(mx < INFINITY))) {   // rare: leave those elements to the epilogue
                        mx = 0.f;
#pragma unroll
                        for (int c = 0; c < 8; ++c) {
                            if (!(fabsf(y[c]) < INFINITY)) {
                                y[c] = 0.f;
                                *odd_values = 1;
                            }
                            mx = max_abs(mx, y[c]);
                        }
                        mx = group8_max(mx);
                    }
                    const int e = row_exponent(mx, 60);
                    store_terms<BF16>(vb, (uint32_t)(row * 128 + ((dl ^ (row & 7)) << 4)), y, pow2_biased(268 - e));
                    if (dl == 0) {
                        const bool there = page >= 0 && pos + 4 * i + sub < n.key1;
                        keys[kTileKeys + 4 * i + sub] = there ? (float)(e - 141) : -INFINITY;
                        keys[2 * kTileKeys + 4 * i + sub] = pow2_biased(268 - e);
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
            if (warp == kSoftmaxWarps + kLoadWarps && lane == 0 && n.steps > 0) {
                const uint32_t sb = smem_u32(smem);
                auto issue_s = [&](int j) -> bool {
                    const uint32_t jj = base + (uint32_t)j, b = jj & 1u;
                    if (!wait(&k_full[b], (jj >> 1) & 1u)) return false;
                    asm volatile("tcgen05.fence::after_thread_sync;");
                    const uint32_t kb = sb + kOffK + b * 2 * kTermBytes, d = tmem + b * kTileKeys;
#pragma unroll
                    for (int ks = 0; ks < kHeadDim / 16; ++ks) {
                        const uint32_t q_hi = tmem + kColQ + 8u * ks, q_lo = q_hi + 32u;
                        const uint64_t k_hi = sw128_desc(kb + 32u * ks);
                        mma_f16_ta(d, q_lo, k_hi, kIdescS, ks ? 1u : 0u);
                        if constexpr (!BF16) mma_f16_ta(d, q_hi, sw128_desc(kb + kTermBytes + 32u * ks), kIdescS, 1u);
                        mma_f16_ta(d, q_hi, k_hi, kIdescS, 1u);
                    }
                    mma_commit(smem_u32(&s_full[b]));
                    return true;
                };
                bool go = wait(q_full, unit_no & 1u) && issue_s(0) && (n.steps < 2 || issue_s(1));
                for (int j = 0; go && j < n.steps; ++j) {
                    const uint32_t jj = base + (uint32_t)j, b = jj & 1u;
                    if (!wait(p_full, jj & 1u) || !wait(&v_full[b], (jj >> 1) & 1u)) break;
                    asm volatile("tcgen05.fence::after_thread_sync;");
                    const uint32_t vb = sb + kOffV + b * 2 * kTermBytes, d = tmem + kColO;
#pragma unroll
                    for (int ks = 0; ks < kTileKeys / 16; ++ks) {
                        const uint32_t p_hi = tmem + kColP + 8u * ks, p_lo = p_hi + 64u;
                        const uint64_t v_hi = sw128_desc(vb + 2048u * ks);
                        mma_f16_ta(d, p_lo, v_hi, kIdescO, (j | ks) ? 1u : 0u);
                        if constexpr (!BF16) mma_f16_ta(d, p_hi, sw128_desc(vb + kTermBytes + 2048u * ks), kIdescO, 1u);
                        mma_f16_ta(d, p_hi, v_hi, kIdescO, 1u);
                    }
                    mma_commit(smem_u32(o_full));
                    mma_commit(smem_u32(&v_free[b]));
                    // S of step j + 2 into the buffer that step j's softmax has read
                    if (j + 2 < n.steps && !issue_s(j + 2)) break;
                }
                // arrives once every MMA issued above has completed, also when cut short
                mma_commit(smem_u32(drained));
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
