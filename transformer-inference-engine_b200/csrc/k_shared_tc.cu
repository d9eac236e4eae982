// k_shared_tc.cu -- attention over a prefix that many rows share, on tcgen05: 128 rows of a
// group (its new tokens times the query heads of a K/V head) against 64 keys a step.
//
// The numbers are those of ops_shared.cu: Q, scaled, the weights P and, over fp32 pages, K and
// V are sums of three bf16 terms, exactly; levels of 8 bits and bf16 numbers are one. S = Q K^T
// and the step's O = P V are sums of the terms' products (six for fp32, three for the others),
// the small ones first, since the MMA cuts its sums off. Each step's O starts at zero and is
// added, in fp32 registers, to what a row has: O = O 2^(m_before - m) + step's.
//
// A CTA has all roles and half of an SM: two CTAs fill each other's waits. 12 warps:
//   0-3   softmax: a thread per row. Read S from TMEM, add the step before's O to the row's, write
//         P, three terms of two bf16 a column, into TMEM. With bf16 pages a step's 64 scores stay in
//         registers and the next step's S is computed meanwhile; the other formats' loaders need
//         those registers, and S is read twice (maximum; weights).
//   4-7   loaders: a page of 16 keys each; K and V as terms into 128-byte-swizzled rows
//         (K K-major; V as it lies, MN-major). The next step's rows are in registers by then;
//         bf16 rows need no conversion and are copied to three stages, two steps ahead.
//   8     allocates TMEM and issues the MMAs. 9-11 only complete the warpgroup.
// TMEM (256 columns): P 96, S 64, O 64. Shared memory: Q 48 KB, K and V 8 KB a term each.
// The MMAs complete in order. A warp arrives at no barrier for a step before that
// barrier's phase of the step before has completed (loaders wait for S, softmax warps for O).
//
// Measured (B200, the whole call: this kernel, the sequences' own positions, the join): 64
// answers x 1-4 tokens over bf16 pages, 14336 shared positions, 8 K/V heads: 116 us (on mma.sync
// 271), about 80 of them this kernel's. Steps to it: a pair of threads per row, which exchange their
// maxima, 133; a thread per row and pairs of fp32 numbers in an instruction, 120; S of the next step
// ahead, 118; its keys told of before the next rows are asked for (a page's table entry a step sooner), 113;
// a barrier for each stage, and places and sums that are there before any wait, 116. What bounds it is the way
// round a step: of about 5000 cycles (two CTAs side by side) a softmax warp takes 700 for S and the
// maximum, 800 to add O, 1600 for weights and terms (512 of them exponentials, at the rate of the SM), 700 to
// write and report P; P V and the waits take the others. Issue slots are 48 % used, the tensor pipe
// 33 %. A wait that reads the timer at every try takes 1 us.
//
// Every wait is bounded (2 s): on expiry it raises the abort flag, which ends every other wait;
// the roles run out without storing, the copies and MMAs issued are drained and TMEM is freed. The join finds
// places and parts of this call all the same, since they are written before anything is waited for: a part
// that was not finished has a maximum and a sum that are NaN, and so has the row.
#include <cuda.h>

#include <cuda_bf16.h>

#include "shared_attn.cuh"
#include "shared_stages.h"

namespace tie {
namespace {

#include "tc_ptx.cuh"

constexpr int kThreads = 384, kSoftmaxWarps = 4, kLoadWarps = 4, kMmaWarp = 8;
constexpr unsigned kAll = 0xffffffffu;
constexpr uint32_t kDrainLimitNs = 2000000000u;
constexpr int kKeys = kTcPages * kPageRows;            // of a step
// registers a thread: at launch, and as the warpgroups share them out (rows that are converted
// take the loaders more)
constexpr int kRegsLaunch = 80, kRegsMma = 24;
template <int FMT>
constexpr int kRegsLoad = FMT == TIE_KV_F32 ? 80 : FMT == TIE_KV_BF16 ? 48 : 64;
template <int FMT>
constexpr int kRegsSoftmax = 3 * kRegsLaunch - kRegsMma - kRegsLoad<FMT>;
template <int FMT>
constexpr bool kRegsFit = 128 * (kRegsSoftmax<FMT> + kRegsLoad<FMT> + kRegsMma) <= kThreads * kRegsLaunch && kRegsSoftmax<FMT> % 8 == 0;
static_assert(kRegsFit<TIE_KV_F32> && kRegsFit<TIE_KV_BF16> && kRegsFit<TIE_KV_INT8>, "register split");

constexpr uint32_t kQTerm = kTcRows * 128, kKvTerm = kKeys * 128;    // bytes of a term
constexpr uint32_t kColP = 0, kColS = 96, kColO = 160, kTmemCols = 256;

template <int FMT>
struct Tc {
    static constexpr int kTerms = FMT == TIE_KV_F32 ? 3 : 1;
    // bf16 rows go from memory straight to their places, two steps ahead, and need few of the loaders'
    // registers: a step's scores stay in the softmax warps', and the next one's are computed meanwhile
    static constexpr bool kAhead = FMT == TIE_KV_BF16;
    static constexpr uint32_t kStages = kAhead ? 3 : 1;
    using Stage = Stages<kStages>;
    static constexpr uint32_t kStage = 2 * kTerms * kKvTerm, kValues = kTerms * kKvTerm;    // bytes of a stage; to its values
    static constexpr uint32_t kOffQ = 0, kOffKv = 3 * kQTerm;
    static constexpr uint32_t kOffScales = kOffKv + kStages * kStage;    // [step % 2][key, value][64]
    static constexpr uint32_t kOffThere = kOffScales + 4 * kKeys * 4;    // [step % 4][page]: its positions
    static constexpr uint32_t kOffBars = kOffThere + 4 * kTcPages * 4;
    static constexpr uint32_t kBytes = kOffBars + (7 + kStages + 1) / 2 * 16;
};

// kind::f16 with bf16 operands, fp32 accumulation, M = 128, N = 64
constexpr uint32_t kIdesc = (1u << 4) | (1u << 7) | (1u << 10) | (64u >> 3 << 17) | ((uint32_t)(kTcRows >> 4) << 24);
constexpr uint32_t kIdescO = kIdesc | (1u << 16);      // B is MN-major

// 32 columns of the warp's 32 lanes read, 16 written
__device__ __forceinline__ void tmem_begin32(uint32_t taddr, uint32_t* r) {
    __syncwarp();
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr));
}
// The reads are done. What a read is to return is an operand, so that no use of it comes before this.
__device__ __forceinline__ void tmem_wait_ld(uint32_t* r) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
                 :
                 : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
    __syncwarp();
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
                 ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
                 : "memory");
}

__device__ __forceinline__ float max3(float x, float y, float z) {
    float m;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(m) : "f"(x), "f"(y), "f"(z));
    return m;
}

// Bytes 0 and 2 of a word, as signed levels, in a pair of bf16: 0x4300 | u is 128 + u for
// u < 128, and 0x4380 is 256, so (128 + low 7 bits) - (128 + sign bit) is the level.
__device__ __forceinline__ uint32_t levels2(uint32_t w) {
    const uint32_t low = (w & 0x007f007fu) | 0x43004300u, sign = (w & 0x00800080u) | 0x43004300u;
    const __nv_bfloat162 v = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&low), *reinterpret_cast<const __nv_bfloat162*>(&sign));
    return *reinterpret_cast<const uint32_t*>(&v);
}

// 8 elements of a row of a page, as they lie
template <int FMT>
struct Row8 {
    static constexpr int kWords = FMT == TIE_KV_F32 ? 8 : FMT == TIE_KV_BF16 ? 4 : 2;
    uint32_t x[kWords];
    __device__ __forceinline__ void load(const char* p) {
        if constexpr (kWords == 8)
            asm volatile("ld.global.nc.L1::no_allocate.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                         : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3]), "=r"(x[4]), "=r"(x[5]), "=r"(x[6]), "=r"(x[7])
                         : "l"(p));
        else if constexpr (kWords == 4)
            asm volatile("ld.global.nc.L1::no_allocate.v4.b32 {%0, %1, %2, %3}, [%4];"
                         : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3])
                         : "l"(p));
        else
            asm volatile("ld.global.nc.L1::no_allocate.v2.b32 {%0, %1}, [%2];" : "=r"(x[0]), "=r"(x[1]) : "l"(p));
    }
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int i = 0; i < kWords; ++i) x[i] = 0u;
    }
    // its terms, 16 bytes each, `term` bytes apart
    __device__ __forceinline__ void store(uint8_t* to, uint32_t term) const {
        if constexpr (FMT == TIE_KV_F32) {
            uint32_t t[4][3];
#pragma unroll
            for (int i = 0; i < 4; ++i) split3(__uint_as_float(x[2 * i]), __uint_as_float(x[2 * i + 1]), t[i]);
#pragma unroll
            for (int e = 0; e < 3; ++e) *reinterpret_cast<uint4*>(to + e * term) = make_uint4(t[0][e], t[1][e], t[2][e], t[3][e]);
        } else if constexpr (FMT == TIE_KV_BF16) {
            *reinterpret_cast<uint4*>(to) = make_uint4(x[0], x[1], x[2], x[3]);
        } else {
            uint32_t y[4];
#pragma unroll
            for (int i = 0; i < 2; ++i) {          // bytes 0, 2 and 1, 3 as pairs, then in order
                const uint32_t even = levels2(x[i]), odd = levels2(x[i] >> 8);
                y[2 * i] = __byte_perm(even, odd, 0x5410);
                y[2 * i + 1] = __byte_perm(even, odd, 0x7632);
            }
            *reinterpret_cast<uint4*>(to) = make_uint4(y[0], y[1], y[2], y[3]);
        }
    }
};

// A part of an item, as every role finds it for itself.
struct Job {
    int row0, rows, i0, head, keys;    // the unit's first row and its rows, the item's first of them, K/V head, positions
    int b0, b1;                        // steps
    int whole, parts;                  // whole: no stretch cuts it; parts: how many the item has, if this is the first
    const int32_t* table;
};

template <int FMT>
__global__ void __launch_bounds__(kThreads, 2) shared_tc_kernel(const __grid_constant__ SharedArgs a) {
    using T = Tc<FMT>;
    constexpr int kTerms = T::kTerms;
    // (what comes before the call is done before the kernel after this one may begin)
    pdl_wait();
    pdl_trigger();
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    float* s_scales = reinterpret_cast<float*>(smem + T::kOffScales);
    int* s_there = reinterpret_cast<int*>(smem + T::kOffThere);
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + T::kOffBars);
    uint64_t* q_full = bars;             // an item's Q written (loader warps)
    uint64_t* k_full = bars + 1;         // a step's keys written (loader warps)
    uint64_t* v_full = bars + 2;         // a step's values written (loader warps)
    uint64_t* s_full = bars + 3;         // a step's S computed (commit); its scales and what is there of it
                                         // written (loader warps)
    uint64_t* s_free = bars + 4;         // a step's S read (softmax warps, kAhead)
    uint64_t* p_full = bars + 5;         // a step's P written, the O before it read (softmax warps)
    uint64_t* drained = bars + 6;        // every MMA done (commit)
    uint64_t* o_full = bars + 7;         // [stage] a step's O computed, its stage read (commit): shared_stages.h
    __shared__ uint32_t s_tmem;
    __shared__ volatile int s_abort;
    __shared__ ScheduleScratch<kThreads> scratch;
    const int t = threadIdx.x, warp = t >> 5, lane = t & 31;
    const Line& line = a.line[0];

    if (t == 0) {
        mbar_init(smem_u32(q_full), kLoadWarps);
        mbar_init(smem_u32(k_full), kLoadWarps);
        mbar_init(smem_u32(v_full), kLoadWarps);
        mbar_init(smem_u32(s_full), 1 + kLoadWarps);
        mbar_init(smem_u32(p_full), kSoftmaxWarps);
        mbar_init(smem_u32(s_free), kSoftmaxWarps);
        for (uint32_t i = 0; i < T::kStages; ++i) mbar_init(smem_u32(o_full + i), 1);
        mbar_init(smem_u32(drained), 1);
        s_abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == kMmaWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                     ::"r"(smem_u32(&s_tmem)), "r"(kTmemCols));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    // (the line lies behind everything else: the roles walk it to the end)
    const Plan plan = build_plan<kThreads>(a, line.u0, line.u1, smem + T::kBytes, &scratch, t);
    const long long* const base = plan.base;
    asm volatile("tcgen05.fence::before_thread_sync;");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;");
    const uint32_t tmem = s_tmem;
    const int n_units = line.u1 - line.u0, me = blockIdx.x;
    const long long total = base[n_units], share = share_of(line, total);
    long long x = me * share;
    const long long end = min(x + share, total);
    int u = x < end ? owner_of<long long>(base, n_units, x) : 0;
    // the next part from place x of unit u on that has steps, in this CTA's stretch
    auto find_at = [&](long long& x, int& u, Job& job) -> bool {
        while (x < end) {
            while (base[u + 1] <= x) ++u;          // (units without rows have no places)
            const UnitShape s = unit_shape(a, plan.n, line.u0 + u);
            const int places = unit_places(s, line);
            const long long in = x - base[u], item = quotient(in, places);
            const int off = (int)(in - item * places);
            const int stop = (int)min((long long)places, off + (end - x));
            const long long first = x - off;       // the item's first place
            x += stop - off;
            if (stop - 1 <= max(off - 1, 0)) continue;
            const int tile = (int)quotient(item, line.heads);
            job.row0 = s.row0;
            job.rows = s.rows;
            job.i0 = tile * kTcRows;
            job.head = (int)item - tile * line.heads;
            job.keys = s.keys;
            job.b0 = max(off - 1, 0);
            job.b1 = stop - 1;
            job.table = a.ptable + (size_t)(line.u0 + u) * a.pwidth;
            const bool begins = first + 1 >= me * share;
            job.whole = begins && first + places <= (me + 1) * share;
            job.parts = job.whole ? 1 : begins ? 1 + (int)quotient(first + places - 1 - me * share, share) : 0;
            return true;
        }
        return false;
    };
    auto find = [&](Job& job) -> bool { return find_at(x, u, job); };
    auto wait = [&](const uint64_t* bar, uint32_t parity) -> bool {
        const uint32_t b = smem_u32(bar);
        uint32_t t0 = 0;                 // (the timer is not looked at before a wait has become long)
        for (uint32_t i = 1; !mbar_try_wait(b, parity); ++i) {
            if ((i & 255u) != 0) continue;
            if (i == 256) t0 = nanoseconds();
            if (s_abort || nanoseconds() - t0 > a.wait_ns) {
                s_abort = 1;
                return false;
            }
        }
        return true;
    };
    auto wait_all = [&](const uint64_t* bar, uint32_t phase) -> bool { return __all_sync(kAll, wait(bar, phase & 1u)); };
    // the O of a step is computed
    auto wait_o = [&](uint32_t step) -> bool { return wait_all(o_full + T::Stage::of(step), T::Stage::phase(step)); };
    auto arrive = [&](const uint64_t* bar) {
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(bar));
    };
    Job job;
    uint32_t f = 0, un = 0;              // steps and items so far
    bool ok = true;

    if (warp < kSoftmaxWarps) {
        // ------------------------------------------------------------ softmax
        // (tcgen05.ld and .st are the warp's: so is every condition around them)
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsSoftmax<FMT>));
        constexpr int kChunk = T::kAhead ? 64 : 32;       // scores in registers at a time
        const int r = warp * 32 + lane;
        const uint32_t lanes = tmem + ((uint32_t)(warp * 32) << 16);
        // where this thread's row of a part goes (-1: it has none): of the whole items' rows, or of the parts'
        auto place_of = [&](const Job& job) -> long long {
            const int i = job.i0 + r;
            if (i >= job.rows) return -1;
            const int tok = a.by_group(i), h = job.head * a.group + i - tok * a.group;
            return (long long)(job.row0 + tok) * a.n_head + h;
        };
        auto slot_of = [&](const Job& job) { return (2 * (size_t)me + (job.parts > 0)) * kTcRows + r; };
        auto ml_of = [&](const Job& job, long long place) {
            return reinterpret_cast<float2*>(job.whole ? a.whole_ml[0] + 2 * place : line.part_ml + 2 * slot_of(job));
        };
        {
            // what the join reads, as it is if nothing more comes of it (the first S is on its way meanwhile)
            long long ahead = x;
            int unit = u;
            Job part;
            while (find_at(ahead, unit, part)) {
                const long long place = place_of(part);
                if (place < 0) continue;
                if (part.parts) a.place[0][place] = make_int2(part.whole ? -1 : (int)slot_of(part), part.parts);
                *ml_of(part, place) = make_float2(NAN, NAN);
            }
        }
        for (; ok && find(job); ++un) {
            float m = -INFINITY, alpha = 1.f;
            Float2x l(0.f, 0.f), o[32];
#pragma unroll
            for (int d = 0; d < 32; ++d) o[d] = Float2x(0.f, 0.f);
            // the step before has left its O: it is relative to that step's maximum
            auto add_step = [&]() {
                const Float2x by(alpha, alpha);
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    uint32_t y[32];
                    tmem_begin32(lanes + kColO + 32u * h, y);
                    tmem_wait_ld(y);
#pragma unroll
                    for (int d = 0; d < 16; ++d)
                        o[16 * h + d] = fma2(o[16 * h + d], by, Float2x(__uint_as_float(y[2 * d]), __uint_as_float(y[2 * d + 1])));
                }
            };
#pragma unroll 1
            for (int b = job.b0; b < job.b1; ++b, ++f) {
                if (!(ok = wait_all(s_full, f))) break;
                asm volatile("tcgen05.fence::after_thread_sync;");
                const int4 there = *reinterpret_cast<const int4*>(s_there + (f & 3u) * kTcPages);
                const bool all = there.x + there.y + there.z + there.w == kKeys;
                const float4* ks = reinterpret_cast<const float4*>(s_scales + (f & 1u) * 2 * kKeys);
                const float4* vs = ks + kKeys / 4;
                // the step's scores c0 ..
                auto scores = [&](int c0, uint32_t (&y)[kChunk]) {
#pragma unroll
                    for (int i = 0; i < kChunk; i += 32) tmem_begin32(lanes + kColS + c0 + i, y + i);
#pragma unroll
                    for (int i = 0; i < kChunk; i += 32) tmem_wait_ld(y + i);
                    if constexpr (T::kAhead) {
                        asm volatile("tcgen05.fence::before_thread_sync;");
                        arrive(s_free);
                    }
                    if constexpr (FMT == TIE_KV_INT8) {
#pragma unroll
                        for (int i = 0; i < kChunk / 4; ++i) {
                            const float4 z = ks[c0 / 4 + i];
                            y[4 * i] = __float_as_uint(__uint_as_float(y[4 * i]) * z.x);
                            y[4 * i + 1] = __float_as_uint(__uint_as_float(y[4 * i + 1]) * z.y);
                            y[4 * i + 2] = __float_as_uint(__uint_as_float(y[4 * i + 2]) * z.z);
                            y[4 * i + 3] = __float_as_uint(__uint_as_float(y[4 * i + 3]) * z.w);
                        }
                    }
                    if (!all) {
                        const int n0 = c0 ? there.z : there.x, n1 = c0 ? there.w : there.y;
#pragma unroll
                        for (int i = 0; i < kChunk; ++i)
                            if ((i & 15) >= (i < 16 ? n0 : i < 32 ? n1 : i < 48 ? there.z : there.w)) y[i] = 0xff800000u;
                    }
                };
                uint32_t y[kChunk];
                float top = -INFINITY;
#pragma unroll 1
                for (int c0 = 0; c0 < kKeys; c0 += kChunk) {
                    scores(c0, y);
                    float a0 = max3(top, __uint_as_float(y[0]), __uint_as_float(y[1])), a1 = max3(-INFINITY, __uint_as_float(y[2]), __uint_as_float(y[3]));
#pragma unroll
                    for (int i = 4; i < kChunk; i += 4) {
                        a0 = max3(a0, __uint_as_float(y[i]), __uint_as_float(y[i + 1]));
                        a1 = max3(a1, __uint_as_float(y[i + 2]), __uint_as_float(y[i + 3]));
                    }
                    top = fmaxf(a0, a1);
                }
                // (the step before's O is computed: so P may be written over its P)
                if (b > job.b0) {
                    if (!(ok = wait_o(f - 1))) break;
                    asm volatile("tcgen05.fence::after_thread_sync;");
                    add_step();
                }
                const float m_new = fmaxf(m, top), from = m_new == -INFINITY ? 0.f : m_new;
                alpha = ex2_ftz(m - from);
                m = m_new;
                l = l * Float2x(alpha, alpha);
                const Float2x less(-from, -from), weight(kWeight, kWeight);
#pragma unroll 1
                for (int c0 = 0; c0 < kKeys; c0 += kChunk) {
                    if constexpr (kChunk < kKeys) scores(c0, y);
#pragma unroll
                    for (int h = 0; h < kChunk / 32; ++h) {
                        float w[32];
#pragma unroll
                        for (int i = 0; i < 32; i += 2) {
                            float x0, x1;
                            (Float2x(__uint_as_float(y[32 * h + i]), __uint_as_float(y[32 * h + i + 1])) + less).get(x0, x1);
                            const Float2x e = Float2x(ex2_ftz(x0), ex2_ftz(x1)) * weight;
                            l = l + e;
                            e.get(w[i], w[i + 1]);
                        }
                        if constexpr (FMT == TIE_KV_INT8) {
#pragma unroll
                            for (int i = 0; i < 8; ++i) {
                                const float4 z = vs[c0 / 4 + 8 * h + i];
                                w[4 * i] *= z.x;
                                w[4 * i + 1] *= z.y;
                                w[4 * i + 2] *= z.z;
                                w[4 * i + 3] *= z.w;
                            }
                        }
#pragma unroll
                        for (int e = 0; e < 3; ++e) {
                            uint32_t p[16];
#pragma unroll
                            for (int i = 0; i < 16; ++i) {
                                p[i] = terms2(w[2 * i], w[2 * i + 1]);
                                if (e < 2) rest2(w[2 * i], w[2 * i + 1]);
                            }
                            tmem_st16(lanes + kColP + 32u * e + c0 / 2 + 16u * h, p);
                        }
                    }
                }
                asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                asm volatile("tcgen05.fence::before_thread_sync;");
                arrive(p_full);
            }
            if (!ok || !(ok = wait_o(f - 1))) break;
            asm volatile("tcgen05.fence::after_thread_sync;");
            // (the next item's first P, which lets its O begin, is written after this)
            add_step();
            const long long place = place_of(job);
            if (place >= 0) {
                float* to = job.whole ? a.whole_o[0] + place * kHeadDim : line.part_o + slot_of(job) * kHeadDim;
                float l0, l1;
                l.get(l0, l1);
                *ml_of(job, place) = make_float2(m, l0 + l1);
#pragma unroll
                for (int d = 0; d < 16; ++d) {
                    float4 v;
                    o[2 * d].get(v.x, v.y);
                    o[2 * d + 1].get(v.z, v.w);
                    reinterpret_cast<float4*>(to)[d] = v;
                }
            }
            __syncwarp();
        }
    } else if (warp < kSoftmaxWarps + kLoadWarps) {
        // ------------------------------------------------------------ loaders
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsLoad<FMT>));
        constexpr int kBytes = FMT == TIE_KV_F32 ? 4 : FMT == TIE_KV_BF16 ? 2 : 1;
        const int lw = warp - kSoftmaxWarps, sub = lane >> 3, dl = lane & 7;
        const size_t w = (size_t)a.n_kv_head * kHeadDim * kBytes;     // bytes of a row
        Row8<FMT> k[4], v[4];
        float ks = 0.f, vs = 0.f;
        int page = 0, there = 0;             // of the step that is loaded: this warp's page, its positions
        int now_at = 0;                      // the step that f counts
        int entry = -1;                      // of the step after it (looked up a step ahead)
        auto entry_of = [&](int b) {
            const int p = b * kTcPages + lw;
            return job.keys > p * kPageRows ? __ldg(job.table + p) : -1;
        };
        auto page_of = [&](int b) {          // steps in order, from `entry`'s
            const int left = job.keys - (b * kTcPages + lw) * kPageRows, e = entry;
            entry = entry_of(b + 1);
            const bool mapped = e >= 0 && e < a.n_pages;
            page = mapped ? e : 0;           // (what is not there is read from the pool's first page, and cleared)
            there = mapped ? min(left, kPageRows) : 0;
        };
        auto row_at = [&](const void* pool, int i) {
            return static_cast<const char*>(pool) + ((size_t)page * kPageRows + 4 * i + sub) * w + (size_t)job.head * kHeadDim * kBytes +
                   8 * dl * kBytes;
        };
        auto load_k = [&]() {
#pragma unroll
            for (int i = 0; i < 4; ++i) k[i].load(row_at(a.k, i));
            if constexpr (FMT == TIE_KV_INT8) ks = __ldg(a.ks + ((size_t)page * a.n_kv_head + job.head) * kPageRows + (lane & 15));
        };
        auto load_v = [&]() {
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i].load(row_at(a.v, i));
            if constexpr (FMT == TIE_KV_INT8) vs = __ldg(a.vs + ((size_t)page * a.n_kv_head + job.head) * kPageRows + (lane & 15));
        };
        auto store = [&](uint8_t* to, Row8<FMT>(&rows)[4], int n) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (4 * i + sub >= n) rows[i].zero();
                const int row = lw * kPageRows + 4 * i + sub;
                rows[i].store(to + row * 128 + ((dl ^ (row & 7)) << 4), kKvTerm);
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        };
        for (; ok && find(job); ++un) {
            // a step's rows, and zeros for what is not there, to its stage, once that has been read
            auto copy = [&](int b) -> bool {
                if (b < job.b1) {
                    const uint32_t step = f + (uint32_t)(b - now_at);
                    if (T::Stage::used(step) && !wait_o(T::Stage::before(step))) return false;
                    page_of(b);
                    if (lane == 0) s_there[(step & 3u) * kTcPages + lw] = there;
                    const uint32_t to = smem_u32(smem + T::kOffKv + T::Stage::of(step) * T::kStage);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int row = lw * kPageRows + 4 * i + sub;
                        const uint32_t at = to + row * 128 + ((dl ^ (row & 7)) << 4);
                        const int bytes = 4 * i + sub < there ? 16 : 0;
                        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(at), "l"(row_at(a.k, i)), "r"(bytes) : "memory");
                        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(at + T::kValues), "l"(row_at(a.v, i)), "r"(bytes)
                                     : "memory");
                    }
                }
                asm volatile("cp.async.commit_group;" ::: "memory");
                return true;
            };
            now_at = job.b0;
            entry = entry_of(job.b0);
            if constexpr (T::kAhead) {
                if (!(ok = copy(job.b0) && copy(job.b0 + 1))) break;
            } else {
                page_of(job.b0);
            }
            if constexpr (FMT == TIE_KV_INT8) {
                load_k();
                load_v();
            }
            // Q: 32 rows a warp, four times four. (The last S of the item before has been waited for.)
#pragma unroll 1
            for (int i0 = 0; i0 < 8; i0 += 4) {
                Row8<TIE_KV_F32> q[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int at = job.i0 + lw * 32 + 4 * (i0 + i) + sub;
                    if (at < job.rows) {
                        const int tok = a.by_group(at), h = job.head * a.group + at - tok * a.group;
                        const float4* from = reinterpret_cast<const float4*>(a.q + (size_t)(job.row0 + tok) * a.ldq + h * kHeadDim + 8 * dl);
                        const float4 y = __ldg(from), z = __ldg(from + 1);
                        const float s[8] = {y.x, y.y, y.z, y.w, z.x, z.y, z.z, z.w};
#pragma unroll
                        for (int d = 0; d < 8; ++d) q[i].x[d] = __float_as_uint(s[d]);
                    } else {
                        q[i].zero();
                    }
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int row = lw * 32 + 4 * (i0 + i) + sub;
#pragma unroll
                    for (int d = 0; d < 8; ++d) q[i].x[d] = __float_as_uint(__uint_as_float(q[i].x[d]) * a.scale2);
                    q[i].store(smem + T::kOffQ + row * 128 + ((dl ^ (row & 7)) << 4), kQTerm);
                }
            }
            if constexpr (FMT == TIE_KV_F32) {     // (in registers that Q has left)
                load_k();
                load_v();
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            arrive(q_full);
            if constexpr (T::kAhead) {
                auto arrive_copied = [&]() {
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    arrive(s_full);
                    if (lane == 0) mbar_arrive(smem_u32(k_full));
                };
                asm volatile("cp.async.wait_group 1;" ::: "memory");
                arrive_copied();
#pragma unroll 1
                for (int b = job.b0; b < job.b1; ++b, ++f) {
                    now_at = b;
                    if (!(ok = wait_all(s_full, f))) break;
                    if (b + 1 < job.b1) {        // the next step's rows were asked for a step ago
                        asm volatile("cp.async.wait_group 0;" ::: "memory");
                        arrive_copied();
                    }
                    if (b + 2 < job.b1 && !(ok = copy(b + 2))) break;
                }
            } else {
#pragma unroll 1
                for (int b = job.b0; b < job.b1; ++b, ++f) {
                    // (the step before's S has been waited for: K is free)
                    const int now = there;
                    store(smem + T::kOffKv, k, now);
                    if constexpr (FMT == TIE_KV_INT8) {
                        if (lane < kPageRows) {
                            float* to = s_scales + (f & 1u) * 2 * kKeys + lw * kPageRows + lane;
                            to[0] = lane < now ? ks : 0.f;
                            to[kKeys] = lane < now ? vs : 0.f;
                        }
                    }
                    if (lane == 0) s_there[(f & 3u) * kTcPages + lw] = now;
                    arrive(s_full);
                    if (lane == 0) mbar_arrive(smem_u32(k_full));
                    if (b + 1 < job.b1) {
                        page_of(b + 1);
                        load_k();
                    }
                    if (f && !(ok = wait_o(f - 1))) break;       // the step before's V has been read
                    store(smem + T::kOffKv + T::kValues, v, now);
                    arrive(v_full);
                    if (b + 1 < job.b1) load_v();
                    if (!(ok = wait_all(s_full, f))) break;      // K has been read
                }
            }
        }
        if constexpr (T::kAhead) asm volatile("cp.async.wait_all;" ::: "memory");      // (cut short: copies are on their way)
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsMma));
        if (warp == kMmaWarp) {
            // ------------------------------------------------------------ MMA
            const uint32_t sb = __shfl_sync(kAll, smem_u32(smem), 0), tm = __shfl_sync(kAll, tmem, 0);
            // products of terms (of A, of B), the smallest first: two and zero, ...
            constexpr int kProducts = kTerms == 3 ? 6 : 3;
            constexpr uint32_t kA = kTerms == 3 ? 0x001102u : 0x012u;      // a digit each, the first lowest
            constexpr uint32_t kB = kTerms == 3 ? 0x010120u : 0x000u;
            // (a drill: a wait for what does not come)
            if (a.stall && (blockIdx.x & 1)) ok = wait_all(drained, 0);
            for (; ok && find(job); ++un) {
                if (!(ok = wait_all(q_full, un))) break;
                const int steps = __shfl_sync(kAll, job.b1 - job.b0, 0);
                auto stage = [&](uint32_t step) { return sb + T::kOffKv + T::Stage::of(step) * T::kStage; };
                // S of a step whose keys are there, where the S before it has been read
                auto scores = [&](uint32_t step) -> bool {
                    if (!wait_all(k_full, step)) return false;
                    asm volatile("tcgen05.fence::after_thread_sync;");
#pragma unroll 1
                    for (int z = 0; z < kProducts; ++z) {
                        const uint32_t q = sb + T::kOffQ + (kA >> (4 * z) & 15u) * kQTerm;
                        const uint32_t k = stage(step) + (kB >> (4 * z) & 15u) * kKvTerm;
#pragma unroll
                        for (int s = 0; s < 4; ++s)
                            mma_f16(tm + kColS, sw128_desc(q + 32u * s), sw128_desc(k + 32u * s), kIdesc, z || s ? 1u : 0u);
                    }
                    commit_elected(smem_u32(s_full));
                    return true;
                };
                if (T::kAhead && !(ok = scores(f))) break;
#pragma unroll 1
                for (int b = 0; b < steps; ++b, ++f) {
                    if constexpr (T::kAhead) {
                        if (b + 1 < steps && !(ok = wait_all(s_free, f) && scores(f + 1))) break;
                    } else if (!(ok = scores(f))) {
                        break;
                    }
                    // (copied rows: k_full was for both)
                    if (!(ok = wait_all(p_full, f) && (T::kAhead || wait_all(v_full, f)))) break;
                    asm volatile("tcgen05.fence::after_thread_sync;");
#pragma unroll 1
                    for (int z = 0; z < kProducts; ++z) {
                        const uint32_t p = tm + kColP + (kA >> (4 * z) & 15u) * 32u;
                        const uint32_t v = stage(f) + T::kValues + (kB >> (4 * z) & 15u) * kKvTerm;
#pragma unroll
                        for (int s = 0; s < 4; ++s)
                            mma_f16_ta(tm + kColO, p + 8u * s, sw128_desc(v + 2048u * s), kIdescO, z || s ? 1u : 0u);
                    }
                    commit_elected(smem_u32(o_full + T::Stage::of(f)));
                }
            }
            // every MMA issued completes before TMEM is freed, also when cut short
            commit_elected(smem_u32(drained));
            const uint32_t t0 = nanoseconds();
            while (!mbar_try_wait(smem_u32(drained), 0))
                if (nanoseconds() - t0 > kDrainLimitNs) {
                    s_abort = 1;
                    break;
                }
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;");
    if (warp == kMmaWarp)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols));
    if (t == 0 && s_abort && a.status) *a.status = MODEL_ERR_DEVICE;
}

}  // namespace

int shared_tc_ctas(int sms) { return 2 * sms; }

cudaError_t launch_shared_tc(const SharedArgs& a, int format, cudaStream_t st) {
    auto* kernel = format == TIE_KV_INT8 ? shared_tc_kernel<TIE_KV_INT8>
                                         : format == TIE_KV_BF16 ? shared_tc_kernel<TIE_KV_BF16> : shared_tc_kernel<TIE_KV_F32>;
    const size_t fixed = 1024 + (format == TIE_KV_INT8 ? Tc<TIE_KV_INT8>::kBytes
                                                       : format == TIE_KV_BF16 ? Tc<TIE_KV_BF16>::kBytes : Tc<TIE_KV_F32>::kBytes);
    // (always the most that any call wants: calls on other threads set it too)
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                               (int)(fixed + plan_bytes(kOpsMaxSeqs, kOpsMaxSeqs, kOpsMaxSeqs)));
    if (e != cudaSuccess) return e;
    const size_t smem = fixed + plan_bytes(a.line[0].u1 - a.line[0].u0, a.n_seq, a.n_group);
    return launch_pdl(kernel, dim3((unsigned)a.line[0].teams), dim3(kThreads), smem, st, a);
}

}  // namespace tie
