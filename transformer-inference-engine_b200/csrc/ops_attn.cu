// ops_attn.cu -- causal attention of new tokens over a paged cache: the entry
// point, the streaming kernel for sequences of few rows, and the join of split
// sequences.
//
// The reference attends one new token of its one sequence (src/model.c:826-850)
// or a whole prompt to itself (src/model.c:705-732); here any number of new
// tokens per sequence attend to everything cached before them and to
// themselves:
//
//   out = sum_j softmax_j(scale q . k_j) v_j,   j <= ctx + i,
//
// with an online softmax (running maximum and sum in fp32) over the keys, each
// read once through the page table.
#include "paged_attn.cuh"

#include <cooperative_groups.h>
#include <cuda_bf16.h>

#include <climits>
#include <cmath>

namespace tie {
namespace {

namespace cg = cooperative_groups;

// ------------------------------------------------------- few rows: streaming --
// Bound by the reading of K and V. A CTA of 8 warps per unit; warp w takes the
// unit's pages w, w + 8, ... Its lanes load a page's 16 keys and values as 16
// 16-byte loads each (lane = 16 half + dl: position 2 i + half, dims 4 dl ..
// 4 dl + 3; 8-byte loads for bf16), all in flight before the first product.
// The 8 partial dot products a lane holds per row are summed over the 16 lanes
// of a half by exchanging halves of the set (8 shuffles, not 32), which leaves
// one score per lane pair; each probability then goes back to the lanes of its
// half by one shuffle per position. The warps' (max, sum, output) are joined
// in shared memory.
constexpr int kFewThreads = 256, kFewWarps = kFewThreads / 32;
constexpr unsigned kAll = 0xffffffffu;
// Weights are 2^(s - max) times this, so that the sum of as many of them as there are
// positions (2^30) times any finite value stays finite.
constexpr float kWeight = 0x1p-30f;

template <bool BF16>
__device__ __forceinline__ float4 load4(const void* base, size_t at) {
    if constexpr (BF16) {
        const uint2 u = __ldg(reinterpret_cast<const uint2*>(static_cast<const __nv_bfloat16*>(base) + at));
        return make_float4(__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xffff0000u), __uint_as_float(u.y << 16),
                           __uint_as_float(u.y & 0xffff0000u));
    } else {
        return __ldg(reinterpret_cast<const float4*>(static_cast<const float*>(base) + at));
    }
}

struct FewSmem {
    float m[kFewWarps][kFewRows], l[kFewWarps][kFewRows];
    float o[kFewWarps][kFewRows][kHeadDim];
};

// Every `stride`-th page of [p0 + warp, p1) of sequence s for its rows (R, of
// which q.rows are real) of K/V head g; leaves each warp's partial in `sm`.
template <int R, bool BF16>
__device__ __forceinline__ void few_rows(const PagedAttnArgs& a, const SeqShape& q, int s, int g, int p0, int p1,
                                         int stride, FewSmem* sm) {
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5, half = lane >> 4, dl = lane & 15;
    float qv[R][4], o[R][4], m[R], l[R];
    int last[R];                       // the last position each row sees
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int i = min(r, q.rows - 1), tok = i / a.group;
        last[r] = q.ctx + tok;
        const float4 x = __ldg(reinterpret_cast<const float4*>(a.q + (size_t)(q.row0 + tok) * a.ldq +
                                                               (g * a.group + i % a.group) * kHeadDim + 4 * dl));
        qv[r][0] = x.x * a.scale2; qv[r][1] = x.y * a.scale2; qv[r][2] = x.z * a.scale2; qv[r][3] = x.w * a.scale2;
        o[r][0] = o[r][1] = o[r][2] = o[r][3] = 0.f;
        m[r] = -INFINITY;
        l[r] = 0.f;
    }
    const size_t w = (size_t)a.n_kv_head * kHeadDim;
    const int32_t* table = a.table + (size_t)s * a.width;
    const int own = 2 * ((dl >> 3 & 1) * 4 + (dl >> 2 & 1) * 2 + (dl >> 1 & 1)) + half;   // this lane's position of a page
    int page = p0 + warp < p1 ? __ldg(table + p0 + warp) : -1;
    for (int p = p0 + warp; p < p1; p += stride) {
        const int cur = page;
        if (p + stride < p1) page = __ldg(table + p + stride);
        if (cur < 0 || cur >= a.n_pages) continue;         // an unmapped page holds no positions
        const size_t at = ((size_t)cur * kPageRows + half) * w + g * kHeadDim + 4 * dl;
        float4 kk[8], vv[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) kk[i] = load4<BF16>(a.k, at + 2 * i * w);
#pragma unroll
        for (int i = 0; i < 8; ++i) vv[i] = load4<BF16>(a.v, at + 2 * i * w);
        const int pos0 = p * kPageRows;
        const bool whole = pos0 + kPageRows - 1 <= last[0];   // rows are in token order: last[0] is the least
#pragma unroll
        for (int r = 0; r < R; ++r) {
            float d[8];
#pragma unroll
            for (int i = 0; i < 8; ++i)
                d[i] = fmaf(kk[i].w, qv[r][3], fmaf(kk[i].z, qv[r][2], fmaf(kk[i].y, qv[r][1], kk[i].x * qv[r][0])));
            const bool b3 = dl & 8, b2 = dl & 4, b1 = dl & 2;
#pragma unroll
            for (int i = 0; i < 4; ++i)
                d[i] = (b3 ? d[i + 4] : d[i]) + __shfl_xor_sync(kAll, b3 ? d[i] : d[i + 4], 8);
#pragma unroll
            for (int i = 0; i < 2; ++i)
                d[i] = (b2 ? d[i + 2] : d[i]) + __shfl_xor_sync(kAll, b2 ? d[i] : d[i + 2], 4);
            float sc = (b1 ? d[1] : d[0]) + __shfl_xor_sync(kAll, b1 ? d[0] : d[1], 2);
            sc += __shfl_xor_sync(kAll, sc, 1);
            if (!whole && pos0 + own > last[r]) sc = -INFINITY;
            float mx = sc;
#pragma unroll
            for (int x = 2; x < 32; x <<= 1) mx = fmaxf(mx, __shfl_xor_sync(kAll, mx, x));
            const float m_new = fmaxf(m[r], mx), base = m_new == -INFINITY ? 0.f : m_new;
            const float alpha = ex2_ftz(m[r] - base), pr = kWeight * ex2_ftz(sc - base);
            m[r] = m_new;
            l[r] = fmaf(l[r], alpha, pr);                  // two lanes hold each position: halved at the end
#pragma unroll
            for (int c = 0; c < 4; ++c) o[r][c] *= alpha;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float pi = __shfl_sync(kAll, pr, (lane & 16) | (i << 1));
                // a position the row does not see may hold anything: its value is not multiplied
                if (whole || pos0 + 2 * i + half <= last[r]) {
                    o[r][0] = fmaf(pi, vv[i].x, o[r][0]);
                    o[r][1] = fmaf(pi, vv[i].y, o[r][1]);
                    o[r][2] = fmaf(pi, vv[i].z, o[r][2]);
                    o[r][3] = fmaf(pi, vv[i].w, o[r][3]);
                }
            }
        }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
#pragma unroll
        for (int x = 1; x < 32; x <<= 1) l[r] += __shfl_xor_sync(kAll, l[r], x);
#pragma unroll
        for (int c = 0; c < 4; ++c) o[r][c] += __shfl_xor_sync(kAll, o[r][c], 16);
        if (r < q.rows) {
            if (lane == 0) { sm->m[warp][r] = m[r]; sm->l[warp][r] = 0.5f * l[r]; }
            if (half == 0)
                *reinterpret_cast<float4*>(&sm->o[warp][r][4 * dl]) = make_float4(o[r][0], o[r][1], o[r][2], o[r][3]);
        }
    }
}

// the same for as many rows as there are, at most RMAX
template <int RMAX, bool BF16>
__device__ __forceinline__ void few_rows_n(const PagedAttnArgs& a, const SeqShape& q, int s, int g, int p0, int p1,
                                           int stride, FewSmem* sm) {
    if (RMAX == 1 || q.rows == 1) few_rows<1, BF16>(a, q, s, g, p0, p1, stride, sm);
    else if (RMAX == 2 || q.rows == 2) few_rows<(RMAX < 2 ? RMAX : 2), BF16>(a, q, s, g, p0, p1, stride, sm);
    else if (RMAX == 4 || q.rows <= 4) few_rows<(RMAX < 4 ? RMAX : 4), BF16>(a, q, s, g, p0, p1, stride, sm);
    else few_rows<RMAX, BF16>(a, q, s, g, p0, p1, stride, sm);
}

// Row r, dim d of the warps' partials joined. (Here and in the other joins a partial that
// has seen no key is all zeros, and one whose factor is zero is still multiplied: a value
// that is not finite stays so, as it does within a warp.)
struct Joined {
    float m, l, o;
};
__device__ __forceinline__ Joined join_warps(const FewSmem& sm, int r, int d) {
    Joined j{sm.m[0][r], 0.f, 0.f};
#pragma unroll
    for (int w = 1; w < kFewWarps; ++w) j.m = fmaxf(j.m, sm.m[w][r]);
    const float base = j.m == -INFINITY ? 0.f : j.m;
#pragma unroll
    for (int w = 0; w < kFewWarps; ++w) {
        const float f = ex2_ftz(sm.m[w][r] - base);
        j.l = fmaf(sm.l[w][r], f, j.l);
        j.o = fmaf(sm.o[w][r][d], f, j.o);
    }
    return j;
}

// Every sequence of the batch has few rows: a cluster of CTAs per (sequence,
// K/V head), no schedule, no partials in memory and no second launch. The CTAs
// take the sequence's pages 8 by 8 in turn and join through each other's shared
// memory. The hardware hands the clusters out as SMs come free, which balances
// ragged batches better than equal shares: 256 sequences of up to 1000 positions,
// 12 heads, fp32 take 127 us (6.2 TB/s, 95 % of the measured copy rate) against
// 144 us with few_rows_kernel (cluster_ctas has the choice between them).
template <int RMAX, bool BF16>
__global__ void __launch_bounds__(kFewThreads, RMAX <= 2 ? 2 : 1) few_cluster_kernel(PagedAttnArgs a, int ctas) {
    __shared__ __align__(16) FewSmem sm;
    __shared__ float c_m[kFewRows], c_l[kFewRows], c_o[kFewRows][kHeadDim];
    cg::cluster_group cluster = cg::this_cluster();
    const int unit = blockIdx.x / ctas, rank = blockIdx.x % ctas, t = threadIdx.x;
    const int g = unit % a.n_kv_head, s = unit / a.n_kv_head;
    const SeqShape q = seq_shape(a, s);
    if (!q.rows) return;               // the whole cluster
    few_rows_n<RMAX, BF16>(a, q, s, g, rank * kFewWarps, pages_of(q), ctas * kFewWarps, &sm);
    __syncthreads();
    auto out_at = [&](int r, int d) -> float& {
        return a.out[(size_t)(q.row0 + r / a.group) * a.ldo + (g * a.group + r % a.group) * kHeadDim + d];
    };
    for (int e = t; e < q.rows * kHeadDim; e += kFewThreads) {
        const int r = e / kHeadDim, d = e % kHeadDim;
        const Joined j = join_warps(sm, r, d);
        if (ctas == 1) {
            out_at(r, d) = j.l == 0.f ? 0.f : j.o / j.l;
        } else {
            c_o[r][d] = j.o;
            if (d == 0) { c_m[r] = j.m; c_l[r] = j.l; }
        }
    }
    if (ctas == 1) return;
    cluster.sync();
    for (int e = rank * kFewThreads + t; e < q.rows * kHeadDim; e += ctas * kFewThreads) {
        const int r = e / kHeadDim, d = e % kHeadDim;
        float mx = -INFINITY;
        for (int c = 0; c < ctas; ++c) mx = fmaxf(mx, *cluster.map_shared_rank(&c_m[r], c));
        const float base = mx == -INFINITY ? 0.f : mx;
        float l = 0.f, o = 0.f;
        for (int c = 0; c < ctas; ++c) {
            const float f = ex2_ftz(*cluster.map_shared_rank(&c_m[r], c) - base);
            l = fmaf(*cluster.map_shared_rank(&c_l[r], c), f, l);
            o = fmaf(*cluster.map_shared_rank(&c_o[r][d], c), f, o);
        }
        out_at(r, d) = l == 0.f ? 0.f : o / l;
    }
    cluster.sync();                    // the others have read this CTA's shared memory
}

template <int RMAX, bool BF16>
__global__ void __launch_bounds__(kFewThreads, RMAX <= 2 ? 2 : 1) few_rows_kernel(PagedAttnArgs a) {
    pdl_trigger();
    extern __shared__ int s_sched[];
    __shared__ ScheduleScratch<kFewThreads> scratch;
    __shared__ __align__(16) FewSmem sm;
    const int t = threadIdx.x;
    Schedule sch;
    build_schedule<kFewThreads>(a, s_sched, &scratch, t, &sch);
    const int units = sch.unit[a.n_seq];
    if (blockIdx.x == 0 && t == 0) *a.n_records = sch.part[a.n_seq];
    for (int u = blockIdx.x; u < units; u += gridDim.x) {
        const int s = owner_of<int>(sch.unit, a.n_seq, u);
        const SeqShape q = seq_shape(a, s);
        const int sp = splits_of(q, sch.chunk), in = u - sch.unit[s], g = in % a.n_kv_head, split = in / a.n_kv_head;
        const int p0 = split * sch.chunk, p1 = min(p0 + sch.chunk, pages_of(q));
        few_rows_n<RMAX, BF16>(a, q, s, g, p0, p1, kFewWarps, &sm);
        if (sp > 1 && t == 0) a.record[0][sch.part[s] + in] = JoinRecord{split ? 0 : sp, q.rows, q.row0, 0, g, {0, 0, 0}};
        __syncthreads();
        for (int e = t; e < q.rows * kHeadDim; e += kFewThreads) {
            const int r = e / kHeadDim, d = e % kHeadDim;
            const auto [mx, l, o] = join_warps(sm, r, d);
            if (sp == 1) {
                a.out[(size_t)(q.row0 + r / a.group) * a.ldo + (g * a.group + r % a.group) * kHeadDim + d] =
                    l == 0.f ? 0.f : o / l;
            } else {
                const size_t pu = (size_t)(sch.part[s] + in) * kFewRows + r;
                a.part_o[0][pu * kHeadDim + d] = o;
                if (d == 0) { a.part_ml[0][2 * pu] = mx; a.part_ml[0][2 * pu + 1] = l; }
            }
        }
        __syncthreads();
    }
    // (nothing above needs the tensor-core kernel's results, but what waits for this
    // kernel waits for both)
    pdl_wait();
}

// ------------------------------------------------------------------ the join --
// A warp per (row, head) of what was cut adds its parts in order, lane l dims
// 2 l and 2 l + 1. Part k's row lies at row_at(k) of the kind's partials.
constexpr int kJoinThreads = 256, kJoinRows = 32;

// kAhead parts are on their way at a time: a tile is cut into two or three, one long
// sequence into hundreds.
template <int kAhead, typename RowAt>
__device__ __forceinline__ void join_row(const PagedAttnArgs& a, int kind, int parts, const RowAt& row_at, int lane,
                                         float* out) {
    float2 ml[kAhead], v[kAhead];
    auto ask = [&](int k0) {
#pragma unroll
        for (int u = 0; u < kAhead; ++u)
            if (u == 0 || k0 + u < parts) {
                const size_t at = row_at(k0 + u);
                ml[u] = *reinterpret_cast<const float2*>(a.part_ml[kind] + 2 * at);
                v[u] = *reinterpret_cast<const float2*>(a.part_o[kind] + at * kHeadDim + 2 * lane);
            }
    };
    float mx = lane < parts ? a.part_ml[kind][2 * row_at(lane)] : -INFINITY;
    ask(0);
    for (int k = lane + 32; k < parts; k += 32) mx = fmaxf(mx, a.part_ml[kind][2 * row_at(k)]);
#pragma unroll
    for (int o = 16; o; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(kAll, mx, o));
    const float base = mx == -INFINITY ? 0.f : mx;
    float l = 0.f, ox = 0.f, oy = 0.f;
    for (int k0 = 0; k0 < parts; k0 += kAhead) {
        if (k0) ask(k0);
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            if (k0 + u >= parts) break;
            const float f = ex2_ftz(ml[u].x - base);
            l = f > 0.f ? fmaf(ml[u].y, f, l) : l + weigh(ml[u].y, ml[u].x - base);
            ox = fmaf(v[u].x, f, ox);
            oy = fmaf(v[u].y, f, oy);
        }
    }
    *reinterpret_cast<float2*>(out + 2 * lane) = l == 0.f ? make_float2(0.f, 0.f) : make_float2(ox / l, oy / l);
}

// The kernels that cut left records of what is to be joined, so that nothing of the
// schedule is built again (with it: 27 us after 48 mixed sequences).
__global__ void __launch_bounds__(kJoinThreads, 4) join_kernel(PagedAttnArgs a) {
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
    pdl_wait();
    auto out_of = [&](const JoinRecord& rec, int r) {
        const int i = rec.i0 + r, token = i / a.group;
        return a.out + (size_t)(rec.token0 + token) * a.ldo + (rec.g * a.group + i - token * a.group) * kHeadDim;
    };
    // tensor-core tiles
    if (!a.only_few)
        for (int x = blockIdx.x; x < a.ctas * (kTileRows / kJoinRows); x += gridDim.x) {
            const int c = x / (kTileRows / kJoinRows), r0 = x % (kTileRows / kJoinRows) * kJoinRows;
            const JoinRecord rec = a.record[1][c];
            if (!rec.parts) continue;
            for (int r = r0 + warp; r < min(r0 + kJoinRows, rec.n_rows); r += kJoinThreads / 32)
                join_row<4>(a, 1, rec.parts, [&](int k) { return ((size_t)2 * (c + k) + (k == 0)) * kTileRows + r; }, lane,
                         out_of(rec, r));
        }
    // streaming units: a sequence's come in groups of `parts` per head
    static_assert(kJoinThreads / 32 == kFewRows, "a warp for each row of a unit");
    if (a.group <= kFewRows) {
        const int n = *a.n_records;
        for (int u = blockIdx.x; u < n; u += gridDim.x) {
            const JoinRecord rec = a.record[0][u];
            if (warp < (rec.parts ? rec.n_rows : 0))
                join_row<8>(a, 0, rec.parts, [&](int k) { return (size_t)(u + k * a.n_kv_head) * kFewRows + warp; }, lane,
                         out_of(rec, warp));
        }
    }
}

// CTAs per (sequence, K/V head) of few_cluster_kernel: as many as fit about four
// per SM, at most a portable cluster; 0 for few_rows_kernel, which shares the
// keys out evenly over all SMs and joins with a second kernel. The tables' width
// bounds the contexts; a warp of the cluster has width / (8 x CTAs) pages at
// most. On the GPU alone, bf16 (cluster / shared out, us):
//   1 sequence, 1 head     1000 positions 4.1 / 9.3, 4000 6.5 / 9.5, 8000 (7.8 pages a
//                          warp) 9.4 / 9.5, 16,000 15.4 / 10.9, 32,000 26.4 / 14.7
//   1 sequence, 12 heads   8000 10.0 / 11.8, 16,000 (15.6) 15.8 / 17.0, 32,000 38.1 / 28.1
//   16 sequences, 12 heads 1000 13.6 / 15.8, 4000 52.1 / 59.6, 16,000 (125) 174.6 / 188.9
// so 8 pages a warp where the clusters take less than half of the SMs, 16 up to two a SM,
// and 64 where they fill the GPU: up to where one long sequence among short ones would be
// left to a single cluster. The same rule was measured for fp32 and for 4 and 8 rows, whose
// CTAs an SM holds one of (cluster / shared out, a call after a flush of the caches, about 6 us
// of it the call's own; fp32, bf16 within 10 % but for the last line):
//   1 sequence, 1 head     8 rows: 4000 20 / 22, 8000 31 / 25, 16,000 49 / 27; 1 row: 8000 16 / 16
//   1 sequence, 12 heads   8 rows: 8000 33 / 43, 16,000 55 / 61, 32,000 94 / 96; 1 row: 16,000 35 / 37
//   16 sequences, 12 heads 8 rows: 4000 145 / 197, 16,000 488 / 641; 1 row: 4000 88 / 92 (bf16 68 / 72)
int cluster_ctas(int n_seq, int n_kv_head, int pages_per_seq, int sms) {
    const long long units = (long long)n_seq * n_kv_head;
    int ctas = 1;
    while (ctas < 8 && 2 * ctas * units <= 4LL * sms && ctas * kFewWarps < pages_per_seq) ctas *= 2;
    const int a_warp = units * ctas >= 2LL * sms ? 64 : 2 * units * ctas >= sms ? 16 : 8;
    return pages_per_seq <= a_warp * kFewWarps * ctas ? ctas : 0;
}

cudaError_t launch_few_cluster(const PagedAttnArgs& a, bool bf16, int rows, int ctas, cudaStream_t st) {
    void (*kernel)(PagedAttnArgs, int) = nullptr;
    if (bf16)
        kernel = rows <= 1 ? few_cluster_kernel<1, true> : rows <= 2 ? few_cluster_kernel<2, true>
                 : rows <= 4 ? few_cluster_kernel<4, true> : few_cluster_kernel<8, true>;
    else
        kernel = rows <= 1 ? few_cluster_kernel<1, false> : rows <= 2 ? few_cluster_kernel<2, false>
                 : rows <= 4 ? few_cluster_kernel<4, false> : few_cluster_kernel<8, false>;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(a.n_seq * a.n_kv_head * ctas));
    cfg.blockDim = dim3(kFewThreads);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)ctas;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, a, ctas);
}

// Streaming units aimed at when sequences are split: four per SM (two CTAs
// resident). A split sequence has more pages than a chunk, so its units number
// at most twice its pages over the chunk: all partials fit 2 x target units.
int target_of(int sms) { return 4 * sms; }

size_t part_rows(int kind, int sms) {
    return kind ? 2 * (size_t)sms * kTileRows : 2 * (size_t)target_of(sms) * kFewRows;
}
size_t run_floats(int sms) { return (size_t)sms * kTileRows * kHeadDim; }
size_t records(int kind, int sms) { return kind ? sms : 2 * (size_t)target_of(sms); }
size_t scratch_bytes(int sms) {
    return ((part_rows(0, sms) + part_rows(1, sms)) * (kHeadDim + 2) + run_floats(sms)) * sizeof(float) +
           (records(0, sms) + records(1, sms) + 1) * sizeof(JoinRecord);
}

}  // namespace
}  // namespace tie

using namespace tie;

extern "C" size_t tie_attention_paged_workspace(void) {
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) { cudaGetLastError(); return 0; }
    return scratch_bytes(sm_count(dev));
}

extern "C" model_status tie_attention_paged(const float* q, int ldq, int n_head, const void* k_pages,
                                            const void* v_pages, int kv_format, int n_pages, int n_kv_head,
                                            const int32_t* page_table, int pages_per_seq, const int32_t* row_start,
                                            const int32_t* ctx_lens, int n_seq, int max_new, int rows, float scale,
                                            float* out, int ldo, void* workspace, size_t workspace_bytes,
                                            int32_t* status, void* stream) {
    if (!k_pages || !v_pages || !page_table || !row_start || !ctx_lens || !workspace) return MODEL_ERR_ARG;
    if (rows && (!q || !out)) return MODEL_ERR_ARG;           // arrays without rows have no address
    if (!pool_shape_ok(kv_format, n_pages, n_kv_head) || n_head <= 0 || n_head % n_kv_head || n_head > 8192)
        return MODEL_ERR_ARG;
    if (pages_per_seq <= 0 || n_seq <= 0 || max_new < 0 || rows < 0 || !std::isfinite(scale)) return MODEL_ERR_ARG;
    const int w = n_head * kHeadDim;
    if (ldq < w || ldo < w || (ldq & 3) || (ldo & 3)) return MODEL_ERR_ARG;
    if (!aligned16(q) || !aligned(k_pages, 32) || !aligned(v_pages, 32) || !aligned16(out) || !aligned16(workspace))
        return MODEL_ERR_ARG;
    if (n_seq > kOpsMaxSeqs || pages_per_seq > kOpsMaxPages / 2) return MODEL_ERR_CAPACITY;
    // units are counted in int32: at most one per row and head, and one per
    // sequence and K/V head, before any split
    if ((long long)rows * n_head + (long long)n_seq * n_kv_head > INT_MAX / 2) return MODEL_ERR_CAPACITY;
    if (rows == 0 || max_new == 0) return MODEL_OK;
    OnDeviceOf dev(out);
    if (dev.status() != MODEL_OK) return dev.status();
    const int sms = sm_count(dev.device());
    if (workspace_bytes < scratch_bytes(sms)) return MODEL_ERR_CAPACITY;
    PagedAttnArgs a{};
    a.q = q; a.ldq = ldq; a.n_head = n_head;
    a.k = k_pages; a.v = v_pages;
    a.n_pages = n_pages; a.n_kv_head = n_kv_head; a.group = n_head / n_kv_head;
    a.table = page_table; a.width = pages_per_seq;
    a.row_start = row_start; a.ctx = ctx_lens;
    a.n_seq = n_seq; a.max_new = max_new; a.rows = rows;
    a.scale2 = (float)((double)scale * 1.4426950408889634);
    a.out = out; a.ldo = ldo;
    float* f = static_cast<float*>(workspace);
    a.run_o = f;
    f += run_floats(sms);
    for (int kind = 0; kind < 2; ++kind) {
        a.part_o[kind] = f;
        f += part_rows(kind, sms) * kHeadDim;
    }
    for (int kind = 0; kind < 2; ++kind) {
        a.part_ml[kind] = f;
        f += part_rows(kind, sms) * 2;
    }
    JoinRecord* rec = reinterpret_cast<JoinRecord*>(f);
    a.record[0] = rec;
    a.record[1] = rec + records(0, sms);
    a.n_records = &a.record[1][records(1, sms)].parts;
    a.target = target_of(sms);
    a.ctas = sms;
    a.status = status;
    const bool bf16 = kv_format == TIE_KV_BF16;
    const long long most = (long long)max_new * a.group;      // rows of one sequence and K/V head
    a.only_few = most <= kFewRows;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (a.only_few) {
        const int ctas = cluster_ctas(n_seq, n_kv_head, pages_per_seq, sms);
        if (ctas > 0) {
            TIE_OP_CU(launch_few_cluster(a, bf16, (int)most, ctas, st));
            ++op_launches;
            return MODEL_OK;
        }
    }
    const size_t smem = (size_t)(n_seq + 1) * sizeof(long long);
    if (!a.only_few) TIE_OP_CU(launch_paged_attn_tc(a, bf16, st));
    if (a.group <= kFewRows) {
        const int rmax = most <= 1 ? 1 : most <= 2 ? 2 : most <= 4 ? 4 : kFewRows;
        void (*kernel)(PagedAttnArgs) = nullptr;
        if (bf16)
            kernel = rmax == 1 ? few_rows_kernel<1, true> : rmax == 2 ? few_rows_kernel<2, true>
                     : rmax == 4 ? few_rows_kernel<4, true> : few_rows_kernel<8, true>;
        else
            kernel = rmax == 1 ? few_rows_kernel<1, false> : rmax == 2 ? few_rows_kernel<2, false>
                     : rmax == 4 ? few_rows_kernel<4, false> : few_rows_kernel<8, false>;
        // the prefix sums of many sequences pass the 48 KB that a kernel has unasked
        // (always the most that any call wants: calls on other threads set it too)
        if (smem + sizeof(FewSmem) > 44 * 1024)
            TIE_OP_CU(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                           (kOpsMaxSeqs + 1) * (int)sizeof(long long)));
        // beside the tensor-core kernel's last CTAs, where there is one
        const dim3 grid((unsigned)(sms * (rmax <= 2 ? 2 : 1)));
        if (a.only_few) kernel<<<grid, kFewThreads, smem, st>>>(a);
        else TIE_OP_CU(launch_pdl(kernel, grid, dim3(kFewThreads), smem, st, a));
        TIE_OP_CU(cudaGetLastError());
    }
    TIE_OP_CU(launch_pdl(join_kernel, dim3((unsigned)sms * (a.only_few ? 2 : 8)), dim3(kJoinThreads), 0, st, a));
    op_launches += 1 + !a.only_few + (a.group <= kFewRows);
    return MODEL_OK;
}
