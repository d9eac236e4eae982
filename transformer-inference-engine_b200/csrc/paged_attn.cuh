// paged_attn.cuh -- what the kernels of attention over the paged cache share:
// the arguments, the schedule that every CTA derives from the lengths on the
// device, and the partial results of sequences whose keys are split.
//
// Row (i, h) of sequence s is its new token i and query head h, at position
// ctx_s + i. The heads of one K/V head and a sequence's tokens together form
// the rows that share keys: row index i * group + (h mod group). They are cut
// into tiles, a tile's keys into splits; a unit is (sequence, tile, split, K/V
// head), the head fastest, so CTAs that run together read one page's
// neighbouring rows. Sequences of few rows (at most kFewRows) are units of the
// streaming kernel, the others of the tensor-core kernel; both kinds are
// scheduled from the same arrays, by each kernel for itself (a scan of the
// lengths costs less than a launch that would leave it in memory).
#pragma once

#include "ops.h"

namespace tie {

constexpr int kFewRows = 8;        // rows of a streaming unit
constexpr int kTileRows = 128;     // rows of a tensor-core unit
constexpr int kTileKeys = 128;     // keys of one of its steps

struct PagedAttnArgs {
    const float* q;
    int ldq, n_head;
    const void *k, *v;
    int n_pages, n_kv_head, group;
    const int32_t* table;
    int width;
    const int32_t *row_start, *ctx;
    int n_seq, max_new, rows;
    float scale2;                  // score scale * log2(e): the softmax runs in powers of two
    float* out;
    int ldo;
    // partials of split units, per kind (0 streaming, 1 tensor core)
    float* part_o[2];              // [unit][tile rows][64], unnormalised
    float* part_ml[2];             // [unit][tile rows][2]: maximum (power-of-two domain), sum
    int target[2];                 // units wanted of each kind when the work is split
    int only_few;                  // every sequence is of the streaming kind
    int* status;
};

__host__ __device__ inline int tile_rows_of(int kind) { return kind ? kTileRows : kFewRows; }
__host__ __device__ inline int step_keys_of(int kind) { return kind ? kTileKeys : kPageRows; }
// fewest steps (of step_keys_of keys) worth a unit of their own
__host__ __device__ inline int min_steps_of(int kind) { return kind ? 2 : 8; }

// One sequence as the schedule sees it; rows == 0 for one to leave alone
// (no new tokens, or lengths outside the caller's bounds).
struct SeqShape {
    int row0, ctx, tokens, rows, kind, tiles, steps;
};

__device__ __forceinline__ SeqShape seq_shape(const PagedAttnArgs& a, int s) {
    SeqShape q{};
    const int r0 = __ldg(a.row_start + s), r1 = __ldg(a.row_start + s + 1), c = __ldg(a.ctx + s);
    if (r0 < 0 || r1 <= r0 || r1 > a.rows || r1 - r0 > a.max_new || c < 0) return q;
    if ((long long)c + (r1 - r0) > (long long)a.width * kPageRows) return q;
    q.row0 = r0;
    q.ctx = c;
    q.tokens = r1 - r0;
    q.rows = q.tokens * a.group;
    q.kind = !a.only_few && q.rows > kFewRows;
    q.tiles = (q.rows + tile_rows_of(q.kind) - 1) / tile_rows_of(q.kind);
    q.steps = (c + q.tokens + step_keys_of(q.kind) - 1) / step_keys_of(q.kind);
    return q;
}

// The schedule of one kind in shared memory: prefix sums over the sequences of
// the units, and of the units that leave partials.
struct Schedule {
    int* unit;                     // [n_seq + 1]
    int* part;                     // [n_seq + 1]
    int chunk;                     // steps per split
};

template <int THREADS>
struct ScheduleScratch {
    long long total[THREADS / 32];
    int a[THREADS / 32], b[THREADS / 32];
};

// Splits of a sequence at `chunk` steps per split.
__device__ __forceinline__ int splits_of(const SeqShape& q, int chunk) { return (q.steps + chunk - 1) / chunk; }

// Builds the schedule of `kind` with all THREADS threads of the CTA (thread t
// of them); ends with a barrier.
template <int THREADS>
__device__ __forceinline__ void build_schedule(const PagedAttnArgs& a, int kind, int* smem, ScheduleScratch<THREADS>* sc,
                                               int t, Schedule* out) {
    constexpr unsigned kAllLanes = 0xffffffffu;
    const int lane = t & 31, warp = t >> 5;
    const int per = (a.n_seq + THREADS - 1) / THREADS;
    out->unit = smem;
    out->part = smem + a.n_seq + 1;
    long long work = 0;
    for (int k = 0; k < per; ++k) {
        const int s = t * per + k;
        if (s >= a.n_seq) break;
        const SeqShape q = seq_shape(a, s);
        if (q.rows && q.kind == kind) work += (long long)a.n_kv_head * q.tiles * q.steps;
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) work += __shfl_xor_sync(kAllLanes, work, o);
    if (lane == 0) sc->total[warp] = work;
    __syncthreads();
    long long total = 0;
#pragma unroll
    for (int w = 0; w < THREADS / 32; ++w) total += sc->total[w];
    const long long even = (total + a.target[kind] - 1) / a.target[kind];
    out->chunk = (int)(even > min_steps_of(kind) ? even : min_steps_of(kind));
    int units = 0, parts = 0;
    for (int k = 0; k < per; ++k) {
        const int s = t * per + k;
        if (s >= a.n_seq) break;
        const SeqShape q = seq_shape(a, s);
        if (!q.rows || q.kind != kind) continue;
        const int sp = splits_of(q, out->chunk), n = a.n_kv_head * q.tiles * sp;
        units += n;
        if (sp > 1) parts += n;
    }
    int iu = units, ip = parts;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(kAllLanes, iu, o), p = __shfl_up_sync(kAllLanes, ip, o);
        if (lane >= o) { iu += u; ip += p; }
    }
    if (lane == 31) { sc->a[warp] = iu; sc->b[warp] = ip; }
    __syncthreads();
    int bu = iu - units, bp = ip - parts;
    for (int w = 0; w < warp; ++w) { bu += sc->a[w]; bp += sc->b[w]; }
    for (int k = 0; k < per; ++k) {
        const int s = t * per + k;
        if (s >= a.n_seq) break;
        out->unit[s] = bu;
        out->part[s] = bp;
        const SeqShape q = seq_shape(a, s);
        if (q.rows && q.kind == kind) {
            const int sp = splits_of(q, out->chunk), n = a.n_kv_head * q.tiles * sp;
            bu += n;
            if (sp > 1) bp += n;
        }
        if (s == a.n_seq - 1) { out->unit[a.n_seq] = bu; out->part[a.n_seq] = bp; }
    }
    __syncthreads();
}

// The last s < n with base[s] <= x.
__device__ __forceinline__ int owner_of(const int* base, int n, int x) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (base[mid] <= x) lo = mid;
        else hi = mid;
    }
    return lo;
}

// 2^x on the special-function unit (ex2.approx.ftz: relative error about
// 2^-22, results below 2^-126 flush to zero).
__device__ __forceinline__ float ex2_ftz(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Tensor-core kernel (k_paged_tc.cu) for the sequences of kind 1.
cudaError_t launch_paged_attn_tc(const PagedAttnArgs& a, bool bf16, int sms, cudaStream_t st);

}  // namespace tie
