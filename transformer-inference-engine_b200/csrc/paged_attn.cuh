// paged_attn.cuh -- what the kernels of attention over the paged cache share:
// the arguments, the schedule that every CTA derives from the lengths on the
// device, and the partial results of sequences whose keys are split.
//
// Row (i, h) of sequence s is its new token i and query head h, at position
// ctx_s + i. The heads of one K/V head and a sequence's tokens together form
// the rows that share keys: row index i * group + (h mod group). Sequences of
// few rows (at most kFewRows) go to the streaming kernel, the others to the
// tensor-core kernel; each kernel derives its schedule from the lengths for
// itself (a scan of the lengths costs less than a launch that would leave it in
// memory).
//   Streaming (kind 0): a unit is (sequence, split of the keys, K/V head), the
// head fastest, so CTAs that run together read one page's neighbouring rows.
//   Tensor cores (kind 1): the rows are cut into tiles, whose steps over the keys
// count as jobs (two a step when the tile has more than 128 rows). All tiles of the
// batch stand in one line -- by sequence, tile, K/V head -- each with its jobs behind
// a few places that stand for what a tile costs besides; every CTA takes an equal
// stretch of the line. A tile that a stretch cuts leaves partial results.
#pragma once

#include "ops.h"

namespace tie {

// Rows of a streaming unit at most. Streaming and tensor cores, each for all rows, 8 K/V heads
// (us, a call after a flush of the caches, about 6 of them the call's own; fp32, bf16 in brackets):
//   1 sequence, 1000 cached:   1 row 10 and 43 (10, 37), 8 rows 14 and 43 (14, 39),
//                              16 rows 31 and 45 (32, 39), 48 rows 33 and 47 (37, 41)
//   8 sequences, 1000 cached:  8 rows 49 and 53 (49, 45), 12 rows 45 and 57 (47, 47), 24 rows 66 and 57 (64, 47)
//   64 sequences, 4000 cached: 1 row 174 and 520 (117, 360), 4 rows 240 and 522 (234, 362),
//                              8 rows 334 and 522 (336, 364), 12 rows 522 and 526 (494, 371)
// So the rule holds where there are many sequences; one alone would stream up to 48 rows.
constexpr int kFewRows = 8;
constexpr int kHalfRows = 128;     // rows of one MMA of the tensor-core kernel
constexpr int kTileRows = 256;     // rows of its tiles
constexpr int kTileKeys = 128;     // keys of one of its steps

// What the join has to know of a cut tile: its first part lies where the record does.
struct __align__(16) JoinRecord {
    int parts, n_rows;             // parts 0: nothing to join here
    int token0, i0, g;             // the sequence's first row of out, the tile's first row, K/V head
    int pad[3];
};

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
    // partials, per kind: of split units (streaming), two per CTA (tensor cores)
    float* part_o[2];              // [unit][tile rows][64], unnormalised
    float* part_ml[2];             // [unit][tile rows][2]: maximum (power-of-two domain), sum
    float* run_o;                  // [CTA][stream][64 / 4][128 rows][4]: running sums (tensor cores)
    JoinRecord* record[2];         // [unit with partials], [CTA]: written by the kernels that cut
    int* n_records;                // streaming units with partials
    int target;                    // streaming units wanted when the work is split
    int ctas;                      // CTAs of the tensor-core kernel
    int only_few;                  // every sequence is of the streaming kind
    int* status;
};

// fewest pages worth a streaming unit of their own (four for each warp), fewest
// jobs worth a tensor-core CTA
constexpr int kMinUnitPages = 32, kMinJobs = 2;

// One sequence as the schedule sees it; rows == 0 for one to leave alone
// (no new tokens, or lengths outside the caller's bounds).
struct SeqShape {
    int row0, ctx, tokens, rows, kind, tiles;
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
    q.tiles = (q.rows + kTileRows - 1) / kTileRows;
    return q;
}

template <int THREADS>
struct ScheduleScratch {
    long long total[THREADS / 32];
    int a[THREADS / 32], b[THREADS / 32];
};

// Sum over the CTA's threads of `v`, and in *before the sum over lower threads.
template <int THREADS>
__device__ __forceinline__ long long scan_threads(long long v, ScheduleScratch<THREADS>* sc, int t, long long* before) {
    const int lane = t & 31, warp = t >> 5;
    long long in = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long u = __shfl_up_sync(0xffffffffu, in, o);
        if (lane >= o) in += u;
    }
    __syncthreads();
    if (lane == 31) sc->total[warp] = in;
    __syncthreads();
    long long all = 0, low = 0;
#pragma unroll
    for (int w = 0; w < THREADS / 32; ++w) {
        if (w < warp) low += sc->total[w];
        all += sc->total[w];
    }
    *before = low + in - v;
    return all;
}

// ----------------------------------------------------------- streaming units --
// Prefix sums over the sequences of the units, and of the units that leave
// partials, in shared memory.
struct Schedule {
    int* unit;                     // [n_seq + 1]
    int* part;                     // [n_seq + 1]
    int chunk;                     // pages per split
};

__device__ __forceinline__ int pages_of(const SeqShape& q) { return (q.ctx + q.tokens + kPageRows - 1) / kPageRows; }
__device__ __forceinline__ int splits_of(const SeqShape& q, int chunk) { return (pages_of(q) + chunk - 1) / chunk; }

// Built with all THREADS threads of the CTA (thread t of them); ends with a
// barrier.
template <int THREADS>
__device__ __forceinline__ void build_schedule(const PagedAttnArgs& a, int* smem, ScheduleScratch<THREADS>* sc, int t,
                                               Schedule* out) {
    const int per = (a.n_seq + THREADS - 1) / THREADS;
    out->unit = smem;
    out->part = smem + a.n_seq + 1;
    long long work = 0, before;
    for (int k = 0; k < per; ++k) {
        const int s = t * per + k;
        if (s >= a.n_seq) break;
        const SeqShape q = seq_shape(a, s);
        if (q.rows && !q.kind) work += (long long)a.n_kv_head * pages_of(q);
    }
    const long long even = (scan_threads<THREADS>(work, sc, t, &before) + a.target - 1) / a.target;
    // (no sequence has as many pages as the pool can have)
    out->chunk = (int)(even < kMinUnitPages ? kMinUnitPages : even < kOpsMaxPages ? even : kOpsMaxPages);
    long long units = 0;           // units in the low half, units with partials in the high half
    for (int k = 0; k < per; ++k) {
        const int s = t * per + k;
        if (s >= a.n_seq) break;
        const SeqShape q = seq_shape(a, s);
        if (!q.rows || q.kind) continue;
        const int sp = splits_of(q, out->chunk);
        const long long n = (long long)a.n_kv_head * sp;
        units += n + (sp > 1 ? n << 32 : 0);
    }
    scan_threads<THREADS>(units, sc, t, &before);
    int bu = (int)before, bp = (int)(before >> 32);
    for (int k = 0; k < per; ++k) {
        const int s = t * per + k;
        if (s >= a.n_seq) break;
        out->unit[s] = bu;
        out->part[s] = bp;
        const SeqShape q = seq_shape(a, s);
        if (q.rows && !q.kind) {
            const int sp = splits_of(q, out->chunk), n = a.n_kv_head * sp;
            bu += n;
            if (sp > 1) bp += n;
        }
        if (s == a.n_seq - 1) { out->unit[a.n_seq] = bu; out->part[a.n_seq] = bp; }
    }
    __syncthreads();
}

// ----------------------------------------------------------- tensor-core jobs --
// The line: base[s] places before sequence s, all of them in base[n_seq]; CTA c
// has places [c * share, (c + 1) * share).
struct JobLine {
    long long* base;               // [n_seq + 1], shared memory
    long long share;
};

// places before a tile's jobs: loading Q, and the results' way out (1, 2, 3, 4: 48 sequences of 60
// new rows behind 450, 25 heads, fp32 239, 233, 236, 232 us, bf16 190, 184, 186, 182; 8 of 256 behind
// 512, 12 heads, fp32 84, 84, 84, 88; a long chunk 860 with each)
constexpr int kTilePlaces = 2;

__device__ __forceinline__ int tile_n_rows(const SeqShape& q, int tile) { return min(kTileRows, q.rows - tile * kTileRows); }
// keys that a tile's rows see, and its steps over them
__device__ __forceinline__ int tile_keys(const PagedAttnArgs& a, const SeqShape& q, int tile) {
    return q.ctx + (tile * kTileRows + tile_n_rows(q, tile) - 1) / a.group + 1;
}
__device__ __forceinline__ int tile_steps(const PagedAttnArgs& a, const SeqShape& q, int tile) {
    return (tile_keys(a, q, tile) + kTileKeys - 1) / kTileKeys;
}
// places of a tile for one K/V head
__device__ __forceinline__ int tile_places(const PagedAttnArgs& a, const SeqShape& q, int tile) {
    return (tile_steps(a, q, tile) << (tile_n_rows(q, tile) > kHalfRows)) + kTilePlaces;
}
__device__ __forceinline__ long long seq_places(const PagedAttnArgs& a, const SeqShape& q) {
    long long n = 0;
    for (int tile = 0; tile < q.tiles; ++tile) n += tile_places(a, q, tile);
    return n * a.n_kv_head;
}

template <int THREADS>
__device__ __forceinline__ void build_line(const PagedAttnArgs& a, long long* smem, ScheduleScratch<THREADS>* sc, int t,
                                           JobLine* out) {
    const int per = (a.n_seq + THREADS - 1) / THREADS;
    out->base = smem;
    long long mine = 0, before;
    for (int k = 0; k < per; ++k) {
        const int s = t * per + k;
        if (s >= a.n_seq) break;
        const SeqShape q = seq_shape(a, s);
        if (q.rows && q.kind) mine += seq_places(a, q);
    }
    const long long total = scan_threads<THREADS>(mine, sc, t, &before);
    for (int k = 0; k < per; ++k) {
        const int s = t * per + k;
        if (s >= a.n_seq) break;
        out->base[s] = before;
        if (per > 1) {             // a thread's only sequence needs no second look
            const SeqShape q = seq_shape(a, s);
            if (q.rows && q.kind) before += seq_places(a, q);
        }
    }
    if (t == 0) out->base[a.n_seq] = total;
    const long long even = (total + a.ctas - 1) / a.ctas;
    out->share = even > kTilePlaces + kMinJobs ? even : kTilePlaces + kMinJobs;
    __syncthreads();
}

// A tile and K/V head in the line: places [first, end), its jobs from `jobs` on.
struct LineUnit {
    SeqShape q;
    int s, tile, g;
    long long first, jobs, end;
};

// The last s < n with base[s] <= x.
template <typename T>
__device__ __forceinline__ int owner_of(const T* base, int n, T x) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (base[mid] <= x) lo = mid;
        else hi = mid;
    }
    return lo;
}

// The unit that holds place x (x < all places).
__device__ __forceinline__ LineUnit unit_at(const PagedAttnArgs& a, const JobLine& line, long long x) {
    LineUnit u;
    u.s = owner_of<long long>(line.base, a.n_seq, x);
    u.q = seq_shape(a, u.s);
    long long at = line.base[u.s];
    int each;
    u.tile = 0;
    for (;;) {
        each = tile_places(a, u.q, u.tile);
        const long long n = (long long)each * a.n_kv_head;
        if (x < at + n || u.tile == u.q.tiles - 1) break;
        at += n;
        ++u.tile;
    }
    u.g = (int)((x - at) / each);
    u.first = at + (long long)u.g * each;
    u.jobs = u.first + kTilePlaces;
    u.end = u.first + each;
    return u;
}

// The unit after u: the next K/V head, tile, or sequence with rows of this kind
// (the caller knows that there is one).
__device__ __forceinline__ void unit_next(const PagedAttnArgs& a, LineUnit& u) {
    if (++u.g == a.n_kv_head) {
        u.g = 0;
        if (++u.tile == u.q.tiles) {
            u.tile = 0;
            while (++u.s < a.n_seq - 1) {
                u.q = seq_shape(a, u.s);
                if (u.q.rows && u.q.kind) break;
            }
            if (u.s == a.n_seq - 1) u.q = seq_shape(a, u.s);
        }
    }
    u.first = u.end;
    u.jobs = u.first + kTilePlaces;
    u.end = u.first + tile_places(a, u.q, u.tile);
}

// 2^x on the special-function unit (ex2.approx.ftz: relative error about
// 2^-22, results below 2^-126 flush to zero).
__device__ __forceinline__ float ex2_ftz(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// l 2^d for d <= 0. The row sum of a part of the tensor-core kernel is between 2^-106 and
// 2^126 (its maximum counts the values' exponents), so where 2^d flushes l 2^d need not.
__device__ __forceinline__ float weigh(float l, float d) {
    const float half = ex2_ftz(0.5f * d);
    return d >= -126.f ? l * ex2_ftz(d) : l * half * half;
}

// Tensor-core kernel (k_paged_tc.cu) for the sequences of kind 1.
cudaError_t launch_paged_attn_tc(const PagedAttnArgs& a, bool bf16, cudaStream_t st);

}  // namespace tie
