// shared_attn.cuh -- what the kernels of attention over shared positions have in common: the
// arguments, and the line of work that every CTA derives from the lengths on the device.
// (ops_shared.cu has the mathematics and the plan of the whole.)
#pragma once

#include "paged_attn.cuh"
#include "quant.cuh"

namespace tie {

// Weights are 2^(s - max) times this, so that the sum of as many of them as there are
// positions (2^30) times any finite value stays finite.
constexpr float kWeight = 0x1p-30f;
// Fewest pages worth a warp's stretch: two steps over fp32 pages (16 keys), one over others (32). With one
// and with two steps, us: one sequence of 1000, fp32, 11.6 and 10.8; 16 sequences behind 700, fp32, 14.1 and
// 14.1, 8 bits 12.2 and 13.7; 32 behind 700, bf16, 13.8 and 14.8. (Three: 1 to 2 more than two.)
constexpr int kMinPages = 2;

// A line: units [u0, u1) (a unit below n_group is a group's prefix, the others are
// sequences), cut into stretches for `teams` teams: of a warp per K/V head (heads 1), or
// CTAs, to which an item's K/V heads are items side by side (heads: as many).
struct Line {
    int u0, u1, nt, pages, teams;      // nt: an item has 8 nt rows; pages: of a step
    int heads, per;                    // per: rows of a part
    float* part_o;                     // [2 * warps or CTAs][per][64]: its parts of the item it goes on with
    float* part_ml;                    // and of the one that it begins; (maximum, sum)
};

struct SharedArgs {
    const float* q;
    int ldq, n_head, group, n_kv_head;
    Divisor by_group;
    const void *k, *v;
    const float *ks, *vs;
    int n_pages;
    const int32_t* table;
    int width;
    const int32_t *row_start, *ctx;
    int n_seq, max_new, rows;
    const int32_t* ptable;
    int pwidth;
    const int32_t *plen, *gstart;
    int n_group;
    float scale2;                      // score scale * log2(e): the softmax runs in powers of two
    float* out;
    int ldo;
    float* whole_o[2];                 // [prefix, own][row][head][64]: items that no stretch cuts
    float* whole_ml[2];                // (only where rows have two sources)
    int2* place[2];                    // [prefix, own][row][head]: the row of its first part in the line's parts,
                                       // or -1: whole; how many parts
    Line line[2];                      // for prefixes and for sequences; one line, or one each
    int* status;
    uint32_t wait_ns;                  // how long k_shared_tc.cu waits for anything; stall: every other CTA of it
    int stall;                         // waits for what does not come
};

// What a unit's rows are, and its keys. rows == 0: nothing to do.
struct UnitShape {
    int row0, tokens, rows, keys;      // keys: positions in its pages
    int ctx;                           // own: row i sees positions <= ctx + i / group; prefix: all
};

// The lengths: the caller's arrays, or a CTA's copy of them in shared memory.
struct Lengths {
    const int32_t *row_start, *ctx, *gstart, *plen;
};

__device__ __forceinline__ UnitShape unit_shape(const SharedArgs& a, const Lengths& n, int u) {
    UnitShape s{};
    if (u < a.n_group) {
        const int s0 = n.gstart[u], s1 = n.gstart[u + 1], keys = n.plen[u];
        if (s0 < 0 || s1 <= s0 || s1 > a.n_seq || keys <= 0 || keys > (long long)a.pwidth * kPageRows) return s;
        const int r0 = n.row_start[s0], r1 = n.row_start[s1];
        if (r0 < 0 || r1 <= r0 || r1 > a.rows) return s;
        s.row0 = r0;
        s.tokens = r1 - r0;
        s.keys = keys;
        s.ctx = keys;
    } else {
        const int q = u - a.n_group;
        const int r0 = n.row_start[q], r1 = n.row_start[q + 1], c = n.ctx[q];
        if (r0 < 0 || r1 <= r0 || r1 > a.rows || r1 - r0 > a.max_new || c < 0) return s;
        if ((long long)c + (r1 - r0) > (long long)a.width * kPageRows) return s;
        s.row0 = r0;
        s.tokens = r1 - r0;
        s.keys = c + s.tokens;
        s.ctx = c;
    }
    s.rows = s.tokens * a.group;
    return s;
}
// places of one of its items, and its items
__device__ __forceinline__ int unit_places(const UnitShape& s, const Line& l) {
    const int step = l.pages * kPageRows;
    return (s.keys - 1) / step + 2;
}
__device__ __forceinline__ long long unit_items(const UnitShape& s, const Line& l) {
    return (long long)((s.rows + 8 * l.nt - 1) / (8 * l.nt)) * l.heads;
}

// x / y of numbers that are nearly always small (a division of 64 bits is a hundred instructions)
__device__ __forceinline__ long long quotient(long long x, long long y) {
    return ((x | y) >> 32) == 0 ? (long long)((unsigned)x / (unsigned)y) : x / y;
}

__device__ __forceinline__ long long share_of(const Line& l, long long total) {
    const long long even = quotient(total + l.teams - 1, l.teams);
    const int least = l.pages < kMinPages ? kMinPages / l.pages : 1;
    return even > least ? even : least;
}

// A CTA's copy of the lengths and the line in shared memory: base[u - u0] places before unit u, all
// of them in base[u1 - u0]. (Copied at once: looked up one after another, again for each
// item, they took a kernel 2 to 3 us more to start.) Ends with a barrier.
struct Plan {
    Lengths n;
    long long* base;
};
inline size_t plan_bytes(int units, int n_seq, int n_group) {
    return (size_t)(units + 1) * sizeof(long long) + (size_t)(2 * n_seq + 2 * n_group + 2) * sizeof(int32_t);
}
template <int THREADS>
__device__ __forceinline__ Plan build_plan(const SharedArgs& a, int u0, int u1, void* smem, ScheduleScratch<THREADS>* sc, int t) {
    const int n = u1 - u0, per = (n + THREADS - 1) / THREADS;
    long long* base = static_cast<long long*>(smem);
    int32_t* const start = reinterpret_cast<int32_t*>(base + n + 1);
    int32_t* const ctx = start + a.n_seq + 1;
    int32_t* const gstart = ctx + a.n_seq;
    int32_t* const plen = gstart + a.n_group + 1;
    for (int i = t; i <= a.n_seq; i += THREADS) {
        start[i] = __ldg(a.row_start + i);
        if (i < a.n_seq) ctx[i] = __ldg(a.ctx + i);
    }
    if (a.n_group)
        for (int i = t; i <= a.n_group; i += THREADS) {
            gstart[i] = __ldg(a.gstart + i);
            if (i < a.n_group) plen[i] = __ldg(a.plen + i);
        }
    __syncthreads();
    const Plan plan{Lengths{start, ctx, gstart, plen}, base};
    auto places_of = [&](int u) -> long long {
        const UnitShape s = unit_shape(a, plan.n, u);
        const Line& l = a.line[u >= a.n_group];
        return s.rows ? unit_items(s, l) * unit_places(s, l) : 0;
    };
    long long mine = 0, before;
    for (int i = 0; i < per; ++i) {
        const int u = u0 + t * per + i;
        if (u < u1) mine += places_of(u);
    }
    const long long total = scan_threads<THREADS>(mine, sc, t, &before);
    for (int i = 0; i < per; ++i) {
        const int u = u0 + t * per + i;
        if (u >= u1) break;
        base[u - u0] = before;
        if (per > 1) before += places_of(u);       // a thread's only unit needs no second look
    }
    if (t == 0) base[n] = total;
    __syncthreads();
    return plan;
}

// Terms of two numbers: [0] the largest.
__device__ __forceinline__ void split3(float lo, float hi, uint32_t (&x)[3]) {
    x[0] = terms2(lo, hi);
    rest2(lo, hi);
    x[1] = terms2(lo, hi);
    rest2(lo, hi);
    x[2] = terms2(lo, hi);
}

// Tensor-core kernel (k_shared_tc.cu) for prefixes of many rows: items of 128 rows, steps of 64 keys.
constexpr int kTcRows = 128, kTcPages = 4;
int shared_tc_ctas(int sms);
cudaError_t launch_shared_tc(const SharedArgs& a, int format, cudaStream_t st);

}  // namespace tie
