// ops_shared.cu -- attention of a batch's new tokens over their sequences' own pages and
// over pages that groups of sequences share (a common prompt), which are read for all of
// a group's rows together; pages in fp32, bf16 or 8 bits.
//
// The reference attends one new token of its one sequence to that sequence's cache
// (src/model.c:826-850). Here row r of sequence s, in group g, attends to
//   the group's prefix_lens[g] first positions, and its own ctx + i + 1 cached ones:
//   out = sum_j p_j v_j / sum_j p_j,   p_j = exp(scale q . k_j - m),
// with the maximum m and both sums carried along in fp32 (a softmax in one pass). What
// a warp has seen of a row's keys is (m, sum, weighted values); such parts are joined as
// one pass would have gone on: sums scaled by exp(m_part - m).
//
// Work. An item is rows that share keys (a sequence's new tokens or a group's, times the query
// heads of one K/V head; 8 to 32 rows) and all pages of those keys. All items of a call, those
// of prefixes and those of sequences, stand in one line, each as many places as it has steps, and
// one for what it costs besides. A team of as many warps as there are K/V heads, each with one
// of them, takes an equal stretch of the line, whatever the lengths are; every warp works alone
// (no barriers). Heads side by side read whole rows of a page at about one time: a warp that
// walked its head's pages by itself, head after head, got 3.3 TB/s out of 8-bit pages (64 bytes of
// a row, with nobody beside it). An item that a stretch cuts leaves parts, which a second
// kernel joins. A prefix of many rows and many scores goes to tcgen05 (k_shared_tc.cu).
//
// Products over fp32 and bf16 pages run on bf16 MMAs (m16n8k16). An fp32 number is exactly the sum
// of three bf16 terms, a bf16 number is one; products of terms below 2^-24 of the whole are
// left out (six MMAs a product over fp32 pages, three over bf16). No operand is scaled, so
// any finite value keeps its bits. Levels of 8 bits are operands of integer MMAs (run_steps_q8).
// Keys are the MMA's 16 rows, so the rows of a decode step (one for each query head of a
// K/V head, where it has no prefix) fill its 8 columns as far as they go. K and V go from memory
// into operand registers without shared memory: a lane's 16 dims of a key may be any 16 of
// the sum, so it takes 16 in a row, and each lane's 8 dims of 4 values are packed in pairs of keys.
//
// Measured (B200, whole calls): 64 sequences of up to 4000 positions, 8-bit pages (127 MB), one token
// each, 39 us: 27 of steps (4.7 TB/s; 600 instructions for 32 keys of a head), the others the start (4)
// and the join; 40 % of DRAM's rate and 47 % of issue slots over all. Steps copied to shared memory, with 16 warps an SM instead of
// 12, reads with hints for the L2 and pairs of numbers per instruction in the 8-bit path each
// took 39 too (the same 64 bytes of a row a warp, all of them: pages as a whole were not tried). 256 answers of a
// token behind 700 positions, fp32, 74 us, 42 % of DRAM's rate and 41 % of issue slots: neither is full, 12
// warps an SM with a step ahead each wait for it. (Numbers in pairs in the fp32 split: 76 -> 74.) 24 groups in
// 8 bits 55 us, 4 beams 11.4: two launches in turn.
#include <cuda_bf16.h>

#include <climits>
#include <cmath>
#include <type_traits>

#include "shared_attn.cuh"

namespace tie {
namespace {

constexpr int kThreads = 128, kWarps = kThreads / 32;
constexpr unsigned kAll = 0xffffffffu;
// Pages of a step.
template <int FMT, int NT>
constexpr int kPages = FMT == TIE_KV_F32 ? 1 : FMT == TIE_KV_BF16 ? (NT > 2 ? 1 : 2) : 2;

// CTAs on an SM
template <int FMT, int NT>
constexpr int kCtas = NT <= 2 ? 3 : 2;

// ------------------------------------------------------------------ operands --
template <int WORDS>
__device__ __forceinline__ void load_words(const void* base, size_t byte, uint32_t (&w)[WORDS]) {
    const char* p = static_cast<const char*>(base) + byte;
    if constexpr (WORDS == 2) {
        asm volatile("ld.global.nc.L1::no_allocate.v2.b32 {%0, %1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "l"(p));
    } else if constexpr (WORDS == 4) {
        asm volatile("ld.global.nc.L1::no_allocate.v4.b32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
                     : "l"(p));
    } else {
#pragma unroll
        for (int i = 0; i < WORDS / 8; ++i)
            asm volatile("ld.global.nc.L1::no_allocate.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                         : "=r"(w[8 * i]), "=r"(w[8 * i + 1]), "=r"(w[8 * i + 2]), "=r"(w[8 * i + 3]), "=r"(w[8 * i + 4]),
                           "=r"(w[8 * i + 5]), "=r"(w[8 * i + 6]), "=r"(w[8 * i + 7])
                         : "l"(p + 32 * i));
    }
}

__device__ __forceinline__ uint32_t transposed(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

// The MMA cuts its sums off, towards zero, so the products of the terms are added in two
// sets: d += the largest terms' product, and e += the others', which are 2^-8 of it (a product of
// terms below 2^-24 of the whole is left out). With all in one chain of 24 MMAs the error of the
// result was 2.0e-6 over fp32 pages (2-norm, 1000 positions), in two sets it is 4.0e-7.
// Products of terms (of A, of B) in the order they are added; the last one is the largest.
template <int NA>
struct Products {
    static constexpr int kSmall = NA == 3 ? 5 : 2;
    // 0 2, 2 0, 1 1, 1 0, 0 1, 0 0 and, of a single term, 0 2, 0 1, 0 0
    static __device__ __forceinline__ constexpr int a(int x) { return NA == 1 ? 0 : x == 1 ? 2 : x == 2 || x == 3 ? 1 : 0; }
    static __device__ __forceinline__ constexpr int b(int x) { return NA == 1 ? 2 - x : x == 0 ? 2 : x == 2 || x == 4 ? 1 : 0; }
};
// Products [FROM, TO) for R accumulators, which take turns: an MMA that waits for the one before it
// waits its whole latency.
template <bool FIRST, int FROM, int TO, int R, int NA, typename A, typename B0, typename B1>
__device__ __forceinline__ void add_products(float (&d)[R][4], const A& fa, const B0& b0, const B1& b1) {
#pragma unroll
    for (int x = FROM; x < TO; ++x)
#pragma unroll
        for (int r = 0; r < R; ++r) {
            using P = Products<NA>;
            if (FIRST && x == FROM) mma_bf16(d[r], fa(r, P::a(x)), b0(r, P::b(x)), b1(r, P::b(x)), {0.f, 0.f, 0.f, 0.f});
            else mma_bf16(d[r], fa(r, P::a(x)), b0(r, P::b(x)), b1(r, P::b(x)));
        }
}

// --------------------------------------------------------------- the products --
// What a lane loads of a page: keys g and g + 8, dims 16 c .. 16 c + 15 of each; values of
// keys 2 c, 2 c + 1, 2 c + 8, 2 c + 9, dims 8 g .. 8 g + 7 (g = lane / 4, c = lane % 4).
template <int FMT>
struct Format;
template <>
struct Format<TIE_KV_F32> {
    static constexpr int kBytes = 4, kTerms = 3;
    // the A operand of the k step s of 16 dims (of 4 c .. of each lane): keys
    static __device__ __forceinline__ void keys(const uint32_t (&k)[2][16], int s, uint32_t (&a)[3][4]) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const uint32_t* w = &k[r & 1][4 * s + 2 * (r >> 1)];
            uint32_t x[3];
            split3(__uint_as_float(w[0]), __uint_as_float(w[1]), x);
            a[0][r] = x[0];
            a[1][r] = x[1];
            a[2][r] = x[2];
        }
    }
    // the A operand of dims 8 g + 2 i and 8 g + 2 i + 1: values
    static __device__ __forceinline__ void values(const uint32_t (&v)[4][8], int i, uint32_t (&a)[3][4]) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int key = 2 * (r >> 1), d = 2 * i + (r & 1);
            uint32_t x[3];
            split3(__uint_as_float(v[key][d]), __uint_as_float(v[key + 1][d]), x);
            a[0][r] = x[0];
            a[1][r] = x[1];
            a[2][r] = x[2];
        }
    }
};
template <>
struct Format<TIE_KV_BF16> {
    static constexpr int kBytes = 2, kTerms = 1;
    static __device__ __forceinline__ void keys(const uint32_t (&k)[2][8], int s, uint32_t (&a)[1][4]) {
#pragma unroll
        for (int r = 0; r < 4; ++r) a[0][r] = k[r & 1][2 * s + (r >> 1)];
    }
    static __device__ __forceinline__ void values(const uint32_t (&v)[4][4], int i, uint32_t (&a)[1][4]) {
#pragma unroll
        for (int r = 0; r < 4; ++r) a[0][r] = __byte_perm(v[2 * (r >> 1)][i], v[2 * (r >> 1) + 1][i], r & 1 ? 0x7632 : 0x5410);
    }
};
template <>
struct Format<TIE_KV_INT8> {
    static constexpr int kBytes = 1;
};

// An item, or a part of one, as one warp has it. It lies in shared memory and is read (volatile)
// where it is needed: in registers it would take those of the operands.
struct Item {
    int row0, rows, i0;                // unit's first row, its rows, the item's first of them
    int ctx, keys;                     // UnitShape's
    int b0, b1;                        // steps
    int own, whole, parts;             // whole: no stretch cuts it; parts: how many it has, if this is the first
    const int32_t* table;
    __device__ __forceinline__ int pages() const volatile { return (keys + kPageRows - 1) / kPageRows; }
    // the last position that row i sees
    __device__ __forceinline__ int last(const SharedArgs& a, int i) const volatile {
        return own ? ctx + a.by_group(min(i, rows - 1)) : keys - 1;
    }
};
using ItemAt = const volatile Item*;

// The values that are not finite of keys [key0, key1) that some of the item's rows see and
// others do not, for the rows that see them. Rare: out of line.
template <int FMT>
__device__ __noinline__ void add_odd(const SharedArgs& a, const int32_t* table, int head, int key0, int key1, int last0, int last1, int dim,
                                     float* o0, float* o1) {
    constexpr int kBytes = Format<FMT>::kBytes;
    for (int key = key0; key < key1; ++key) {
        const int e = __ldg(table + key / kPageRows);
        if (e < 0 || e >= a.n_pages) continue;
        const size_t at = (((size_t)e * kPageRows + key % kPageRows) * a.n_kv_head + head) * kHeadDim + dim;
        for (int d = 0; d < 8; ++d) {
            float v;
            if constexpr (kBytes == 2) v = __bfloat162float(static_cast<const __nv_bfloat16*>(a.v)[at + d]);
            else v = static_cast<const float*>(a.v)[at + d];
            if (fabsf(v) < INFINITY) continue;
            if (key <= last0) o0[d] += v;
            if (key <= last1) o1[d] += v;
        }
    }
}

template <int NT>
struct WarpState {
    float o[NT][4][4];                 // [i][e]: dim 8 g + 2 i + e / 2 of column 2 c + e % 2
    float m[NT][2], l[NT][2];          // of columns 2 c, 2 c + 1 (l: this lane's keys only)
};

// What a warp has in its registers of the step it is at: each half is loaded as soon as the
// half before it has been used, so that the keys of the next step are on their way
// during this one's softmax and values, and its values during the next one's scores. (The
// registers that hold a step anyway are the buffer.)
template <int FMT, int PG>
struct StepLoads {
    static constexpr int kBytes = Format<FMT>::kBytes, KW = 4 * kBytes, VW = 2 * kBytes;
    uint32_t k[PG][2][KW], v[PG][4][VW];
    float ks[PG][2], vs[PG][2];
    int entry[PG];                     // of the step that is loaded next
    unsigned mapped;                   // of its pages
    const char *k_at, *v_at;           // this lane's place in a page of the head
    const char *ks_at, *vs_at;
    unsigned page, scale_page;         // from page to page: bytes
    int w;                             // from row to row: bytes
    int head;
    __device__ __forceinline__ void start(const SharedArgs& a, int of_head, int g, int c) {
        head = of_head;
        w = a.n_kv_head * kHeadDim * kBytes;
        page = (unsigned)w * kPageRows;
        k_at = static_cast<const char*>(a.k) + head * kHeadDim * kBytes + (size_t)g * w + 16 * c * kBytes;
        v_at = static_cast<const char*>(a.v) + head * kHeadDim * kBytes + (size_t)(2 * c) * w + 8 * g * kBytes;
        if constexpr (FMT == TIE_KV_INT8) {
            ks_at = reinterpret_cast<const char*>(a.ks + head * kPageRows + g);
            vs_at = reinterpret_cast<const char*>(a.vs + head * kPageRows + g);
            scale_page = (unsigned)a.n_kv_head * kPageRows * (unsigned)sizeof(float);
        }
    }
    // (what is not mapped is read from the pool's first page, and counts for nothing)
    __device__ __forceinline__ void entries(const int32_t* table, int b, int table_pages, int n_pages) {
        mapped = 0;
#pragma unroll
        for (int p = 0; p < PG; ++p) {
            const int e = b * PG + p < table_pages ? __ldg(table + b * PG + p) : -1;
            const bool ok = e >= 0 && e < n_pages;
            entry[p] = ok ? e : 0;
            mapped |= (unsigned)ok << p;
        }
    }
    __device__ __forceinline__ void keys() {
#pragma unroll
        for (int p = 0; p < PG; ++p) {
            const char* at = k_at + (unsigned long long)(unsigned)entry[p] * page;
            load_words<KW>(at, 0, k[p][0]);
            load_words<KW>(at, 8 * w, k[p][1]);
            if constexpr (FMT == TIE_KV_INT8) {
                const float* s = reinterpret_cast<const float*>(ks_at + (unsigned long long)(unsigned)entry[p] * scale_page);
                ks[p][0] = __ldg(s);
                ks[p][1] = __ldg(s + 8);
            }
        }
    }
    __device__ __forceinline__ void values() {
#pragma unroll
        for (int p = 0; p < PG; ++p) {
            const char* at = v_at + (unsigned long long)(unsigned)entry[p] * page;
            load_words<VW>(at, 0, v[p][0]);
            load_words<VW>(at, w, v[p][1]);
            load_words<VW>(at, 8 * w, v[p][2]);
            load_words<VW>(at, 9 * w, v[p][3]);
            if constexpr (FMT == TIE_KV_INT8) {
                const float* s = reinterpret_cast<const float*>(vs_at + (unsigned long long)(unsigned)entry[p] * scale_page);
                vs[p][0] = __ldg(s);
                vs[p][1] = __ldg(s + 8);
            }
        }
    }
};

// The largest of a column's numbers: over the lanes that hold its keys.
__device__ __forceinline__ float column_max(float x) {
#pragma unroll
    for (int o = 4; o < 32; o <<= 1) x = fmaxf(x, __shfl_xor_sync(kAll, x, o));
    return x;
}

// The running maximum takes in a step's; the factor of what is there already.
__device__ __forceinline__ float move_max(float& m, float& l, float step_max, float* from) {
    const float m_new = fmaxf(m, step_max);
    *from = m_new == -INFINITY ? 0.f : m_new;
    const float alpha = ex2_ftz(m - *from);
    m = m_new;
    l *= alpha;
    return alpha;
}

// ---- fp32 and bf16 pages
// The steps of an item, the first of which is in `in` (at the end: the next item's first, if
// there is one). qs: the warp's operands of Q in shared memory.
template <int FMT, int NT>
__device__ __forceinline__ void run_steps(const SharedArgs& a, ItemAt it, ItemAt next, StepLoads<FMT, kPages<FMT, NT>>& in,
                                          const uint2* qs, int lane, WarpState<NT>& st) {
    using F = Format<FMT>;
    constexpr int PG = kPages<FMT, NT>, VW = 2 * F::kBytes, T = F::kTerms;
    const int g = lane >> 2, c = lane & 3, i0 = it->i0, table_pages = it->pages();
    const int32_t* const table = it->table;
    int last[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) last[n][e] = it->last(a, i0 + 8 * n + 2 * c + e);
    const int least = it->last(a, i0), most = it->last(a, i0 + 8 * NT - 1);
    // (positions behind `most` are seen by none of the rows; an item's own part may have no others)
    const int b1 = max(min(it->b1, most / (PG * kPageRows) + 1), it->b0 + 1);
    for (int b = it->b0; b < b1; ++b) {
        const int pos0 = b * PG * kPageRows;
        const unsigned mapped = in.mapped;
        const bool whole = pos0 + PG * kPageRows - 1 <= least && mapped == (1u << PG) - 1;
        const bool more = b + 1 < b1 || next;
        if (b + 1 < b1) in.entries(table, b + 1, table_pages, a.n_pages);
        else if (next) in.entries(next->table, next->b0, next->pages(), a.n_pages);
        // scores of keys g, g + 8 of each page: s[n PG + p][e], e / 2 the key, e % 2 the column
        constexpr int kAcc = NT * PG, kSmall = Products<T>::kSmall;
        float s[kAcc][4], s_small[kAcc][4];
        auto k_step = [&](auto first, int step) {              // of 16 dims
            constexpr bool kFirst = decltype(first)::value;
            uint32_t fa[PG][T][4];
            uint2 u[NT][3];
#pragma unroll
            for (int p = 0; p < PG; ++p) F::keys(in.k[p], step, fa[p]);
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 3; ++e) u[n][e] = qs[((n * 4 + step) * 3 + e) * 32 + lane];
            auto a_of = [&](int r, int t) -> const uint32_t(&)[4] { return fa[r % PG][t]; };
            auto b0_of = [&](int r, int t) { return u[r / PG][t].x; };
            auto b1_of = [&](int r, int t) { return u[r / PG][t].y; };
            add_products<kFirst, 0, kSmall, kAcc, T>(s_small, a_of, b0_of, b1_of);
            add_products<kFirst, kSmall, kSmall + 1, kAcc, T>(s, a_of, b0_of, b1_of);
        };
        k_step(std::true_type{}, 0);
        k_step(std::false_type{}, 1);
        k_step(std::false_type{}, 2);
        k_step(std::false_type{}, 3);
        if (more) in.keys();
        // values that no row of the item sees are zero; one that is not finite and that only
        // some rows see is left to add_odd
        bool odd = false;
        if (!whole) {
#pragma unroll
            for (int p = 0; p < PG; ++p)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int pos = pos0 + p * kPageRows + 2 * c + (r & 1) + 8 * (r >> 1);
                    if (pos > most || !(mapped >> p & 1)) {
#pragma unroll
                        for (int i = 0; i < VW; ++i) in.v[p][r][i] = 0u;
                    } else if (pos > least) {
#pragma unroll
                        for (int i = 0; i < VW; ++i) {
                            uint32_t& x = in.v[p][r][i];
                            if constexpr (FMT == TIE_KV_F32) {
                                if (magnitude(__uint_as_float(x)) >= kNotFinite) { x = 0u; odd = true; }
                            } else {
                                if ((x & 0x7f80u) == 0x7f80u) { x &= 0xffff0000u; odd = true; }
                                if ((x & 0x7f800000u) == 0x7f800000u) { x &= 0xffffu; odd = true; }
                            }
                        }
                    }
                }
        }
        float alpha[NT][2], from[NT][2];
#pragma unroll
        for (int r = 0; r < kAcc; ++r)
#pragma unroll
            for (int e = 0; e < 4; e += 2)
                (Float2x(s[r][e], s[r][e + 1]) + Float2x(s_small[r][e], s_small[r][e + 1])).get(s[r][e], s[r][e + 1]);
        if (!whole) {
#pragma unroll
            for (int r = 0; r < kAcc; ++r)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (!(mapped >> (r % PG) & 1) || pos0 + (r % PG) * kPageRows + g + 8 * (e >> 1) > last[r / PG][e & 1])
                        s[r][e] = -INFINITY;
        }
        float mx[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                mx[n][e] = fmaxf(s[n * PG][e], s[n * PG][2 + e]);
#pragma unroll
                for (int p = 1; p < PG; ++p) mx[n][e] = fmaxf(mx[n][e], fmaxf(s[n * PG + p][e], s[n * PG + p][2 + e]));
            }
#pragma unroll
        for (int o = 4; o < 32; o <<= 1)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 2; ++e) mx[n][e] = fmaxf(mx[n][e], __shfl_xor_sync(kAll, mx[n][e], o));
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) alpha[n][e] = move_max(st.m[n][e], st.l[n][e], mx[n][e], &from[n][e]);
#pragma unroll
        for (int p = 0; p < PG; ++p) {
            uint32_t pb[NT][2][3];     // the page's weights as B operands: [keys below 8, others][term]
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    float w[2];
                    {
                        const float(&y)[4] = s[n * PG + p];
                        (Float2x(y[2 * h], y[2 * h + 1]) + Float2x(-from[n][0], -from[n][1])).get(w[0], w[1]);
                        const Float2x x = Float2x(ex2_ftz(w[0]), ex2_ftz(w[1])) * Float2x(kWeight, kWeight);
                        (Float2x(st.l[n][0], st.l[n][1]) + x).get(st.l[n][0], st.l[n][1]);
                        x.get(w[0], w[1]);
                    }
                    uint32_t x[3];
                    split3(w[0], w[1], x);
#pragma unroll
                    for (int e = 0; e < 3; ++e) pb[n][h][e] = transposed(x[e]);
                }
            constexpr int kI = NT == 1 ? 2 : 1;    // dims' operands at a time: two accumulators at least take turns
#pragma unroll
            for (int i = 0; i < 4; i += kI) {
                uint32_t fv[kI][T][4];
#pragma unroll
                for (int j = 0; j < kI; ++j) F::values(in.v[p], i + j, fv[j]);
                float d[kI * NT][4];
                add_products<true, 0, kSmall + 1, kI * NT, T>(
                    d, [&](int r, int t) -> const uint32_t(&)[4] { return fv[r / NT][t]; },
                    [&](int r, int t) { return pb[r % NT][0][t]; }, [&](int r, int t) { return pb[r % NT][1][t]; });
#pragma unroll
                for (int r = 0; r < kI * NT; ++r)
#pragma unroll
                    for (int e = 0; e < 4; e += 2) {
                        float &o0 = st.o[r % NT][i + r / NT][e], &o1 = st.o[r % NT][i + r / NT][e + 1];
                        const Float2x o(o0, o1), x(d[r][e], d[r][e + 1]);
                        (p == 0 ? fma2(o, Float2x(alpha[r % NT][0], alpha[r % NT][1]), x) : o + x).get(o0, o1);
                    }
            }
        }
        if (more) in.values();
        if (__any_sync(kAll, odd)) {
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                float extra[2][8] = {};
                add_odd<FMT>(a, it->table, in.head, max(pos0, least + 1), min(pos0 + PG * kPageRows, most + 1), last[n][0], last[n][1], 8 * g,
                             extra[0], extra[1]);
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e) st.o[n][i][e] += extra[e & 1][2 * i + (e >> 1)];
            }
        }
    }
}

// ---- pages in 8 bits
// Levels are operands of integer MMAs (m16n8k32, at the bf16 ones' rate for twice the sums)
// as they lie in memory. A query's elements become integers of 24 bits, relative to its
// largest, and a step's weights (times their values' scales) integers of 23, relative to
// the step's largest of their row: three 8-bit digits each, the top one signed. Sums of a
// digit are exact, and need no conversion: a digit's sum over 64 is below 2^21, so where it starts at the
// bits of 1.5 2^23 it ends as the bits of the fp32 number 1.5 2^23 + sum.
// Against bf16 terms (levels converted, three MMAs of half the depth) that is half the MMAs and a third
// of the instructions.

// Sums of digits start as floats of these bits: 1.5 2^23 for digit 0, 1.5 2^31 for digit 1 (whose
// last place is worth 256), 1.5 2^39 for digit 2 (65536).
constexpr int kStart0 = 0x4b400000, kStart1 = 0x4f400000, kStart2 = 0x53400000;

// d = a b + c, all of c `START`, if FIRST, else d
template <bool SIGNED, bool FIRST, int START>
__device__ __forceinline__ void mma_s8(int (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    const int c0 = FIRST ? START : d[0], c1 = FIRST ? START : d[1], c2 = FIRST ? START : d[2], c3 = FIRST ? START : d[3];
    if constexpr (SIGNED)
        asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
                     "{%10, %11, %12, %13};"
                     : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "r"(c0), "r"(c1), "r"(c2), "r"(c3));
    else
        asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.u8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
                     "{%10, %11, %12, %13};"
                     : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "r"(c0), "r"(c1), "r"(c2), "r"(c3));
}
// the three digits' sums
template <bool FIRST>
__device__ __forceinline__ void mma_digits(int (&d)[3][4], const uint32_t (&a)[4], const uint32_t (&b0)[3], const uint32_t (&b1)[3]) {
    mma_s8<false, FIRST, kStart0>(d[0], a, b0[0], b1[0]);
    mma_s8<false, FIRST, kStart1>(d[1], a, b0[1], b1[1]);
    mma_s8<true, FIRST, kStart2>(d[2], a, b0[2], b1[2]);
}
// d0 + 256 d1 + 65536 d2 of the digits' sums: each step but the last addition is exact or to the last place of
// its result
__device__ __forceinline__ float joined(int d0, int d1, int d2) {
    const float high = __int_as_float(d2) - __int_as_float(kStart2);
    const float low = __int_as_float(d1) - (__int_as_float(kStart1) + __int_as_float(kStart0));
    return high + (low + __int_as_float(d0));
}
__device__ __forceinline__ float pow2_biased(int e) { return __uint_as_float((uint32_t)e << 23); }

template <int NT>
__device__ __forceinline__ void run_steps_q8(const SharedArgs& a, ItemAt it, ItemAt next,
                                             StepLoads<TIE_KV_INT8, kPages<TIE_KV_INT8, NT>>& in, const uint4* qs,
                                             const float* q_unit, int lane, WarpState<NT>& st) {
    constexpr int PG = kPages<TIE_KV_INT8, NT>;
    const int g = lane >> 2, c = lane & 3, i0 = it->i0, table_pages = it->pages();
    const int32_t* const table = it->table;
    int last[NT][2];
    float unit[NT][2];                 // what 1 in a column's integers stands for
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            last[n][e] = it->last(a, i0 + 8 * n + 2 * c + e);
            unit[n][e] = q_unit[8 * n + 2 * c + e];
        }
    const int least = it->last(a, i0), most = it->last(a, i0 + 8 * NT - 1);
    const int b1 = max(min(it->b1, most / (PG * kPageRows) + 1), it->b0 + 1);
    for (int b = it->b0; b < b1; ++b) {
        const int pos0 = b * PG * kPageRows;
        const unsigned mapped = in.mapped;
        const bool whole = pos0 + PG * kPageRows - 1 <= least && mapped == (1u << PG) - 1;
        const bool more = b + 1 < b1 || next;
        if (b + 1 < b1) in.entries(table, b + 1, table_pages, a.n_pages);
        else if (next) in.entries(next->table, next->b0, next->pages(), a.n_pages);
        float s[NT][PG][4];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            uint4 u[3];
#pragma unroll
            for (int e = 0; e < 3; ++e) u[e] = qs[(n * 3 + e) * 32 + lane];
#pragma unroll
            for (int p = 0; p < PG; ++p) {
                int d[3][4];
                const uint32_t f0[4] = {in.k[p][0][0], in.k[p][1][0], in.k[p][0][1], in.k[p][1][1]};
                const uint32_t f1[4] = {in.k[p][0][2], in.k[p][1][2], in.k[p][0][3], in.k[p][1][3]};
                mma_digits<true>(d, f0, {u[0].x, u[1].x, u[2].x}, {u[0].y, u[1].y, u[2].y});
                mma_digits<false>(d, f1, {u[0].z, u[1].z, u[2].z}, {u[0].w, u[1].w, u[2].w});
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    s[n][p][e] = joined(d[0][e], d[1][e], d[2][e]) * unit[n][e & 1] * in.ks[p][e >> 1];
            }
        }
        if (more) in.keys();
        uint32_t vt[PG][8];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            float mx[2] = {-INFINITY, -INFINITY}, alpha[2], from[2], top[2] = {0.f, 0.f}, up[2], down[2];
            if (!whole) {
#pragma unroll
                for (int p = 0; p < PG; ++p)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (!(mapped >> p & 1) || pos0 + p * kPageRows + g + 8 * (e >> 1) > last[n][e & 1]) s[n][p][e] = -INFINITY;
            }
#pragma unroll
            for (int p = 0; p < PG; ++p)
#pragma unroll
                for (int e = 0; e < 4; ++e) mx[e & 1] = fmaxf(mx[e & 1], s[n][p][e]);
#pragma unroll
            for (int e = 0; e < 2; ++e) alpha[e] = move_max(st.m[n][e], st.l[n][e], column_max(mx[e]), &from[e]);
#pragma unroll
            for (int p = 0; p < PG; ++p)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float& x = s[n][p][e];
                    const float w = ex2_ftz(x - from[e & 1]);
                    st.l[n][e & 1] = fmaf(w, kWeight, st.l[n][e & 1]);
                    // (a scale of a key that the row does not see may be anything)
                    const bool none = !whole && x == -INFINITY;
                    x = w * in.vs[p][e >> 1];
                    if (none) x = 0.f;
                    top[e & 1] = max_abs(top[e & 1], x);
                }
#pragma unroll
            for (int e = 0; e < 2; ++e) {
#pragma unroll
                for (int o = 4; o < 32; o <<= 1) top[e] = max_abs(top[e], __shfl_xor_sync(kAll, top[e], o));
                // the largest is below 2^(x - 126): times 2^(148 - x), it is at most 2^22
                const int x = max((int)(__float_as_uint(top[e]) >> 23), 53);
                up[e] = pow2_biased(275 - x);
                down[e] = x >= 255 ? top[e] * 0.f : pow2_biased(x - 51);       // (times kWeight; NaN where there is no largest)
            }
            uint32_t wb[PG][3];            // digits of four keys' weights
#pragma unroll
            for (int p = 0; p < PG; ++p) {
                int w[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) w[e] = __float_as_int(fmaf(s[n][p][e], up[e & 1], __int_as_float(kStart0))) - kStart0;
                const uint32_t x = transposed(__byte_perm(w[0], w[1], 0x5410)), y = transposed(__byte_perm(w[2], w[3], 0x5410));
                const uint32_t z = transposed(__byte_perm(__byte_perm(w[0], w[2], 0x0062), __byte_perm(w[1], w[3], 0x0062), 0x5410));
                wb[p][0] = __byte_perm(x, y, 0x6420);
                wb[p][1] = __byte_perm(x, y, 0x7531);
                wb[p][2] = __byte_perm(z, z, 0x3120);
            }
            if (n == 0) {
                // the values of four keys of a dim side by side (not sooner: they are still on their
                // way during the scores and the softmax)
#pragma unroll
                for (int p = 0; p < PG; ++p)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const uint32_t(&v)[4][2] = in.v[p];
                        const uint32_t x = __byte_perm(v[0][h], v[1][h], 0x5140), y = __byte_perm(v[0][h], v[1][h], 0x7362);
                        const uint32_t z = __byte_perm(v[2][h], v[3][h], 0x5140), w = __byte_perm(v[2][h], v[3][h], 0x7362);
                        vt[p][4 * h] = __byte_perm(x, z, 0x5410);
                        vt[p][4 * h + 1] = __byte_perm(x, z, 0x7632);
                        vt[p][4 * h + 2] = __byte_perm(y, w, 0x5410);
                        vt[p][4 * h + 3] = __byte_perm(y, w, 0x7632);
                    }
            }
#pragma unroll
            for (int p = 0; p < PG; p += 2)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    int d[3][4];
                    const uint32_t fv[4] = {vt[p][2 * i], vt[p][2 * i + 1], vt[p + 1][2 * i], vt[p + 1][2 * i + 1]};
                    mma_digits<true>(d, fv, wb[p], wb[p + 1]);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        float& o = st.o[n][i][e];
                        o = fmaf(joined(d[0][e], d[1][e], d[2][e]), down[e & 1], p == 0 ? o * alpha[e & 1] : o);
                    }
                }
        }
        if (more) in.values();
    }
}

// bytes of a warp's Q operands
template <int NT>
constexpr int kQBytes = NT * 2 * 3 * 32 * (int)sizeof(uint4);

// Items of prefixes have 8 NP rows, those of sequences 8 NO; both stand in one line, so a decode
// step's products with a prefix run beside the reading of its sequences' pages.
template <int FMT, int NP, int NO>
__global__ void __launch_bounds__(kThreads, kCtas<FMT, NP>) shared_kernel(const __grid_constant__ SharedArgs a, int first) {
    // (the call's first kernel waits for what comes before the call, and only then lets the next one
    // begin, which does not wait for it)
    if (first) pdl_wait();
    pdl_trigger();
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ ScheduleScratch<kThreads> scratch;
    __shared__ Item s_items[kWarps][2];
    static_assert(NP >= NO && kPages<FMT, NP> == kPages<FMT, NO>, "one line");
    __shared__ float s_unit[kWarps][8 * NP];       // pages in 8 bits: run_steps_q8's q_unit
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5, g = lane >> 2, c = lane & 3;
    const Line& line = a.line[1];
    uint4* qs = reinterpret_cast<uint4*>(smem) + (size_t)warp * (kQBytes<NP> / sizeof(uint4));
    const Plan plan = build_plan<kThreads>(a, line.u0, line.u1, smem + kWarps * kQBytes<NP>, &scratch, t);
    const long long* const base = plan.base;
    const int n_units = line.u1 - line.u0;
    const long long total = base[n_units], share = share_of(line, total);
    const int me = blockIdx.x * kWarps + warp, team = me / a.n_kv_head;
    long long x = team * share;
    const long long end = team < line.teams ? min(x + share, total) : 0;
    int u = x < end ? owner_of<long long>(base, n_units, x) : 0;
    // the next part of this warp's stretch that has steps
    auto find = [&](Item* to) -> bool {
        while (x < end) {
            while (base[u + 1] <= x) ++u;          // (units without rows have no places)
            const UnitShape s = unit_shape(a, plan.n, line.u0 + u);
            const bool own = line.u0 + u >= a.n_group;
            const int places = unit_places(s, line);
            const long long in = x - base[u], item = quotient(in, places);
            const int off = (int)(in - item * places);
            const int stop = (int)min((long long)places, off + (end - x));
            const long long first = x - off;       // the item's first place
            x += stop - off;
            if (stop - 1 <= max(off - 1, 0)) continue;
            // (the item's first step is in this warp's stretch, and its last place in this one or a later one's)
            const bool begins = first + 1 >= team * share, whole = begins && first + places <= (team + 1) * share;
            __syncwarp();
            if (lane == 0) {
                to->own = own;
                to->row0 = s.row0;
                to->rows = s.rows;
                to->i0 = (int)item * 8 * (own ? NO : NP);
                to->ctx = s.ctx;
                to->keys = s.keys;
                to->b0 = max(off - 1, 0);
                to->b1 = stop - 1;
                to->table = own ? a.table + (size_t)(line.u0 + u - a.n_group) * a.width : a.ptable + (size_t)u * a.pwidth;
                to->whole = whole;
                to->parts = whole ? 1 : begins ? 1 + (int)quotient(first + places - 1 - team * share, share) : 0;
            }
            __syncwarp();
            return true;
        }
        return false;
    };
    const int head = me - team * a.n_kv_head;
    int at = 0;                        // which of the warp's two items is this one
    StepLoads<FMT, kPages<FMT, NP>> in;
    bool here = find(&s_items[warp][0]);
    if (here) {
        ItemAt it = &s_items[warp][0];
        in.start(a, head, g, c);
        in.entries(it->table, it->b0, it->pages(), a.n_pages);
        in.keys();
        in.values();
    }
    auto process = [&](auto height) {
        constexpr int NT = decltype(height)::value;
        ItemAt it = &s_items[warp][at];
        // Q, scaled, as B operands: column g, this lane's 16 dims
        __syncwarp();
        const int row0 = it->row0, n_rows = it->rows, i0 = it->i0;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const int i = min(i0 + 8 * n + g, n_rows - 1), tok = a.by_group(i);
            const float* q = a.q + (size_t)(row0 + tok) * a.ldq + (head * a.group + i - tok * a.group) * kHeadDim + 16 * c;
            float y[16];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float4 v = __ldg(reinterpret_cast<const float4*>(q) + j);
                y[4 * j] = v.x * a.scale2; y[4 * j + 1] = v.y * a.scale2; y[4 * j + 2] = v.z * a.scale2; y[4 * j + 3] = v.w * a.scale2;
            }
            if constexpr (FMT == TIE_KV_INT8) {
                float top = 0.f;
#pragma unroll
                for (int j = 0; j < 16; ++j) top = max_abs(top, y[j]);
                top = max_abs(top, __shfl_xor_sync(kAll, top, 1));
                top = max_abs(top, __shfl_xor_sync(kAll, top, 2));
                const int x = max((int)(__float_as_uint(top) >> 23), 23);    // the largest is below 2^(x - 126)
                const float up = pow2_biased(276 - x);
                uint32_t z[4][3];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    int w[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) w[e] = min(__float2int_rn(y[4 * j + e] * up), (1 << 23) - 1);
#pragma unroll
                    for (int e = 0; e < 3; ++e)
                        z[j][e] = __byte_perm(__byte_perm(w[0], w[1], 0x40 + 0x11 * e), __byte_perm(w[2], w[3], 0x40 + 0x11 * e), 0x5410);
                }
#pragma unroll
                for (int e = 0; e < 3; ++e) qs[(n * 3 + e) * 32 + lane] = make_uint4(z[0][e], z[1][e], z[2][e], z[3][e]);
                if (c == 0) s_unit[warp][8 * n + g] = x >= 255 ? top * 0.f : pow2_biased(x - 22);
            } else {
                uint2* const to = reinterpret_cast<uint2*>(qs);
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    uint32_t x[3], z[3];
                    split3(y[4 * k], y[4 * k + 1], x);
                    split3(y[4 * k + 2], y[4 * k + 3], z);
#pragma unroll
                    for (int e = 0; e < 3; ++e) to[((n * 4 + k) * 3 + e) * 32 + lane] = make_uint2(x[e], z[e]);
                }
            }
        }
        __syncwarp();
        WarpState<NT> st;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int e = 0; e < 2; ++e) { st.m[n][e] = -INFINITY; st.l[n][e] = 0.f; }
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) st.o[n][i][e] = 0.f;
        }
        const bool more = find(&s_items[warp][at ^ 1]);
        ItemAt next = more ? &s_items[warp][at ^ 1] : nullptr;
        if constexpr (FMT == TIE_KV_INT8) run_steps_q8<NT>(a, it, next, in, qs, s_unit[warp], lane, st);
        else run_steps<FMT, NT>(a, it, next, in, reinterpret_cast<const uint2*>(qs), lane, st);
        // where the result goes: out, the rows' own place, or a part of this warp's
        const int whole = it->whole, parts = it->parts, own = it->own, end_row0 = it->row0, end_rows = it->rows, end_i0 = it->i0;
        const size_t slot = (2 * (size_t)me + (parts > 0)) * line.per;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
#pragma unroll
                for (int o = 4; o < 32; o <<= 1) st.l[n][e] += __shfl_xor_sync(kAll, st.l[n][e], o);
                const int in_item = 8 * n + 2 * c + e, i = end_i0 + in_item;
                if (i >= end_rows) continue;
                const int tok = a.by_group(i), h = head * a.group + i - tok * a.group;
                const size_t row = end_row0 + tok, place = row * a.n_head + h;
                if (parts && g == 0) a.place[own][place] = make_int2(whole ? -1 : (int)slot + in_item, parts);
                float f = 1.f, *to;
                if (whole && a.n_group == 0) {
                    f = st.l[n][e] == 0.f ? 0.f : 1.f / st.l[n][e];
                    to = a.out + row * a.ldo + h * kHeadDim;
                } else {
                    to = whole ? a.whole_o[own] + place * kHeadDim : line.part_o + (slot + in_item) * kHeadDim;
                    float* ml = whole ? a.whole_ml[own] + 2 * place : line.part_ml + 2 * (slot + in_item);
                    if (g == 0) *reinterpret_cast<float2*>(ml) = make_float2(st.m[n][e], st.l[n][e]);
                }
                float4* p = reinterpret_cast<float4*>(to + 8 * g);
                const float(&o)[4][4] = st.o[n];
                if (f == 0.f) {
                    p[0] = p[1] = make_float4(0.f, 0.f, 0.f, 0.f);
                } else {
                    p[0] = make_float4(o[0][e] * f, o[0][2 + e] * f, o[1][e] * f, o[1][2 + e] * f);
                    p[1] = make_float4(o[2][e] * f, o[2][2 + e] * f, o[3][e] * f, o[3][2 + e] * f);
                }
            }
        at ^= 1;
        here = more;
    };
    while (here) {
        if (NP == NO || s_items[warp][at].own) process(std::integral_constant<int, NO>{});
        else process(std::integral_constant<int, NP>{});
    }
    // (nothing above needs another kernel's results, but what waits for this kernel waits
    // for the one before it too)
    pdl_wait();
}

// ------------------------------------------------------------------ the join --
// A row's parts from both sources, in one line: the sequence's own first. Part 0 of a cut
// item lies in its warp's second place, the others in the first ones of the head's warps in
// the teams that follow.
struct Parts {
    const float *o[2], *ml[2];         // [prefix, own]: the part that is first
    int n[2], per[2], apart[2];        // per: rows of a place; apart: warps or CTAs from part to part
    __device__ __forceinline__ void at(int k, const float** to, const float** ml_to) const {
        const int w = k < n[1], j = w ? k : k - n[1];
        const size_t row = j == 0 ? 0 : ((size_t)2 * j * apart[w] - 1) * per[w];
        *to = o[w] + row * kHeadDim;
        *ml_to = ml[w] + 2 * row;
    }
};

// A warp adds parts k0, k0 + dk, ... to what it has of a row: lane l dims 2 l, 2 l + 1.
struct RowSum {
    float m, l, x, y;
};
__device__ __forceinline__ void add_parts(RowSum& r, const Parts& z, int k0, int dk, int lane) {
    constexpr int kAhead = 8;
    const int n = z.n[0] + z.n[1];
    for (int k = k0; k < n; k += kAhead * dk) {
        float2 ml[kAhead], v[kAhead];
        float m = r.m;
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            ml[j] = make_float2(-INFINITY, 0.f);
            v[j] = make_float2(0.f, 0.f);
            if (k + j * dk < n) {
                const float *o, *of;
                z.at(k + j * dk, &o, &of);
                ml[j] = __ldcg(reinterpret_cast<const float2*>(of));
                v[j] = __ldcg(reinterpret_cast<const float2*>(o) + lane);
            }
        }
#pragma unroll
        for (int j = 0; j < kAhead; ++j) m = fmaxf(m, ml[j].x);
        const float from = m == -INFINITY ? 0.f : m, f = ex2_ftz(r.m - from);
        r.m = m;
        r.l *= f;
        r.x *= f;
        r.y *= f;
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            // (a part that has seen no key is all zeros; one whose factor is zero is still
            // multiplied: a value that is not finite stays so)
            const float e = ex2_ftz(ml[j].x - from);
            r.l = fmaf(ml[j].y, e, r.l);
            r.x = fmaf(v[j].x, e, r.x);
            r.y = fmaf(v[j].y, e, r.y);
        }
    }
}

// CTAs (s, y) take sequence s's rows: a row and query head by a warp, or by all warps of the
// CTA where there are few rows (and many parts of each, then). What the rows of a sequence
// that is left out hold in `place` is nothing: they are told by the lengths.
template <bool WIDE>
__global__ void __launch_bounds__(kThreads) shared_join_kernel(const __grid_constant__ SharedArgs a) {
    __shared__ int s_group;
    __shared__ RowSum s_sum[kWarps][32];
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5, q = blockIdx.x;
    const Lengths lengths{a.row_start, a.ctx, a.gstart, a.plen};
    const UnitShape s = unit_shape(a, lengths, a.n_group + q);
    if (!s.rows) {
        pdl_wait();                    // (whoever waits for this kernel waits for the one before it too)
        return;
    }
    bool grouped = false;
    if (a.n_group) {
        if (t == 0) s_group = -1;
        __syncthreads();
        for (int u = t; u < a.n_group; u += kThreads)
            if (__ldg(a.gstart + u) <= q && q < __ldg(a.gstart + u + 1)) atomicMax(&s_group, u);
        __syncthreads();
        if (s_group >= 0) {
            const UnitShape p = unit_shape(a, lengths, s_group);
            grouped = p.rows && s.row0 >= p.row0 && s.row0 + s.tokens <= p.row0 + p.tokens;
        }
    }
    pdl_wait();
    const long long pairs = (long long)s.tokens * a.n_head;
    for (long long i = WIDE ? blockIdx.y : (long long)blockIdx.y * kWarps + warp; i < pairs;
         i += WIDE ? gridDim.y : (long long)gridDim.y * kWarps) {
        const int row = s.row0 + (int)((unsigned)i / (unsigned)a.n_head), h = (int)((unsigned)i % (unsigned)a.n_head);
        const size_t at = (size_t)row * a.n_head + h;
        Parts z;
#pragma unroll
        for (int w = 0; w < 2; ++w) {
            const bool there = w || grouped;
            const int2 where = there ? __ldcg(a.place[w] + at) : make_int2(0, 0);
            const Line& l = a.line[w];
            z.n[w] = where.y;
            z.per[w] = l.per;
            z.apart[w] = l.heads == 1 ? a.n_kv_head : 1;
            z.o[w] = where.x < 0 ? a.whole_o[w] + at * kHeadDim : l.part_o + (size_t)where.x * kHeadDim;
            z.ml[w] = where.x < 0 ? a.whole_ml[w] + 2 * at : l.part_ml + 2 * (size_t)where.x;
        }
        if (a.n_group == 0 && z.n[1] == 1) continue;      // written already
        RowSum r{-INFINITY, 0.f, 0.f, 0.f};
        add_parts(r, z, WIDE ? warp : 0, WIDE ? kWarps : 1, lane);
        if constexpr (WIDE) {
            s_sum[warp][lane] = r;
            __syncthreads();
            if (warp == 0) {
                float m = r.m;
#pragma unroll
                for (int v = 1; v < kWarps; ++v) m = fmaxf(m, s_sum[v][lane].m);
                const float from = m == -INFINITY ? 0.f : m;
                float f = ex2_ftz(r.m - from);
                r = RowSum{m, r.l * f, r.x * f, r.y * f};
#pragma unroll
                for (int v = 1; v < kWarps; ++v) {
                    const RowSum u = s_sum[v][lane];
                    f = ex2_ftz(u.m - from);
                    r.l = fmaf(u.l, f, r.l);
                    r.x = fmaf(u.x, f, r.x);
                    r.y = fmaf(u.y, f, r.y);
                }
            }
        }
        if (!WIDE || warp == 0) {
            const float2 y = r.l == 0.f ? make_float2(0.f, 0.f) : make_float2(r.x / r.l, r.y / r.l);
            *(reinterpret_cast<float2*>(a.out + (size_t)row * a.ldo + h * kHeadDim) + lane) = y;
        }
        if constexpr (WIDE) __syncthreads();
    }
}

// --------------------------------------------------------------- the entry ----
// Prefixes go to k_shared_tc.cu from this many rows of a group and K/V head, on average, and this
// many scores (as the tables' width bounds them): its tiles have 128 rows, and it is a kernel
// more, which nothing else runs beside. One group, 8 heads, a token each, without and with
// it, us (fp32; bf16; 8 bits):
//   128 sequences behind  700 (0.7 M scores)  23 and 24;  19 and 22;  18 and 22
//    64 sequences behind 4000 (2.0 M)         31 and 32;  24 and 29;  22 and 28
//   128 sequences behind 4000 (4.1 M)         46 and 36;  33 and 32;  29 and 31
//   256 sequences behind 4000 (8.2 M)         75 and 53;  53 and 46;  48 and 46
// (256 sequences behind 700, 12 heads, with 300 positions of their own, fp32, 2.2 M: 75 and 92; 640
// rows a head behind 14336, 8 heads, bf16, 73 M: 271 and 116.) The lengths are on the device, so a table much wider than
// its prefixes takes the slower one of these.
constexpr int kTcFrom = 64;
constexpr long long tc_scores(int format) { return format == TIE_KV_F32 ? 3000000 : format == TIE_KV_BF16 ? 4000000 : 8000000; }
int most_warps(int sms) { return sms * 16; }

// floats of the workspace: parts of two lines, and the whole items of two sources
size_t part_floats(int sms) { return (size_t)2 * most_warps(sms) * 32 * (kHeadDim + 2); }
// (and their places)
size_t workspace_floats(int sms, long long pairs) { return 2 * part_floats(sms) + (size_t)2 * pairs * (kHeadDim + 2 + 2); }

using Kernel = void (*)(SharedArgs, int);
// What is launched for items of 8 np and 8 no rows: 1 1, 2 1, 2 2 or 4 4.
struct Variant {
    Kernel kernel;
    int pages, ctas;                   // of a step; on an SM
    size_t q_bytes;
};
template <int FMT, int NP, int NO>
Variant variant() {
    return Variant{shared_kernel<FMT, NP, NO>, kPages<FMT, NP>, kCtas<FMT, NP>, (size_t)kWarps * kQBytes<NP>};
}
template <int FMT>
Variant variant_of(int np, int no) {
    return np == 1 ? variant<FMT, 1, 1>() : np == 4 ? variant<FMT, 4, 4>() : no == 1 ? variant<FMT, 2, 1>() : variant<FMT, 2, 2>();
}

constexpr uint32_t kWaitLimitNs = 2000000000u;         // of a wait in k_shared_tc.cu
thread_local uint32_t drill_ns = 0;                    // of the next one's, by tie_attention_shared_wait_drill

}  // namespace
}  // namespace tie

using namespace tie;

extern "C" model_status tie_attention_shared_wait_drill(uint64_t limit_ns) {
    if (limit_ns == 0 || limit_ns > kWaitLimitNs) return MODEL_ERR_ARG;
    drill_ns = (uint32_t)limit_ns;
    return MODEL_OK;
}

extern "C" size_t tie_attention_shared_workspace(int rows, int n_head) {
    int dev = 0;
    if (rows < 0 || n_head <= 0) return 0;
    if (cudaGetDevice(&dev) != cudaSuccess) { cudaGetLastError(); return 0; }
    return workspace_floats(sm_count(dev), (long long)rows * n_head) * sizeof(float);
}

extern "C" model_status tie_attention_shared(const float* q, int ldq, int n_head, const void* k_pages, const void* v_pages,
                                             const float* k_scales, const float* v_scales, int kv_format, int n_pages,
                                             int n_kv_head, const int32_t* page_table, int pages_per_seq,
                                             const int32_t* row_start, const int32_t* ctx_lens, int n_seq, int max_new,
                                             int rows, const int32_t* prefix_table, int pages_per_prefix,
                                             const int32_t* prefix_lens, const int32_t* group_start, int n_group, float scale,
                                             float* out, int ldo, void* workspace, size_t workspace_bytes, int32_t* status,
                                             void* stream) {
    if (!k_pages || !v_pages || !page_table || !row_start || !ctx_lens || !workspace) return MODEL_ERR_ARG;
    if (rows && (!q || !out)) return MODEL_ERR_ARG;           // arrays without rows have no address
    const bool q8 = kv_format == TIE_KV_INT8;
    if (!pool_shape_ok(q8 ? (int)TIE_KV_F32 : kv_format, n_pages, n_kv_head) || n_head <= 0 || n_head % n_kv_head || n_head > 8192)
        return MODEL_ERR_ARG;
    if (q8 ? !k_scales || !v_scales : k_scales || v_scales) return MODEL_ERR_ARG;
    if (pages_per_seq <= 0 || n_seq <= 0 || max_new < 0 || rows < 0 || !std::isfinite(scale)) return MODEL_ERR_ARG;
    if (n_group < 0 || (n_group ? !prefix_table || !prefix_lens || !group_start || pages_per_prefix <= 0
                                : prefix_table || prefix_lens || group_start))
        return MODEL_ERR_ARG;
    const int w = n_head * kHeadDim;
    if (ldq < w || ldo < w || (ldq & 3) || (ldo & 3)) return MODEL_ERR_ARG;
    if (!aligned16(q) || !aligned(k_pages, 32) || !aligned(v_pages, 32) || !aligned16(k_scales) || !aligned16(v_scales) ||
        !aligned16(out) || !aligned16(workspace))
        return MODEL_ERR_ARG;
    if (n_seq > kOpsMaxSeqs || n_group > kOpsMaxSeqs || pages_per_seq > kOpsMaxPages / 2 || pages_per_prefix > kOpsMaxPages / 2)
        return MODEL_ERR_CAPACITY;
    const long long pairs = (long long)rows * n_head;
    if (pairs > INT_MAX / 2) return MODEL_ERR_CAPACITY;
    if (rows == 0 || max_new == 0) return MODEL_OK;
    OnDeviceOf dev(out);
    if (dev.status() != MODEL_OK) return dev.status();
    const int sms = sm_count(dev.device());
    if (workspace_bytes < workspace_floats(sms, pairs) * sizeof(float)) return MODEL_ERR_CAPACITY;
    SharedArgs a{};
    a.q = q; a.ldq = ldq; a.n_head = n_head; a.group = n_head / n_kv_head; a.by_group = divisor(a.group); a.n_kv_head = n_kv_head;
    a.k = k_pages; a.v = v_pages; a.ks = k_scales; a.vs = v_scales; a.n_pages = n_pages;
    a.table = page_table; a.width = pages_per_seq; a.row_start = row_start; a.ctx = ctx_lens;
    a.n_seq = n_seq; a.max_new = max_new; a.rows = rows;
    a.ptable = prefix_table; a.pwidth = pages_per_prefix; a.plen = prefix_lens; a.gstart = group_start; a.n_group = n_group;
    a.scale2 = (float)((double)scale * 1.4426950408889634);
    a.out = out; a.ldo = ldo; a.status = status;
    float* f = static_cast<float*>(workspace);
    for (int i = 0; i < 2; ++i) {
        a.line[i].part_o = f;
        a.line[i].part_ml = f + part_floats(sms) / (kHeadDim + 2) * kHeadDim;
        f += part_floats(sms);
    }
    // (the values of both sources first: they are 16-byte aligned whatever `pairs` is)
    for (int i = 0; i < 2; ++i) {
        a.whole_o[i] = f + i * pairs * kHeadDim;
        a.whole_ml[i] = f + 2 * pairs * kHeadDim + i * pairs * 2;
        a.place[i] = reinterpret_cast<int2*>(f + 2 * pairs * (kHeadDim + 2) + i * pairs * 2);
    }
    // Rows that share keys, at most of a sequence and on average of a group, say how high the items are.
    const long long per_seq = (long long)max_new * a.group, per_group = n_group ? ((long long)rows * a.group - 1) / n_group + 1 : 0;
    const bool tc = per_group >= kTcFrom && pairs * ((long long)pages_per_prefix * kPageRows) >= tc_scores(kv_format);
    const int no = per_seq <= 8 ? 1 : per_seq <= 16 ? 2 : 4;
    const int np = tc || no > 1 || per_group <= 8 ? no : 2;
    const Variant v = q8 ? variant_of<TIE_KV_INT8>(np, no)
                         : kv_format == TIE_KV_BF16 ? variant_of<TIE_KV_BF16>(np, no) : variant_of<TIE_KV_F32>(np, no);
    for (int i = 0; i < 2; ++i) {
        Line& l = a.line[i];
        l.nt = i ? no : np;
        l.per = 8 * np;
        l.pages = v.pages;
        l.heads = 1;
        l.u0 = 0;
        l.u1 = n_group + n_seq;
        l.teams = sms * v.ctas * kWarps / n_kv_head;
        if (l.teams == 0) return MODEL_ERR_CAPACITY;          // (the K/V heads that are taken fit the GPU's warps)
    }
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (tc) {
        Line& l = a.line[0];
        l.nt = kTcRows / 8;
        l.per = kTcRows;
        l.pages = kTcPages;
        l.heads = n_kv_head;
        l.u1 = n_group;
        l.teams = shared_tc_ctas(sms);
        a.line[1].u0 = n_group;
        a.wait_ns = drill_ns ? drill_ns : kWaitLimitNs;
        a.stall = drill_ns != 0;
        drill_ns = 0;
        TIE_OP_CU(launch_shared_tc(a, kv_format, st));
        ++op_launches;
    } else {
        a.line[1].part_o = a.line[0].part_o;                  // one line
        a.line[1].part_ml = a.line[0].part_ml;
    }
    {
        const Line& l = a.line[1];
        const size_t smem = v.q_bytes + plan_bytes(l.u1 - l.u0, n_seq, n_group);
        // (always the most that any call wants: calls on other threads set it too)
        if (smem > 32 * 1024)
            TIE_OP_CU(cudaFuncSetAttribute(v.kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                           (int)(v.q_bytes + plan_bytes(2 * kOpsMaxSeqs, kOpsMaxSeqs, kOpsMaxSeqs))));
        TIE_OP_CU(launch_pdl(v.kernel, dim3((unsigned)(sms * v.ctas)), dim3(kThreads), smem, st, a, (int)!tc));
        ++op_launches;
    }
    const long long most_pairs = (long long)max_new * n_head;         // of a sequence
    const bool wide = pairs <= 8LL * sms;
    auto* join = wide ? shared_join_kernel<true> : shared_join_kernel<false>;
    const long long y = wide ? most_pairs : (most_pairs + kWarps - 1) / kWarps;
    TIE_OP_CU(launch_pdl(join, dim3((unsigned)n_seq, (unsigned)(y < 256 ? y : 256)), dim3(kThreads), 0, st, a));
    ++op_launches;
    return MODEL_OK;
}
