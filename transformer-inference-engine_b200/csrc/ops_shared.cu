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
// Work. An item is 8 NT rows that share keys (a sequence's new tokens or a group's, times
// the query heads of one K/V head) and all pages of those keys. All items of a call stand
// in one line, each as many places as it has steps of PG pages, and one for what it
// costs besides; every warp of the grid takes an equal stretch of the line, whatever
// the lengths are, and works alone (no barriers). An item that a stretch cuts leaves parts,
// which a second kernel joins; it finds them from the lengths, as the first one cut them.
//
// Products run on bf16 MMAs (m16n8k16). An fp32 number is exactly the sum of three bf16
// terms, a level of 8 bits and a bf16 number are one; products of terms below 2^-24 of the
// whole are left out (six MMAs a product over fp32 pages, three over the others). No operand
// is scaled, so any finite value keeps its bits. Keys are the MMA's 16 rows, so the rows
// of a decode step (one for each query head of a K/V head, where it has no prefix) fill
// its 8 columns as far as they go. K and V go from memory into operand registers without
// shared memory: a lane's 16 dims of a key may be any 16 of the sum, so it takes 16 in a
// row, and each lane's 8 dims of 4 values are packed in pairs of keys.
#include <cuda_bf16.h>

#include <climits>
#include <cmath>

#include "paged_attn.cuh"
#include "quant.cuh"

namespace tie {
namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr unsigned kAll = 0xffffffffu;
// Weights are 2^(s - max) times this, so that the sum of as many of them as there are
// positions (2^30) times any finite value stays finite.
constexpr float kWeight = 0x1p-30f;
// fewest steps worth a warp's stretch
constexpr int kMinShare = 3;

// Pages of a step: as many as keep 8 KB of a warp's loads on their way, with few rows.
template <int FMT, int NT>
constexpr int kPages = FMT == TIE_KV_F32 ? 1 : FMT == TIE_KV_BF16 ? (NT > 2 ? 1 : 2) : (NT > 2 ? 2 : 4);

// A line: units [u0, u1) (a unit below n_group is a group's prefix, the others are
// sequences), cut into stretches for `warps` warps.
struct Line {
    int u0, u1, nt, pages, warps;      // nt: of the items; pages: of a step
    float* part_o;                     // [2 * warps][8 nt][64]: a warp's parts of the item it goes on with
    float* part_ml;                    // and of the one that it begins; (maximum, sum)
};

struct SharedArgs {
    const float* q;
    int ldq, n_head, group, n_kv_head;
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
    Line line[2];                      // of the prefixes and of the sequences; line[1] may be line[0]
    int one_line;
};

// What a unit's rows are, and its keys. rows == 0: nothing to do.
struct UnitShape {
    int row0, tokens, rows, keys;      // keys: positions in its pages
    int ctx;                           // own: row i sees positions <= ctx + i / group; prefix: all
};

__device__ __forceinline__ UnitShape unit_shape(const SharedArgs& a, int u) {
    UnitShape s{};
    if (u < a.n_group) {
        const int s0 = __ldg(a.gstart + u), s1 = __ldg(a.gstart + u + 1), n = __ldg(a.plen + u);
        if (s0 < 0 || s1 <= s0 || s1 > a.n_seq || n <= 0 || n > (long long)a.pwidth * kPageRows) return s;
        const int r0 = __ldg(a.row_start + s0), r1 = __ldg(a.row_start + s1);
        if (r0 < 0 || r1 <= r0 || r1 > a.rows) return s;
        s.row0 = r0;
        s.tokens = r1 - r0;
        s.keys = n;
        s.ctx = n;
    } else {
        const int q = u - a.n_group;
        const int r0 = __ldg(a.row_start + q), r1 = __ldg(a.row_start + q + 1), c = __ldg(a.ctx + q);
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
__device__ __forceinline__ long long unit_items(const SharedArgs& a, const UnitShape& s, const Line& l) {
    return (long long)((s.rows + 8 * l.nt - 1) / (8 * l.nt)) * a.n_kv_head;
}

__device__ __forceinline__ long long share_of(const Line& l, long long total) {
    const long long even = (total + l.warps - 1) / l.warps;
    return even > kMinShare ? even : kMinShare;
}

// base[u - u0] places before unit u, all of them in base[u1 - u0]. Ends with a barrier.
__device__ __forceinline__ void build_base(const SharedArgs& a, int u0, int u1, long long* base,
                                           ScheduleScratch<kThreads>* sc, int t) {
    const int n = u1 - u0, per = (n + kThreads - 1) / kThreads;
    long long mine = 0, before;
    for (int i = 0; i < per; ++i) {
        const int u = u0 + t * per + i;
        if (u >= u1) break;
        const UnitShape s = unit_shape(a, u);
        const Line& l = a.line[u >= a.n_group];
        if (s.rows) mine += unit_items(a, s, l) * unit_places(s, l);
    }
    const long long total = scan_threads<kThreads>(mine, sc, t, &before);
    for (int i = 0; i < per; ++i) {
        const int u = u0 + t * per + i;
        if (u >= u1) break;
        base[u - u0] = before;
        if (per > 1) {                 // a thread's only unit needs no second look
            const UnitShape s = unit_shape(a, u);
            const Line& l = a.line[u >= a.n_group];
            if (s.rows) before += unit_items(a, s, l) * unit_places(s, l);
        }
    }
    if (t == 0) base[n] = total;
    __syncthreads();
}

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

// Bytes 0 and 2 of a word, as signed levels, in a pair of bf16: 0x4300 | u is 128 + u for
// u < 128, and 0x4380 is 256, so (128 + low 7 bits) - (128 + sign bit) is the level.
__device__ __forceinline__ uint32_t levels2(uint32_t w) {
    const uint32_t low = (w & 0x007f007fu) | 0x43004300u, sign = (w & 0x00800080u) | 0x43004300u;
    const __nv_bfloat162 v = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&low), *reinterpret_cast<const __nv_bfloat162*>(&sign));
    return *reinterpret_cast<const uint32_t*>(&v);
}

__device__ __forceinline__ uint32_t transposed(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

// Terms of two numbers: [0] the largest.
__device__ __forceinline__ void split3(float lo, float hi, uint32_t (&x)[3]) {
    x[0] = terms2(lo, hi);
    lo = rest(lo);
    hi = rest(hi);
    x[1] = terms2(lo, hi);
    x[2] = terms2(rest(lo), rest(hi));
}

// The MMA cuts its sums off, towards zero, so the products of the terms are added in two
// sets: d += the largest terms' product, and e += the others', which are 2^-8 of it (a product of
// terms below 2^-24 of the whole is left out). With all in one chain of 24 MMAs the error of the
// result was 2.0e-6 over fp32 pages (2-norm, 1000 positions), in two sets it is 4.0e-7.
__device__ __forceinline__ void main_product(float (&d)[4], const uint32_t (&a)[4], const uint32_t (&b0)[3],
                                             const uint32_t (&b1)[3]) {
    mma_bf16(d, a, b0[0], b1[0]);
}
template <int NA>
__device__ __forceinline__ void small_products(float (&e)[4], const uint32_t (&a)[NA][4], const uint32_t (&b0)[3],
                                               const uint32_t (&b1)[3]) {
    if constexpr (NA == 3) mma_bf16(e, a[2], b0[0], b1[0]);
    mma_bf16(e, a[0], b0[2], b1[2]);
    if constexpr (NA == 3) {
        mma_bf16(e, a[1], b0[1], b1[1]);
        mma_bf16(e, a[1], b0[0], b1[0]);
    }
    mma_bf16(e, a[0], b0[1], b1[1]);
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
    static constexpr int kApart = 1;   // from the first of a pair of dims to the second
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
    static constexpr int kApart = 1;
};
template <>
struct Format<TIE_KV_INT8> {
    static constexpr int kBytes = 1, kTerms = 1;
    static __device__ __forceinline__ void keys(const uint32_t (&k)[2][4], int s, uint32_t (&a)[1][4]) {
#pragma unroll
        for (int r = 0; r < 4; ++r) a[0][r] = levels2(k[r & 1][s] >> (8 * (r >> 1)));
    }
    static __device__ __forceinline__ void values(const uint32_t (&v)[4][2], int i, uint32_t (&a)[1][4]) {
#pragma unroll
        for (int r = 0; r < 4; r += 2) {
            const uint32_t w = __byte_perm(v[r][i >> 1], v[r + 1][i >> 1], i & 1 ? 0x7632 : 0x5410);
            a[0][r] = levels2(w);
            a[0][r + 1] = levels2(w >> 8);
        }
    }
    static constexpr int kApart = 2;   // bytes 0 and 2 of a word make a pair, and 1 and 3
};

// An item's rows, for one warp: their place in q and out.
struct Item {
    int row0, rows, i0, head;          // unit's first row, its rows, the item's first of them, K/V head
    int ctx, keys;                     // UnitShape's
    bool own;
    const int32_t* table;
    __device__ __forceinline__ int row(const SharedArgs& a, int i) const { return row0 + min(i, rows - 1) / a.group; }
    __device__ __forceinline__ int q_head(const SharedArgs& a, int i) const { return head * a.group + min(i, rows - 1) % a.group; }
    // the last position that row i sees
    __device__ __forceinline__ int last(const SharedArgs& a, int i) const { return own ? ctx + min(i, rows - 1) / a.group : keys - 1; }
};

// The values that are not finite of keys [key0, key1) that some of the item's rows see and
// others do not, for the rows that see them. Rare: out of line.
template <int FMT>
__device__ __noinline__ void add_odd(const SharedArgs& a, const Item& it, int key0, int key1, int last0, int last1, int dim,
                                     float* o0, float* o1) {
    constexpr int kBytes = Format<FMT>::kBytes;
    for (int key = key0; key < key1; ++key) {
        const int e = __ldg(it.table + key / kPageRows);
        if (e < 0 || e >= a.n_pages) continue;
        const size_t at = (((size_t)e * kPageRows + key % kPageRows) * a.n_kv_head + it.head) * kHeadDim + dim;
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

template <int FMT, int NT>
struct WarpState {
    float o[NT][4][4];                 // [i][e]: dim 8 g + 2 i + e / 2 of column 2 c + e % 2
    float m[NT][2], l[NT][2];          // of columns 2 c, 2 c + 1 (l: this lane's keys only)
};

// Steps [b0, b1) of an item. qs: the warp's operands of Q in shared memory.
template <int FMT, int NT>
__device__ __forceinline__ void run_steps(const SharedArgs& a, const Item& it, int b0, int b1, const uint4* qs, int lane,
                                          WarpState<FMT, NT>& st) {
    using F = Format<FMT>;
    constexpr int PG = kPages<FMT, NT>, KW = 4 * F::kBytes, VW = 2 * F::kBytes, T = F::kTerms;
    const int g = lane >> 2, c = lane & 3;
    const size_t w = (size_t)a.n_kv_head * kHeadDim * F::kBytes;      // bytes of a row
    const int n_pages = (it.keys + kPageRows - 1) / kPageRows;
    int last[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) last[n][e] = it.last(a, it.i0 + 8 * n + 2 * c + e);
    const int least = it.last(a, it.i0), most = it.last(a, it.i0 + 8 * NT - 1);
    b1 = min(b1, most / (PG * kPageRows) + 1);     // later positions are seen by none of the rows
    int entry[PG];
    auto entries = [&](int b) {
#pragma unroll
        for (int p = 0; p < PG; ++p) entry[p] = b * PG + p < n_pages ? __ldg(it.table + b * PG + p) : -1;
    };
    if (b0 < b1) entries(b0);
    for (int b = b0; b < b1; ++b) {
        uint32_t kw[PG][2][KW], vw[PG][4][VW];
        float ks[PG][2], vs[PG][2];
        bool mapped[PG];
        const int pos0 = b * PG * kPageRows;
        bool whole = pos0 + PG * kPageRows - 1 <= least;
#pragma unroll
        for (int p = 0; p < PG; ++p) {
            mapped[p] = entry[p] >= 0 && entry[p] < a.n_pages;
            whole = whole && mapped[p];
            if (mapped[p]) {
                const size_t at = (size_t)entry[p] * kPageRows * w + (size_t)it.head * kHeadDim * F::kBytes;
#pragma unroll
                for (int r = 0; r < 2; ++r) load_words<KW>(a.k, at + (g + 8 * r) * w + 16 * c * F::kBytes, kw[p][r]);
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    load_words<VW>(a.v, at + (2 * c + (r & 1) + 8 * (r >> 1)) * w + 8 * g * F::kBytes, vw[p][r]);
                if constexpr (FMT == TIE_KV_INT8) {
                    const size_t s = ((size_t)entry[p] * a.n_kv_head + it.head) * kPageRows + g;
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        ks[p][r] = __ldg(a.ks + s + 8 * r);
                        vs[p][r] = __ldg(a.vs + s + 8 * r);
                    }
                }
            } else {
#pragma unroll
                for (int r = 0; r < 2; ++r) {
#pragma unroll
                    for (int i = 0; i < KW; ++i) kw[p][r][i] = 0u;
                    ks[p][r] = vs[p][r] = 0.f;
                }
#pragma unroll
                for (int r = 0; r < 4; ++r)
#pragma unroll
                    for (int i = 0; i < VW; ++i) vw[p][r][i] = 0u;
            }
        }
        bool odd = false;
        if (b + 1 < b1) entries(b + 1);
        // scores of keys g, g + 8 of each page: s[n][p][e], e / 2 the key, e % 2 the column
        float s[NT][PG][4], s_small[NT][PG][4];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int p = 0; p < PG; ++p)
#pragma unroll
                for (int e = 0; e < 4; ++e) s[n][p][e] = s_small[n][p][e] = 0.f;
#pragma unroll
        for (int k2 = 0; k2 < 2; ++k2) {           // two k steps of 16 dims
            uint32_t fa[2][PG][T][4];
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int p = 0; p < PG; ++p) F::keys(kw[p], 2 * k2 + h, fa[h][p]);
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                uint4 u[3];
#pragma unroll
                for (int e = 0; e < 3; ++e) u[e] = qs[((n * 2 + k2) * 3 + e) * 32 + lane];
                const uint32_t x0[3] = {u[0].x, u[1].x, u[2].x}, x1[3] = {u[0].y, u[1].y, u[2].y};
                const uint32_t y0[3] = {u[0].z, u[1].z, u[2].z}, y1[3] = {u[0].w, u[1].w, u[2].w};
#pragma unroll
                for (int p = 0; p < PG; ++p) {
                    small_products<T>(s_small[n][p], fa[0][p], x0, x1);
                    small_products<T>(s_small[n][p], fa[1][p], y0, y1);
                    main_product(s[n][p], fa[0][p][0], x0, x1);
                    main_product(s[n][p], fa[1][p][0], y0, y1);
                }
            }
        }
        // values that no row of the item sees are zero; one that is not finite and that only
        // some rows see is left to add_odd
        if (!whole) {
#pragma unroll
            for (int p = 0; p < PG; ++p)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int pos = pos0 + p * kPageRows + 2 * c + (r & 1) + 8 * (r >> 1);
                    if (pos > most) {
#pragma unroll
                        for (int i = 0; i < VW; ++i) vw[p][r][i] = 0u;
                    } else if (FMT != TIE_KV_INT8 && pos > least) {
#pragma unroll
                        for (int i = 0; i < VW; ++i) {
                            uint32_t& x = vw[p][r][i];
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
        float alpha[NT][2];
        uint32_t pb[NT][PG][2][3];     // the weights as B operands: [keys below 8, others][term]
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
            for (int p = 0; p < PG; ++p)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float& x = s[n][p][e];
                    x += s_small[n][p][e];
                    if constexpr (FMT == TIE_KV_INT8) x *= ks[p][e >> 1];
                    if (!whole && (!mapped[p] || pos0 + p * kPageRows + g + 8 * (e >> 1) > last[n][e & 1])) x = -INFINITY;
                    mx[e & 1] = fmaxf(mx[e & 1], x);
                }
            float from[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
#pragma unroll
                for (int o = 4; o < 32; o <<= 1) mx[e] = fmaxf(mx[e], __shfl_xor_sync(kAll, mx[e], o));
                const float m_new = fmaxf(st.m[n][e], mx[e]);
                from[e] = m_new == -INFINITY ? 0.f : m_new;
                alpha[n][e] = ex2_ftz(st.m[n][e] - from[e]);
                st.m[n][e] = m_new;
                st.l[n][e] *= alpha[n][e];
            }
#pragma unroll
            for (int p = 0; p < PG; ++p) {
                float w4[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float x = s[n][p][e];
                    w4[e] = kWeight * ex2_ftz(x - from[e & 1]);
                    st.l[n][e & 1] += w4[e];
                    if constexpr (FMT == TIE_KV_INT8) {
                        // (a scale of a key that the row does not see may be anything)
                        const bool seen = whole || (mapped[p] && pos0 + p * kPageRows + g + 8 * (e >> 1) <= last[n][e & 1]);
                        w4[e] = seen ? w4[e] * vs[p][e >> 1] : 0.f;
                    }
                }
                uint32_t x[3];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    split3(w4[2 * h], w4[2 * h + 1], x);
#pragma unroll
                    for (int e = 0; e < 3; ++e) pb[n][p][h][e] = transposed(x[e]);
                }
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            uint32_t fv[PG][T][4];
#pragma unroll
            for (int p = 0; p < PG; ++p) F::values(vw[p], i, fv[p]);
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                float d[4] = {};
#pragma unroll
                for (int p = 0; p < PG; ++p) small_products<T>(d, fv[p], pb[n][p][0], pb[n][p][1]);
#pragma unroll
                for (int p = 0; p < PG; ++p) main_product(d, fv[p][0], pb[n][p][0], pb[n][p][1]);
#pragma unroll
                for (int e = 0; e < 4; ++e) st.o[n][i][e] = fmaf(st.o[n][i][e], alpha[n][e & 1], d[e]);
            }
        }
        if constexpr (FMT != TIE_KV_INT8) {
            if (__any_sync(kAll, odd)) {
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    float more[2][8] = {};
                    add_odd<FMT>(a, it, max(pos0, least + 1), min(pos0 + PG * kPageRows, most + 1), last[n][0], last[n][1],
                                 8 * g, more[0], more[1]);
#pragma unroll
                    for (int i = 0; i < 4; ++i)
#pragma unroll
                        for (int e = 0; e < 4; ++e) st.o[n][i][e] += more[e & 1][2 * i + (e >> 1)];
                }
            }
        }
    }
}

// bytes of a warp's Q operands
template <int NT>
constexpr int kQBytes = NT * 2 * 3 * 32 * (int)sizeof(uint4);

template <int FMT, int NT>
__global__ void __launch_bounds__(kThreads, NT <= 2 ? 2 : 1) shared_kernel(const __grid_constant__ SharedArgs a, int which) {
    using F = Format<FMT>;
    pdl_trigger();
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ ScheduleScratch<kThreads> scratch;
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5, g = lane >> 2, c = lane & 3;
    const Line& line = a.line[which];
    uint4* qs = reinterpret_cast<uint4*>(smem) + (size_t)warp * (kQBytes<NT> / sizeof(uint4));
    long long* base = reinterpret_cast<long long*>(smem + kWarps * kQBytes<NT>);
    build_base(a, line.u0, line.u1, base, &scratch, t);
    const int n_units = line.u1 - line.u0;
    const long long total = base[n_units], share = share_of(line, total);
    const int me = blockIdx.x * kWarps + warp;
    long long x = me * share;
    const long long end = min(x + share, total);
    int u = x < end ? owner_of<long long>(base, n_units, x) : 0;
    while (x < end) {
        while (base[u + 1] <= x) ++u;  // (units without rows have no places)
        const UnitShape s = unit_shape(a, line.u0 + u);
        const int places = unit_places(s, line);
        const long long in = x - base[u], item = in / places;
        const int off = (int)(in - item * places);
        const int stop = (int)min((long long)places, off + (end - x));
        const long long first = x - off;           // the item's first place
        x += stop - off;
        const int b0 = max(off - 1, 0), b1 = stop - 1;
        if (b1 <= b0) continue;
        Item it;
        it.own = line.u0 + u >= a.n_group;
        it.row0 = s.row0;
        it.rows = s.rows;
        it.head = (int)(item % a.n_kv_head);
        it.i0 = (int)(item / a.n_kv_head) * 8 * NT;
        it.ctx = s.ctx;
        it.keys = s.keys;
        it.table = it.own ? a.table + (size_t)(line.u0 + u - a.n_group) * a.width : a.ptable + (size_t)u * a.pwidth;
        // Q, scaled, in three terms, as B operands: column g, the lane's four dims of each k step
        __syncwarp();
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const int i = it.i0 + 8 * n + g;
            const float* q = a.q + (size_t)it.row(a, i) * a.ldq + it.q_head(a, i) * kHeadDim + 16 * c;
            float y[16];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float4 v = __ldg(reinterpret_cast<const float4*>(q) + j);
                y[4 * j] = v.x * a.scale2; y[4 * j + 1] = v.y * a.scale2; y[4 * j + 2] = v.z * a.scale2; y[4 * j + 3] = v.w * a.scale2;
            }
#pragma unroll
            for (int k2 = 0; k2 < 2; ++k2) {
                uint32_t z[4][3];
#pragma unroll
                for (int h = 0; h < 4; ++h) {      // k step 2 k2 + h / 2, register h % 2
                    const int d = 8 * k2 + 4 * (h >> 1) + (h & 1) * (3 - F::kApart);
                    split3(y[d], y[d + F::kApart], z[h]);
                }
#pragma unroll
                for (int e = 0; e < 3; ++e)
                    qs[((n * 2 + k2) * 3 + e) * 32 + lane] = make_uint4(z[0][e], z[1][e], z[2][e], z[3][e]);
            }
        }
        __syncwarp();
        WarpState<FMT, NT> st;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int e = 0; e < 2; ++e) { st.m[n][e] = -INFINITY; st.l[n][e] = 0.f; }
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) st.o[n][i][e] = 0.f;
        }
        run_steps<FMT, NT>(a, it, b0, b1, qs, lane, st);
        // where the result goes: out, the rows' own place, or a part of this warp's
        const int w_first = (int)((first + 1) / share), w_last = (int)((first + places - 1) / share);
        const bool all = w_first == w_last;
        const size_t slot = (2 * (size_t)me + (me == w_first)) * (8 * NT);
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
#pragma unroll
                for (int o = 4; o < 32; o <<= 1) st.l[n][e] += __shfl_xor_sync(kAll, st.l[n][e], o);
                const int in_item = 8 * n + 2 * c + e, i = it.i0 + in_item;
                if (i >= it.rows) continue;
                const size_t row = it.row(a, i), at = row * a.n_head + it.q_head(a, i);
                float f = 1.f, *to;
                if (all && a.n_group == 0) {
                    f = st.l[n][e] == 0.f ? 0.f : 1.f / st.l[n][e];
                    to = a.out + row * a.ldo + it.q_head(a, i) * kHeadDim;
                } else {
                    to = all ? a.whole_o[it.own] + at * kHeadDim : line.part_o + (slot + in_item) * kHeadDim;
                    float* ml = all ? a.whole_ml[it.own] + 2 * at : line.part_ml + 2 * (slot + in_item);
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
    }
    // (nothing above needs another kernel's results, but what waits for this kernel waits
    // for the one before it too)
    pdl_wait();
}

// ------------------------------------------------------------------ the join --
// What a row's parts are, and where: `n` of them from `o`, `ml` on, in steps; part 0 of a cut
// item lies in its warp's second place, the others in their warps' first ones.
struct Source {
    const float *o, *ml;
    int n;
    size_t step;                       // rows of parts from part 0 to part 1, ...
    size_t first;                      // from part 0 to part 1
    __device__ __forceinline__ size_t row(int k) const { return k == 0 ? 0 : first + (size_t)(k - 1) * step; }
};

__device__ __forceinline__ Source source_of(const SharedArgs& a, const long long* base, int u, const UnitShape& s, int i, int row,
                                            int h, bool own) {
    Source z{};
    const Line& l = a.line[own];
    const int per = 8 * l.nt, places = unit_places(s, l);
    const long long item = (long long)(i / per) * a.n_kv_head + h / a.group;
    const long long origin = base[l.u0], total = base[l.u1] - origin, share = share_of(l, total);
    const long long first = base[u] - origin + item * places;
    const int w0 = (int)((first + 1) / share), w1 = (int)((first + places - 1) / share);
    if (w0 == w1) {
        const size_t at = (size_t)row * a.n_head + h;
        z.o = a.whole_o[own] + at * kHeadDim;
        z.ml = a.whole_ml[own] + 2 * at;
        z.n = 1;
    } else {
        const size_t at = (2 * (size_t)w0 + 1) * per + i % per;
        z.o = l.part_o + at * kHeadDim;
        z.ml = l.part_ml + 2 * at;
        z.n = w1 - w0 + 1;
        z.first = per;                 // slots 2 w0 + 1, 2 w0 + 2, 2 w0 + 4, ...
        z.step = 2 * (size_t)per;
    }
    return z;
}

// A warp adds parts k0, k0 + dk, ... of a source to what it has of a row: lane l dims 2 l, 2 l + 1.
struct RowSum {
    float m, l, x, y;
};
__device__ __forceinline__ void add_parts(RowSum& r, const Source& z, int k0, int dk, int lane) {
    constexpr int kAhead = 4;
    for (int k = k0; k < z.n; k += kAhead * dk) {
        float2 ml[kAhead], v[kAhead];
        float m = r.m;
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            ml[j] = make_float2(-INFINITY, 0.f);
            v[j] = make_float2(0.f, 0.f);
            if (k + j * dk < z.n) {
                const size_t at = z.row(k + j * dk);
                ml[j] = __ldcg(reinterpret_cast<const float2*>(z.ml + 2 * at));
                v[j] = __ldcg(reinterpret_cast<const float2*>(z.o + at * kHeadDim) + lane);
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

// A row and query head by a warp, or by all warps of the CTA where there are few rows (and
// many parts of each, then).
template <bool WIDE>
__global__ void __launch_bounds__(kThreads) shared_join_kernel(const __grid_constant__ SharedArgs a) {
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ ScheduleScratch<kThreads> scratch;
    __shared__ RowSum s_sum[kWarps][32];
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
    const int n_units = a.n_group + a.n_seq;
    long long* base = reinterpret_cast<long long*>(smem);
    int* starts = reinterpret_cast<int*>(base + n_units + 1);        // the rows' sequences are looked for here
    int* groups = starts + a.n_seq + 1;
    for (int i = t; i <= a.n_seq; i += kThreads) starts[i] = __ldg(a.row_start + i);
    for (int i = t; i <= a.n_group && a.n_group; i += kThreads) groups[i] = __ldg(a.gstart + i);
    build_base(a, 0, n_units, base, &scratch, t);
    pdl_wait();
    const long long pairs = (long long)a.rows * a.n_head;
    for (long long at = WIDE ? blockIdx.x : (long long)blockIdx.x * kWarps + warp; at < pairs;
         at += WIDE ? gridDim.x : (long long)gridDim.x * kWarps) {
        const int row = (int)(at / a.n_head), h = (int)(at % a.n_head);
        const int q = owner_of<int>(starts, a.n_seq, row);
        const UnitShape s = unit_shape(a, a.n_group + q);
        if (!s.rows || row < s.row0 || row >= s.row0 + s.tokens) continue;
        const Source own = source_of(a, base, a.n_group + q, s, (row - s.row0) * a.group + h % a.group, row, h, true);
        Source shared{};
        if (a.n_group) {
            const int u = owner_of<int>(groups, a.n_group, q);
            const UnitShape p = unit_shape(a, u);
            if (p.rows && q >= groups[u] && q < groups[u + 1] && row >= p.row0 && row < p.row0 + p.tokens)
                shared = source_of(a, base, u, p, (row - p.row0) * a.group + h % a.group, row, h, false);
        } else if (own.n == 1) {
            continue;                  // written already
        }
        RowSum r{-INFINITY, 0.f, 0.f, 0.f};
        add_parts(r, own, WIDE ? warp : 0, WIDE ? kWarps : 1, lane);
        add_parts(r, shared, WIDE ? warp : 0, WIDE ? kWarps : 1, lane);
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
                    const RowSum z = s_sum[v][lane];
                    f = ex2_ftz(z.m - from);
                    r.l = fmaf(z.l, f, r.l);
                    r.x = fmaf(z.x, f, r.x);
                    r.y = fmaf(z.y, f, r.y);
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
constexpr int kMaxCtas = 2;            // CTAs of shared_kernel on an SM
int most_warps(int sms) { return sms * kMaxCtas * kWarps; }

// floats of the workspace: parts of two lines, and the whole items of two sources
size_t part_floats(int sms) { return (size_t)2 * most_warps(sms) * 32 * (kHeadDim + 2); }
size_t workspace_floats(int sms, long long pairs) { return 2 * part_floats(sms) + (size_t)2 * pairs * (kHeadDim + 2); }

using Kernel = void (*)(SharedArgs, int);
template <int FMT>
Kernel kernel_of(int nt) {
    return nt == 1 ? shared_kernel<FMT, 1> : nt == 2 ? shared_kernel<FMT, 2> : shared_kernel<FMT, 4>;
}
template <int FMT>
int pages_of(int nt) {
    return nt == 1 ? kPages<FMT, 1> : nt == 2 ? kPages<FMT, 2> : kPages<FMT, 4>;
}

}  // namespace
}  // namespace tie

using namespace tie;

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
                                             float* out, int ldo, void* workspace, size_t workspace_bytes, void* stream) {
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
    a.q = q; a.ldq = ldq; a.n_head = n_head; a.group = n_head / n_kv_head; a.n_kv_head = n_kv_head;
    a.k = k_pages; a.v = v_pages; a.ks = k_scales; a.vs = v_scales; a.n_pages = n_pages;
    a.table = page_table; a.width = pages_per_seq; a.row_start = row_start; a.ctx = ctx_lens;
    a.n_seq = n_seq; a.max_new = max_new; a.rows = rows;
    a.ptable = prefix_table; a.pwidth = pages_per_prefix; a.plen = prefix_lens; a.gstart = group_start; a.n_group = n_group;
    a.scale2 = (float)((double)scale * 1.4426950408889634);
    a.out = out; a.ldo = ldo;
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
    }
    // rows that share keys, at most of a sequence and on average of a group: the items' height
    auto height = [](long long most) { return most <= 8 ? 1 : most <= 16 ? 2 : 4; };
    const long long per_seq = (long long)max_new * a.group, per_group = n_group ? ((long long)rows * a.group - 1) / n_group + 1 : 0;
    const int nt[2] = {n_group ? height(per_group) : 0, height(per_seq)};
    a.one_line = n_group && nt[0] == nt[1];
    for (int i = 0; i < 2; ++i) {
        Line& l = a.line[i];
        l.nt = nt[i] ? nt[i] : nt[1];
        l.pages = q8 ? pages_of<TIE_KV_INT8>(l.nt) : kv_format == TIE_KV_BF16 ? pages_of<TIE_KV_BF16>(l.nt) : pages_of<TIE_KV_F32>(l.nt);
        l.u0 = i ? n_group : 0;
        l.u1 = i ? n_group + n_seq : n_group;
        l.warps = sms * (l.nt <= 2 ? kMaxCtas : 1) * kWarps;
    }
    if (a.one_line) {
        a.line[0].u1 = n_group + n_seq;
        a.line[1] = a.line[0];
    }
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const size_t most_units = (size_t)2 * kOpsMaxSeqs + 1;
    bool first = true;
    for (int i = 0; i < 2; ++i) {
        const Line& l = a.line[i];
        if (l.u1 == l.u0 || (i == 1 && a.one_line)) continue;
        Kernel kernel = q8 ? kernel_of<TIE_KV_INT8>(l.nt) : kv_format == TIE_KV_BF16 ? kernel_of<TIE_KV_BF16>(l.nt) : kernel_of<TIE_KV_F32>(l.nt);
        const size_t q_bytes = (size_t)kWarps * (l.nt == 1 ? kQBytes<1> : l.nt == 2 ? kQBytes<2> : kQBytes<4>);
        const size_t smem = q_bytes + (size_t)(l.u1 - l.u0 + 1) * sizeof(long long);
        // (always the most that any call wants: calls on other threads set it too)
        if (smem > 32 * 1024)
            TIE_OP_CU(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                           (int)(q_bytes + most_units * sizeof(long long))));
        const dim3 grid((unsigned)(l.warps / kWarps));
        if (first) kernel<<<grid, kThreads, smem, st>>>(a, i);
        else TIE_OP_CU(launch_pdl(kernel, grid, dim3(kThreads), smem, st, a, i));
        TIE_OP_CU(cudaGetLastError());
        ++op_launches;
        first = false;
    }
    const size_t units = (size_t)n_group + n_seq;
    const size_t smem = (units + 1) * sizeof(long long) + (units + 2) * sizeof(int);
    const bool wide = pairs <= 8LL * sms;
    auto* join = wide ? shared_join_kernel<true> : shared_join_kernel<false>;
    if (smem > 32 * 1024)
        TIE_OP_CU(cudaFuncSetAttribute(join, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       (int)(most_units * (sizeof(long long) + sizeof(int)) + 64)));
    const long long ctas = wide ? pairs : (pairs + kWarps - 1) / kWarps;
    TIE_OP_CU(launch_pdl(join, dim3((unsigned)(ctas < 8LL * sms ? ctas : 8LL * sms)), dim3(kThreads), smem, st, a));
    ++op_launches;
    return MODEL_OK;
}
