// ops_cache.cu -- the tables and the rows of a paged K/V cache, on the GPU: the
// page plan of a ragged batch, the store of new key and value rows through its
// slot map, and the reordering of beams' rows.
//
// The reference keeps one sequence's rows in one contiguous block
// (src/kv_cache.c:150-190) and has no batches, pages or beams; page_table.h is
// the host-side allocator these operators agree with (pages of 16 positions, a
// stack of free pages).
#include "ops.h"

#include <cooperative_groups.h>
#include <cuda_bf16.h>

#include <climits>
#include <mutex>

namespace tie {

int sm_count(int device) {
    static std::mutex mu;
    static int known[64] = {0};
    if (device < 0 || device >= 64) return 148;
    std::lock_guard<std::mutex> lock(mu);
    if (!known[device]) {
        int n = 0;
        if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, device) != cudaSuccess) {
            cudaGetLastError();
            return 148;
        }
        known[device] = n;
    }
    return known[device];
}

namespace {

namespace cg = cooperative_groups;

// ------------------------------------------------------------------ page plan --
// Latency bound (a few KB in, three int32 per row out), so it is one launch of
// one cluster: every CTA scans all lengths for itself (4 per thread at most,
// from L2) and then writes its share of the table entries and rows. One
// cluster, because n_free_out may be n_free: the cluster barrier puts every
// CTA's read of it before the one write. 256 sequences of one row: 6.0 us on the
// GPU, of which an empty launch has 2; 72,000 rows of 1500 sequences: 10.3 us,
// bound by the rows' instructions on the cluster's 16 SMs.
constexpr int kPlanThreads = 1024;
constexpr int kPlanPerThread = kOpsMaxSeqs / kPlanThreads;

struct PlanArgs {
    const int32_t *ctx, *fresh;
    int n_seq;
    int32_t* table;
    int width, n_pages;
    const int32_t* free_pages;
    int max_free;
    const int32_t* n_free;
    int32_t *n_free_out, *row_start, *seq_of, *pos_of, *slot_of;
    int max_rows;
    int32_t* status;
};

__device__ __forceinline__ long long warp_scan_ll(long long v, int lane) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long u = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += u;
    }
    return v;
}

__global__ void __launch_bounds__(kPlanThreads) page_plan_kernel(PlanArgs a) {
    extern __shared__ int sm[];
    int* s_row = sm;                      // [n_seq + 1] first row of each sequence
    int* s_need = sm + a.n_seq + 1;       // [n_seq + 1] pages assigned before each sequence
    int* s_ctx = s_need + a.n_seq + 1;    // [n_seq]
    __shared__ long long w_new[32], w_need[32];
    __shared__ int s_bad;                 // 1: a negative length, 2: a sequence beyond its table
    cg::cluster_group cluster = cg::this_cluster();
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
    if (t == 0) s_bad = 0;
    __syncthreads();

    const int n_free = a.n_free ? *a.n_free : 0;
    const long long cap = (long long)a.width * kPageRows;
    // per thread: kPlanPerThread consecutive sequences
    int nw[kPlanPerThread], nd[kPlanPerThread];
    long long sum_new = 0, sum_need = 0;
    int bad = 0;
    const int per = (a.n_seq + kPlanThreads - 1) / kPlanThreads;
#pragma unroll
    for (int k = 0; k < kPlanPerThread; ++k) {
        const int s = t * per + k;
        nw[k] = nd[k] = 0;
        if (k < per && s < a.n_seq) {
            const int c = a.ctx[s], n = a.fresh[s];
            s_ctx[s] = c;
            if (c < 0 || n < 0) bad |= 1;
            else if ((long long)c + n > cap) bad |= 2;
            else {
                nw[k] = n;
                nd[k] = a.n_free ? (int)(((long long)c + n + kPageRows - 1) / kPageRows -
                                         ((long long)c + kPageRows - 1) / kPageRows)
                                 : 0;
            }
        }
        sum_new += nw[k];
        sum_need += nd[k];
    }
    if (bad) atomicOr(&s_bad, bad);
    const long long in_new = warp_scan_ll(sum_new, lane), in_need = warp_scan_ll(sum_need, lane);
    if (lane == 31) { w_new[warp] = in_new; w_need[warp] = in_need; }
    __syncthreads();
    if (warp == 0) {
        w_new[lane] = warp_scan_ll(w_new[lane], lane);
        w_need[lane] = warp_scan_ll(w_need[lane], lane);
    }
    __syncthreads();
    const long long total_new = w_new[31], total_need = w_need[31];
    int st = MODEL_OK;
    if ((s_bad & 1) || n_free < 0 || n_free > a.max_free) st = MODEL_ERR_ARG;
    else if (s_bad || total_new > a.max_rows || total_need > n_free) st = MODEL_ERR_CAPACITY;
    const bool ok = st == MODEL_OK;
    if (ok) {
        long long rn = in_new - sum_new + (warp ? w_new[warp - 1] : 0);
        long long rp = in_need - sum_need + (warp ? w_need[warp - 1] : 0);
#pragma unroll
        for (int k = 0; k < kPlanPerThread; ++k) {
            const int s = t * per + k;
            if (k < per && s < a.n_seq) {
                s_row[s] = (int)rn;
                s_need[s] = (int)rp;
                rn += nw[k];
                rp += nd[k];
            }
        }
        if (t == 0) { s_row[a.n_seq] = (int)total_new; s_need[a.n_seq] = (int)total_need; }
    } else {
        for (int s = t; s <= a.n_seq; s += kPlanThreads) s_row[s] = s_need[s] = 0;
    }
    // every CTA has read n_free
    cluster.sync();
    const int rank = (int)cluster.block_rank(), ctas = (int)cluster.num_blocks();
    const int g = rank * kPlanThreads + t, G = ctas * kPlanThreads;
    if (g == 0) {
        *a.status = st;
        if (a.n_free) *a.n_free_out = n_free - (ok ? (int)total_need : 0);
    }
    for (int s = g; s <= a.n_seq; s += G) a.row_start[s] = s_row[s];
    // the last sequence s with base[s] <= x
    auto owner = [&](const int* base, int x) {
        int lo = 0, hi = a.n_seq;
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (base[mid] <= x) lo = mid;
            else hi = mid;
        }
        return lo;
    };
    // assigned page x of the call is free page n_free - 1 - x
    const int need = s_need[a.n_seq], rows = s_row[a.n_seq];
    for (long long at = g; at < need; at += G) {
        const int x = (int)at, s = owner(s_need, x);
        const int have = (int)(((long long)s_ctx[s] + kPageRows - 1) / kPageRows);
        a.table[(size_t)s * a.width + have + (x - s_need[s])] = a.free_pages[n_free - 1 - x];
    }
    // A warp takes a stretch of rows, 32 at a time and two such groups at once (a row is
    // two loads that depend on one another, so latency counts). The sequence of its
    // first row is found by a search with all lanes, the others by walking on.
    constexpr int kGroups = 2;
    const long long groups = ((long long)a.max_rows + 31) / 32, per_warp = (groups + (G >> 5) - 1) / (G >> 5);
    const long long w0 = (g >> 5) * per_warp, w1 = min(w0 + per_warp, groups);
    int from = -1;                                 // the sequence of the last row so far
    for (long long w = w0; w < w1; w += kGroups) {
        int seq[kGroups], pos[kGroups], page[kGroups];
#pragma unroll
        for (int x = 0; x < kGroups; ++x) {
            seq[x] = pos[x] = page[x] = -1;
            if (w + x >= w1 || 32 * (w + x) >= rows) continue;
            const int first = (int)(32 * (w + x)), r = min(first + lane, rows - 1);
            if (from < 0) {
                int n = a.n_seq;                   // s_row[from] <= first, and not at from + n
                from = 0;
                while (n > 1) {
                    const int step = (n + 31) / 32;    // lane l looks at from + l * step
                    const bool below = lane * step < n && s_row[from + lane * step] <= first;
                    const int at = 31 - __clz(__ballot_sync(0xffffffffu, below));
                    from += at * step;
                    n = min(step, n - at * step);
                }
            }
            int lo = from;
            // (by a search of its own where many without rows lie between)
            bool there = s_row[lo + 1] > r;
#pragma unroll 1
            for (int k = 0; k < 4 && !there; ++k) there = s_row[++lo + 1] > r;
            if (!there) lo = owner(s_row, r);
            from = __shfl_sync(0xffffffffu, lo, 31);
            if (r != first + lane) continue;
            seq[x] = lo;
            const int c = s_ctx[lo], have = (int)(((long long)c + kPageRows - 1) / kPageRows);
            pos[x] = c + (r - s_row[lo]);
            const int j = pos[x] / kPageRows;
            // the entries other threads assign above are taken from the free
            // list itself, not from the table
            page[x] = a.n_free && j >= have ? a.free_pages[n_free - 1 - (s_need[lo] + j - have)]
                                                : a.table[(size_t)lo * a.width + j];
        }
#pragma unroll
        for (int x = 0; x < kGroups; ++x) {
            const long long r = 32 * (w + x) + lane;
            if (w + x >= w1 || r >= a.max_rows) continue;
            a.seq_of[r] = seq[x];
            a.pos_of[r] = pos[x];
            a.slot_of[r] = page[x] >= 0 && page[x] < a.n_pages ? page[x] * kPageRows + pos[x] % kPageRows : -1;
        }
    }
}

// The widest cluster of plan CTAs that the current device runs, asked once per device:
// 16 on B200 (72,000 rows of 1500 sequences: 14.4 us with 8 CTAs, 10.3 with 16).
// Also raises the kernel's shared memory to the most that any call wants.
int widest_plan(int device) {
    static std::mutex mu;
    static int known[64] = {0};
    std::lock_guard<std::mutex> lock(mu);
    if (device >= 0 && device < 64 && known[device]) return known[device];
    const int smem = 3 * (kOpsMaxSeqs + 1) * (int)sizeof(int);
    int widest = 8, fit = 0;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(16);
    cfg.blockDim = dim3(kPlanThreads);
    cfg.dynamicSmemBytes = smem;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 16;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (cudaFuncSetAttribute(page_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) == cudaSuccess &&
        cudaFuncSetAttribute(page_plan_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) == cudaSuccess &&
        cudaOccupancyMaxActiveClusters(&fit, page_plan_kernel, &cfg) == cudaSuccess && fit > 0)
        widest = 16;
    cudaGetLastError();
    if (device >= 0 && device < 64) known[device] = widest;
    return widest;
}

// ---------------------------------------------------------------- row store --
// Memory bound: a thread moves 8 elements of a key row and the same 8 of the
// value row, four 16-byte loads in flight. bf16 pages round to nearest even (an
// error of 2^-8 of the element at most, once). 16,391 rows of 16 heads into bf16
// pages: 32.9 us, 6.1 TB/s of the 6.5 that a copy has; 256 rows of 12 heads, fp32:
// 2.2 us on the GPU.
constexpr int kStoreThreads = 256;

__device__ __forceinline__ uint32_t bf16x2(float lo, float hi) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}

template <bool BF16>
__device__ __forceinline__ void store8(void* pages, size_t at, float4 a, float4 b) {
    if constexpr (BF16) {
        *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(pages) + at) =
            make_uint4(bf16x2(a.x, a.y), bf16x2(a.z, a.w), bf16x2(b.x, b.y), bf16x2(b.z, b.w));
    } else {
        float4* p = reinterpret_cast<float4*>(static_cast<float*>(pages) + at);
        p[0] = a;
        p[1] = b;
    }
}

template <bool BF16>
__global__ void __launch_bounds__(kStoreThreads)
kv_store_kernel(const float* __restrict__ k, const float* __restrict__ v, int ld, const int32_t* __restrict__ slots,
                long long n, int per_row, long long n_slots, void* __restrict__ k_pages, void* __restrict__ v_pages) {
    const long long i = (long long)blockIdx.x * kStoreThreads + threadIdx.x;
    if (i >= n) return;
    const int r = (int)(i / per_row), c = (int)(i % per_row) * 8;
    const size_t from = (size_t)r * ld + c;
    const float4 k0 = __ldg(reinterpret_cast<const float4*>(k + from));
    const float4 k1 = __ldg(reinterpret_cast<const float4*>(k + from) + 1);
    const float4 v0 = __ldg(reinterpret_cast<const float4*>(v + from));
    const float4 v1 = __ldg(reinterpret_cast<const float4*>(v + from) + 1);
    const int slot = __ldg(slots + r);
    if (slot < 0 || slot >= n_slots) return;   // a row behind the last sequence, or without a page
    const size_t to = (size_t)slot * (size_t)(per_row * 8) + c;
    store8<BF16>(k_pages, to, k0, k1);
    store8<BF16>(v_pages, to, v0, v1);
}

// ------------------------------------------------------------------ reorder --
// Memory bound. A unit is one logical page of one request in one layer, keys
// or values; a thread takes one 16-byte vector of it through all beams: it
// loads the vector from every moved beam's parent before it stores any, so a
// permutation of beams (a swap, a cycle) needs no second buffer and no barrier
// -- no other thread touches the same vectors. 24 requests of 5 beams, 337
// positions, 12 layers of 12 heads, fp32: 317 us, 7.2 TB/s (part of the parents'
// rows comes from L2); 2 requests of 4 beams, 37 positions: 8.0 us, the latency of
// the lists and the table before the rows.
constexpr int kReorderThreads = 256;
constexpr int kMaxBeams = 16;

struct ReorderArgs {
    uint4 *k, *v;
    int n_layer;
    size_t layer_vecs;                 // 16-byte vectors from a layer to the next
    int n_pages, row_vecs;             // vectors of one row
    const int32_t *table, *parent, *first, *length;
    int width, n_req, beams;
};

// pages of request r that hold rows to move: [*lo, *hi)
__device__ __forceinline__ bool reorder_range(const ReorderArgs& a, int r, int* lo, int* hi) {
    int f = a.first[r], n = a.length[r];
    if (f < 0) f = 0;
    if (n > a.width * (long long)kPageRows) n = a.width * kPageRows;
    bool moved = false;
    for (int b = 0; b < a.beams; ++b) {
        const int p = a.parent[r * a.beams + b] - r * a.beams;
        moved |= p != b && p >= 0 && p < a.beams;
    }
    if (!moved || f >= n) return false;
    *lo = f / kPageRows;
    *hi = (n + kPageRows - 1) / kPageRows;
    return true;
}

template <int BEAMS>
__global__ void __launch_bounds__(kReorderThreads) kv_reorder_kernel(ReorderArgs a) {
    extern __shared__ int s_base[];    // [n_req + 1] pages to move before each request
    __shared__ int w_sum[kReorderThreads / 32];
    __shared__ int s_src[kMaxBeams], s_dst[kMaxBeams];
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
    const int per = (a.n_req + kReorderThreads - 1) / kReorderThreads;
    int mine = 0;
    for (int k = 0; k < per; ++k) {
        const int r = t * per + k;
        int lo, hi;
        if (r < a.n_req && reorder_range(a, r, &lo, &hi)) mine += hi - lo;
    }
    int in = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, in, o);
        if (lane >= o) in += u;
    }
    if (lane == 31) w_sum[warp] = in;
    __syncthreads();
    int base = in - mine;
    for (int w = 0; w < warp; ++w) base += w_sum[w];
    for (int k = 0; k < per; ++k) {
        const int r = t * per + k;
        if (r >= a.n_req) break;
        int lo, hi;
        s_base[r] = base;
        if (reorder_range(a, r, &lo, &hi)) base += hi - lo;
        if (r == a.n_req - 1) s_base[a.n_req] = base;
    }
    __syncthreads();
    const long long pages = s_base[a.n_req], whole = pages * 2 * a.n_layer;
    const int vecs = a.row_vecs * kPageRows;
    // few pages: each is cut into pieces, so that every CTA has something to move
    const int pieces = whole > 0 ? (int)max(1ll, min(gridDim.x / whole, (long long)(vecs / kReorderThreads))) : 1;
    const int piece_vecs = (vecs + pieces - 1) / pieces;
    const long long units = whole * pieces;
    for (long long u = blockIdx.x; u < units; u += gridDim.x) {
        const int piece = (int)(u % pieces), pg = (int)(u / pieces % pages), lv = (int)(u / pieces / pages);
        int lo = 0, hi = a.n_req;
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (s_base[mid] <= pg) lo = mid;
            else hi = mid;
        }
        const int r = lo;
        int f = max(a.first[r], 0);
        const int len = (int)min((long long)a.length[r], a.width * (long long)kPageRows);
        const int j = f / kPageRows + pg - s_base[r];
        __syncthreads();   // the previous unit's entries are no longer read
        if (t < a.beams) {
            const int s = r * a.beams + t, p = a.parent[s] - r * a.beams;
            const int to = a.table[(size_t)s * a.width + j];
            int from = -1;
            if (p != t && p >= 0 && p < a.beams) from = a.table[(size_t)(s - t + p) * a.width + j];
            const bool move = from >= 0 && from < a.n_pages && to >= 0 && to < a.n_pages && from != to;
            s_src[t] = move ? from : -1;
            s_dst[t] = to;
        }
        __syncthreads();
        uint4* pool = (lv & 1 ? a.v : a.k) + (size_t)(lv >> 1) * a.layer_vecs;
        const int v0 = max(max(f - j * kPageRows, 0) * a.row_vecs, piece * piece_vecs);
        const int v1 = min(min(len - j * kPageRows, kPageRows) * a.row_vecs, (piece + 1) * piece_vecs);
        for (int i = v0 + t; i < v1; i += kReorderThreads) {
            uint4 x[BEAMS];
#pragma unroll
            for (int b = 0; b < BEAMS; ++b)
                if (b < a.beams && s_src[b] >= 0) x[b] = __ldcs(pool + (size_t)s_src[b] * vecs + i);
#pragma unroll
            for (int b = 0; b < BEAMS; ++b)
                if (b < a.beams && s_src[b] >= 0) __stcs(pool + (size_t)s_dst[b] * vecs + i, x[b]);
        }
    }
}

}  // namespace
}  // namespace tie

using namespace tie;

extern "C" model_status tie_page_plan(const int32_t* ctx_lens, const int32_t* new_lens, int n_seq, int32_t* page_table,
                                      int pages_per_seq, int n_pages, const int32_t* free_pages, int max_free,
                                      const int32_t* n_free, int32_t* n_free_out, int32_t* row_start, int32_t* seq_of,
                                      int32_t* pos_of, int32_t* slot_of, int max_rows, int32_t* status, void* stream) {
    if (!ctx_lens || !new_lens || !page_table || !row_start || !seq_of || !pos_of || !slot_of || !status)
        return MODEL_ERR_ARG;
    if (n_seq <= 0 || pages_per_seq <= 0 || n_pages <= 0 || max_rows <= 0) return MODEL_ERR_ARG;
    // n_free says whether there is a free list: an empty one has no address
    if (n_free ? (!n_free_out || max_free < 0 || (max_free && !free_pages)) : (free_pages || n_free_out)) return MODEL_ERR_ARG;
    if (n_seq > kOpsMaxSeqs || n_pages > kOpsMaxPages || pages_per_seq > kOpsMaxPages / 2) return MODEL_ERR_CAPACITY;
    OnDeviceOf dev(row_start);
    if (dev.status() != MODEL_OK) return dev.status();
    PlanArgs a{ctx_lens, new_lens, n_seq, page_table, pages_per_seq, n_pages, free_pages, max_free, n_free, n_free_out,
               row_start, seq_of, pos_of, slot_of, max_rows, status};
    // a CTA per 4096 rows (four of each thread), at most a cluster
    const int ctas = (int)min((long long)widest_plan(dev.device()), (max_rows + 4095LL) / 4096);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)ctas);
    cfg.blockDim = dim3(kPlanThreads);
    cfg.dynamicSmemBytes = 3 * (size_t)(n_seq + 1) * sizeof(int);
    cfg.stream = static_cast<cudaStream_t>(stream);
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)ctas;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    TIE_OP_CU(cudaLaunchKernelEx(&cfg, page_plan_kernel, a));
    ++op_launches;
    return MODEL_OK;
}

extern "C" model_status tie_kv_store(const float* k, const float* v, int ld, const int32_t* slots, int rows,
                                     void* k_pages, void* v_pages, int kv_format, int n_pages, int n_kv_head,
                                     void* stream) {
    if (!k_pages || !v_pages || rows < 0) return MODEL_ERR_ARG;
    if (rows && (!k || !v || !slots)) return MODEL_ERR_ARG;   // arrays without rows have no address
    if (!pool_shape_ok(kv_format, n_pages, n_kv_head)) return MODEL_ERR_ARG;
    const int w = n_kv_head * kHeadDim;
    if (ld < w || (ld & 3) || !aligned16(k) || !aligned16(v) || !aligned16(k_pages) || !aligned16(v_pages))
        return MODEL_ERR_ARG;
    if (rows == 0) return MODEL_OK;
    OnDeviceOf dev(k_pages);
    if (dev.status() != MODEL_OK) return dev.status();
    const long long n = (long long)rows * (w / 8), n_slots = (long long)n_pages * kPageRows;
    const long long blocks = (n + kStoreThreads - 1) / kStoreThreads;
    if (blocks > INT_MAX) return MODEL_ERR_CAPACITY;
    auto* kernel = kv_format == TIE_KV_BF16 ? kv_store_kernel<true> : kv_store_kernel<false>;
    kernel<<<(unsigned)blocks, kStoreThreads, 0, static_cast<cudaStream_t>(stream)>>>(k, v, ld, slots, n, w / 8,
                                                                                      n_slots, k_pages, v_pages);
    TIE_OP_CU(cudaGetLastError());
    ++op_launches;
    return MODEL_OK;
}

extern "C" model_status tie_kv_reorder(void* k_pages, void* v_pages, int kv_format, int n_layer, size_t layer_stride,
                                       int n_pages, int n_kv_head, const int32_t* page_table, int pages_per_seq,
                                       const int32_t* parent, const int32_t* first, const int32_t* length, int n_req,
                                       int beams, void* stream) {
    if (!k_pages || !v_pages || !page_table || !parent || !first || !length) return MODEL_ERR_ARG;
    if (!pool_shape_ok(kv_format, n_pages, n_kv_head) || n_layer <= 0 || pages_per_seq <= 0 || n_req <= 0 || beams <= 0)
        return MODEL_ERR_ARG;
    if (beams > kMaxBeams || n_req > kOpsMaxSeqs || pages_per_seq > kOpsMaxPages / 2) return MODEL_ERR_CAPACITY;
    const size_t size = kv_format == TIE_KV_BF16 ? 2 : 4;
    const size_t row = (size_t)n_kv_head * kHeadDim;
    if (!aligned16(k_pages) || !aligned16(v_pages) || (layer_stride * size) % 16) return MODEL_ERR_ARG;
    if (n_layer > 1 && layer_stride < row * kPageRows * (size_t)n_pages) return MODEL_ERR_ARG;
    // the pages a call can touch are counted in int32
    if ((long long)n_req * pages_per_seq > INT_MAX) return MODEL_ERR_CAPACITY;
    if (beams == 1) return MODEL_OK;   // one beam is its own parent
    OnDeviceOf dev(k_pages);
    if (dev.status() != MODEL_OK) return dev.status();
    ReorderArgs a{};
    a.k = static_cast<uint4*>(k_pages);
    a.v = static_cast<uint4*>(v_pages);
    a.n_layer = n_layer;
    a.layer_vecs = layer_stride * size / 16;
    a.n_pages = n_pages;
    a.row_vecs = (int)(row * size / 16);
    a.table = page_table;
    a.parent = parent;
    a.first = first;
    a.length = length;
    a.width = pages_per_seq;
    a.n_req = n_req;
    a.beams = beams;
    auto* kernel = beams <= 4 ? kv_reorder_kernel<4> : beams <= 8 ? kv_reorder_kernel<8> : kv_reorder_kernel<16>;
    const unsigned grid = (unsigned)sm_count(dev.device()) * (2048 / kReorderThreads);
    kernel<<<grid, kReorderThreads, (size_t)(n_req + 1) * sizeof(int), static_cast<cudaStream_t>(stream)>>>(a);
    TIE_OP_CU(cudaGetLastError());
    ++op_launches;
    return MODEL_OK;
}
