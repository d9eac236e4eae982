// ops_beam.cu -- beam search's selection over beams and vocabulary.
//
// The reference's only selection is the greedy argmax (src/main.c:274-287).
// Here, for each request of `beams` rows of logits x_b with running scores
// score_b,
//
//   total(b, v) = score_b + (x_bv - logsumexp_v x_b)
//
// and the `beams` largest totals are kept (ties: the lowest b * vocab + v); a
// finished beam offers only (eos, score_b). The logits are read once: a CTA
// per (row, slice of the vocabulary) keeps the slice's maximum, its sum of
// exponentials and its `beams` largest logits; a CTA per request then joins
// the slices and picks. Bound by the reading of the logits.
//
// Totals decide an order, so they are formed in double: exponentials in fp32
// (x - max is exact where the terms are large), their sum, the logarithm and
// the totals in double. Which thread adds which element depends on its index
// in the row alone, not on the row's address, so equal rows have equal sums
// and their ties are real ones.
#include "ops.h"

#include <climits>
#include <cmath>

namespace tie {
namespace {

constexpr int kMaxBeams = 16;
constexpr int kScanThreads = 256, kScanWarps = kScanThreads / 32;
constexpr int kBatch = 8;              // elements per thread and pass
constexpr int kPickThreads = 256, kPickWarps = kPickThreads / 32;
constexpr unsigned kAll = 0xffffffffu;

// 2^x, x <= 0 here (ex2.approx.ftz: relative error about 2^-22)
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
constexpr float kLog2e = 1.4426950408889634f;

// What a slice leaves: its maximum, its sum of exp(x - maximum), and its k
// largest logits with their indices, best first (lower index first on ties).
struct Partials {
    float* max;     // [rows][slices]
    double* sum;    // [rows][slices]
    float* val;     // [rows][slices][k]
    int* idx;       // [rows][slices][k]
};

__device__ __forceinline__ bool better(float v, int i, float w, int j) { return v > w || (v == w && i < j); }

__global__ void __launch_bounds__(kScanThreads)
beam_scan_kernel(const float* __restrict__ logits, int ldl, const int32_t* __restrict__ done, int vocab, int slices,
                 int slice_len, int k, Partials out) {
    pdl_trigger();
    __shared__ float s_val[kScanWarps * kMaxBeams];
    __shared__ int s_idx[kScanWarps * kMaxBeams];
    __shared__ float s_max[kScanWarps];
    __shared__ double s_sum[kScanWarps];
    const int row = blockIdx.x / slices, slice = blockIdx.x % slices;
    if (done && done[row]) return;      // a finished beam's logits are not looked at
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
    const int lo = slice * slice_len, hi = min(lo + slice_len, vocab);
    const float* x = logits + (size_t)row * ldl;

    float m = -INFINITY;
    double sum = 0.0;
    // the warp's list: lane j < k holds its (j + 1)th best
    float lv = -INFINITY;
    int li = INT_MAX;
    float worst = -INFINITY;            // lane k - 1's entry
    int worst_i = INT_MAX;
    for (int i0 = lo; i0 < hi; i0 += kScanThreads * kBatch) {
        float v[kBatch];
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
            const int i = i0 + u * kScanThreads + t;
            v[u] = i < hi ? __ldcs(x + i) : -INFINITY;
        }
        float top = v[0];
#pragma unroll
        for (int u = 1; u < kBatch; ++u) top = fmaxf(top, v[u]);   // NaN never wins
        if (top > m) {
            sum *= (double)ex2((m - top) * kLog2e);                // m = -inf: 0
            m = top;
        }
        if (m > -INFINITY) {
            float part = 0.f;
#pragma unroll
            for (int u = 0; u < kBatch; ++u) part += v[u] == v[u] ? ex2((v[u] - m) * kLog2e) : 0.f;
            sum += (double)part;
        }
        if (__any_sync(kAll, worst_i == INT_MAX || top > worst)) {
#pragma unroll 1
            for (int u = 0; u < kBatch; ++u) {
                const int i = i0 + u * kScanThreads + t;
                const float xv = fmaxf(u == 0 ? v[0] : u == 1 ? v[1] : u == 2 ? v[2] : u == 3 ? v[3]
                                       : u == 4 ? v[4] : u == 5 ? v[5] : u == 6 ? v[6] : v[7], -INFINITY);
                unsigned todo = __ballot_sync(kAll, i < hi && better(xv, i, worst, worst_i));
                while (todo) {
                    const int src = __ffs(todo) - 1;
                    todo &= todo - 1;
                    const float cv = __shfl_sync(kAll, xv, src);
                    const int ci = __shfl_sync(kAll, i, src);
                    if (!better(cv, ci, worst, worst_i)) continue;
                    const bool stays = better(lv, li, cv, ci);
                    const int rank = __popc(__ballot_sync(kAll, stays && lane < k));
                    const float uv = __shfl_up_sync(kAll, lv, 1);
                    const int ui = __shfl_up_sync(kAll, li, 1);
                    if (lane == rank) { lv = cv; li = ci; }
                    else if (lane > rank) { lv = uv; li = ui; }
                    worst = __shfl_sync(kAll, lv, k - 1);
                    worst_i = __shfl_sync(kAll, li, k - 1);
                }
            }
        }
    }
    // the CTA's maximum and sum
    float wm = m;
#pragma unroll
    for (int o = 16; o; o >>= 1) wm = fmaxf(wm, __shfl_xor_sync(kAll, wm, o));
    double ws = m > -INFINITY ? sum * (double)ex2((m - wm) * kLog2e) : 0.0;
#pragma unroll
    for (int o = 16; o; o >>= 1) ws += __shfl_xor_sync(kAll, ws, o);
    if (lane == 0) { s_max[warp] = wm; s_sum[warp] = ws; }
    if (lane < k) { s_val[warp * k + lane] = lv; s_idx[warp * k + lane] = li; }
    __syncthreads();
    const size_t at = (size_t)row * slices + slice;
    if (t == 0) {
        float M = s_max[0];
        for (int w = 1; w < kScanWarps; ++w) M = fmaxf(M, s_max[w]);
        double S = 0.0;
        for (int w = 0; w < kScanWarps; ++w)
            if (s_max[w] > -INFINITY) S += s_sum[w] * exp((double)s_max[w] - (double)M);
        out.max[at] = M;
        out.sum[at] = S;
    }
    // each of the warps' entries finds its place among all of them
    if (t < kScanWarps * k) {
        const float v = s_val[t];
        const int i = s_idx[t];
        int rank = 0;
        for (int j = 0; j < kScanWarps * k; ++j)
            rank += better(s_val[j], s_idx[j], v, i) || (s_val[j] == v && s_idx[j] == i && j < t);
        if (rank < k) {
            out.val[at * k + rank] = v;
            out.idx[at * k + rank] = i;     // INT_MAX: the slice has fewer than k elements
        }
    }
}

__global__ void __launch_bounds__(kPickThreads)
beam_pick_kernel(Partials in, int slices, int k, int vocab, int eos, const float* __restrict__ scores,
                 const int32_t* __restrict__ done, int32_t* __restrict__ next, int32_t* __restrict__ parent,
                 float* __restrict__ scores_out, int32_t* __restrict__ done_out) {
    pdl_wait();
    extern __shared__ double s_total[];                    // [k * slices * k] candidates' totals
    __shared__ double s_base[kMaxBeams];                   // score - logsumexp, or NaN
    __shared__ float s_score[kMaxBeams];
    __shared__ int s_done[kMaxBeams];
    __shared__ double w_total[kPickWarps];
    __shared__ long long w_flat[kPickWarps];
    __shared__ int w_at[kPickWarps];
    __shared__ double p_total[kMaxBeams];
    __shared__ long long p_flat[kMaxBeams];
    const int q = blockIdx.x, t = threadIdx.x, lane = t & 31, warp = t >> 5;
    const size_t row0 = (size_t)q * k;
    if (t < k) {
        s_done[t] = done ? done[row0 + t] != 0 : 0;
        s_score[t] = scores[row0 + t];
    }
    __syncthreads();
    for (int b = warp; b < k; b += kPickWarps) {
        if (s_done[b]) continue;
        const size_t at = (row0 + b) * slices;
        float M = -INFINITY;
        for (int s = lane; s < slices; s += 32) M = fmaxf(M, in.max[at + s]);
#pragma unroll
        for (int o = 16; o; o >>= 1) M = fmaxf(M, __shfl_xor_sync(kAll, M, o));
        double S = 0.0;
        for (int s = lane; s < slices; s += 32)
            if (in.max[at + s] > -INFINITY) S += in.sum[at + s] * exp((double)in.max[at + s] - (double)M);
#pragma unroll
        for (int o = 16; o; o >>= 1) S += __shfl_xor_sync(kAll, S, o);
        // a row with no finite logit has no normaliser (NaN)
        if (lane == 0) s_base[b] = M > -INFINITY && M < INFINITY ? (double)M + log(S) : (double)NAN;
    }
    __syncthreads();
    const int per = slices * k, n = k * per;
    auto token_of = [&](int c) {       // candidate c's token, INT_MAX for none
        const int b = c / per, j = c % per;
        if (s_done[b]) return j == 0 ? eos : INT_MAX;
        const double base = (double)s_score[b] - s_base[b];
        // a beam without a finite score: every candidate ties at -inf, the lowest tokens are its best
        if (!(base > (double)-INFINITY)) return j < k && j < vocab ? j : INT_MAX;
        return in.idx[(row0 + b) * per + j];
    };
    for (int c = t; c < n; c += kPickThreads) {
        const int b = c / per;
        double v = (double)-INFINITY;
        if (s_done[b]) v = (double)s_score[b];
        else if (c % per < per) {
            const double base = (double)s_score[b] - s_base[b];
            if (base > (double)-INFINITY)
                v = (double)s_score[b] + ((double)in.val[(row0 + b) * per + c % per] - s_base[b]);
        }
        if (!(v > (double)-INFINITY)) v = (double)-INFINITY;       // NaN counts as -inf
        s_total[c] = v;
    }
    __syncthreads();
    // k rounds of the best remaining candidate
    for (int round = 0; round < k; ++round) {
        double bv = (double)-INFINITY;
        long long bf = LLONG_MAX;
        int bc = -1;
        for (int c = t; c < n; c += kPickThreads) {
            const double v = s_total[c];
            if (!(v >= bv)) continue;                              // taken candidates are NaN
            const int tok = token_of(c);
            if (tok == INT_MAX) continue;
            const long long f = (long long)(c / per) * vocab + tok;
            if (v > bv || f < bf) { bv = v; bf = f; bc = c; }
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) {
            const double ov = __shfl_xor_sync(kAll, bv, o);
            const long long of = __shfl_xor_sync(kAll, bf, o);
            const int oc = __shfl_xor_sync(kAll, bc, o);
            if (ov > bv || (ov == bv && of < bf)) { bv = ov; bf = of; bc = oc; }
        }
        if (lane == 0) { w_total[warp] = bv; w_flat[warp] = bf; w_at[warp] = bc; }
        __syncthreads();
        if (t == 0) {
            for (int w = 1; w < kPickWarps; ++w)
                if (w_total[w] > bv || (w_total[w] == bv && w_flat[w] < bf)) { bv = w_total[w]; bf = w_flat[w]; bc = w_at[w]; }
            p_total[round] = bv;
            p_flat[round] = bf;
            if (bc >= 0) s_total[bc] = (double)NAN;
        }
        __syncthreads();
    }
    // a beam's best child stays in its place, the others take the free places in order
    if (t == 0) {
        unsigned taken = 0, heirs = 0;
        for (int i = 0; i < k; ++i) {
            const int b = (int)(p_flat[i] / vocab);
            if (!(taken >> b & 1)) { taken |= 1u << b; heirs |= 1u << i; }
        }
        for (int i = 0; i < k; ++i) {
            const int b = (int)(p_flat[i] / vocab), tok = (int)(p_flat[i] % vocab);
            int place = b;
            if (!(heirs >> i & 1)) {
                place = __ffs((int)~taken) - 1;
                taken |= 1u << place;
            }
            next[row0 + place] = tok;
            parent[row0 + place] = (int)row0 + b;
            scores_out[row0 + place] = (float)p_total[i];
            if (done_out) done_out[row0 + place] = s_done[b] || tok == eos;
        }
    }
}

// Slices of the vocabulary per row: about four CTAs per SM in all, each of at
// least one pass of its threads (2048 logits).
int slices_for(long long rows, int vocab, int sms) {
    const int most = (vocab + kScanThreads * kBatch - 1) / (kScanThreads * kBatch);
    const long long want = (4LL * sms + rows - 1) / rows;
    return (int)(want < 1 ? 1 : want > most ? most : want);
}

// candidates one pick holds in shared memory
constexpr int kMaxCandidates = 5120;

int slices_of(int n_req, int beams, int vocab, int sms) {
    const int s = slices_for((long long)n_req * beams, vocab, sms);
    const int cap = kMaxCandidates / (beams * beams);
    return s < cap ? s : cap;
}

size_t scratch_bytes(int n_req, int beams, int slices) {
    const size_t at = (size_t)n_req * beams * slices;
    return at * (sizeof(double) + sizeof(float)) + at * beams * (sizeof(float) + sizeof(int));
}

bool shape_ok(int n_req, int beams, int vocab) {
    return n_req > 0 && beams > 0 && vocab > 0;
}

}  // namespace
}  // namespace tie

using namespace tie;

extern "C" size_t tie_beam_select_workspace(int n_req, int beams, int vocab) {
    if (!shape_ok(n_req, beams, vocab) || beams > kMaxBeams) return 0;
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) { cudaGetLastError(); return 0; }
    return scratch_bytes(n_req, beams, slices_of(n_req, beams, vocab, sm_count(dev)));
}

extern "C" model_status tie_beam_select(const float* logits, int ldl, const float* scores, const int32_t* done,
                                        int n_req, int beams, int vocab, int eos_id, int32_t* next, int32_t* parent,
                                        float* scores_out, int32_t* done_out, void* workspace, size_t workspace_bytes,
                                        void* stream) {
    if (!logits || !scores || !next || !parent || !scores_out || !workspace) return MODEL_ERR_ARG;
    if (!shape_ok(n_req, beams, vocab) || ldl < vocab || eos_id >= vocab) return MODEL_ERR_ARG;
    if ((done || done_out) && eos_id < 0) return MODEL_ERR_ARG;
    if (!aligned16(workspace)) return MODEL_ERR_ARG;
    if (beams > kMaxBeams || n_req > kOpsMaxSeqs) return MODEL_ERR_CAPACITY;
    OnDeviceOf dev(next);
    if (dev.status() != MODEL_OK) return dev.status();
    const int slices = slices_of(n_req, beams, vocab, sm_count(dev.device()));
    if (workspace_bytes < scratch_bytes(n_req, beams, slices)) return MODEL_ERR_CAPACITY;
    const size_t at = (size_t)n_req * beams * slices;
    Partials p;
    p.sum = static_cast<double*>(workspace);
    p.max = reinterpret_cast<float*>(p.sum + at);
    p.val = p.max + at;
    p.idx = reinterpret_cast<int*>(p.val + at * beams);
    const int len = (vocab + slices - 1) / slices;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    beam_scan_kernel<<<(unsigned)at, kScanThreads, 0, st>>>(logits, ldl, done, vocab, slices, len, beams, p);
    TIE_OP_CU(cudaGetLastError());
    TIE_OP_CU(launch_pdl(beam_pick_kernel, dim3((unsigned)n_req), dim3(kPickThreads),
                         (size_t)slices * beams * beams * sizeof(double), st, p, slices, beams, vocab, eos_id, scores,
                         done, next, parent, scores_out, done_out));
    return MODEL_OK;
}
