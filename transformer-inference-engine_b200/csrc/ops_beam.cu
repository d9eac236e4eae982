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
// the slices and picks. 96 requests of 6 beams over 50,257 tokens: 37 us (29 the scan,
// 8 the picking), against 17.7 for the logits' bytes. All CTAs are one wave, and each has
// its pass, its bound, a second look and its lists one after the other, so memory idles
// in the later ones (46 % of its rate, 37 % of the issue slots). One request of 4 beams:
// 8.7 us on the GPU, two kernels' latency.
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
constexpr int kBatch = 8;              // elements a thread loads at a time
constexpr int kScanResident = 8;       // CTAs per SM (64 KB of loads in flight)
constexpr int kPickThreads = 512, kPickWarps = kPickThreads / 64;   // pairs of warps
constexpr int kMaxVocab = 1 << 30;     // indices of a row stay in int32 with room for a step
constexpr int kMaxSlices = 32;         // a lane of the picking warps for each
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

// floats (no NaN) as unsigned numbers of the same order, all above 0
__device__ __forceinline__ unsigned order_key(float v) {
    const unsigned b = __float_as_uint(v + 0.f);              // -0 and +0 are equal
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float from_order_key(unsigned k) {
    return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}

__device__ __forceinline__ bool better(float v, int i, float w, int j) { return v > w || (v == w && i < j); }

__global__ void __launch_bounds__(kScanThreads, kScanResident)
beam_scan_kernel(const float* __restrict__ logits, int ldl, const int32_t* __restrict__ done, int vocab, int slices,
                 int slice_len, int k, Partials out) {
    pdl_trigger();
    __shared__ float s_val[kScanWarps * kMaxBeams];
    __shared__ int s_idx[kScanWarps * kMaxBeams];
    __shared__ float s_max[kScanWarps];
    __shared__ double s_sum[kScanWarps];
    __shared__ float s_group[2 * kScanWarps];
    __shared__ int s_count;
    static_assert(2 * kScanWarps >= kMaxBeams, "a bound for every list length");
    const int row = blockIdx.x / slices, slice = blockIdx.x % slices;
    if (done && done[row]) return;      // a finished beam's logits are not looked at
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
    const int lo = slice * slice_len, hi = min(lo + slice_len, vocab);
    const float* x = logits + (size_t)row * ldl;

    // One pass over the slice: a thread's maximum and its sum of exponentials.
    float m = -INFINITY;
    double sum = 0.0;
    for (int i0 = lo; i0 < hi; i0 += kScanThreads * kBatch) {
        float v[kBatch];
        if (i0 + kScanThreads * kBatch <= hi) {
#pragma unroll
            for (int u = 0; u < kBatch; ++u) v[u] = __ldg(x + i0 + u * kScanThreads + t);
        } else {
#pragma unroll
            for (int u = 0; u < kBatch; ++u) {
                const int i = i0 + u * kScanThreads + t;
                v[u] = i < hi ? __ldg(x + i) : -INFINITY;
            }
        }
        float top = -INFINITY;
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
            v[u] = fmaxf(v[u], -INFINITY);                         // NaN counts as -inf
            top = fmaxf(top, v[u]);
        }
        if (top > m) {
            sum *= (double)ex2((m - top) * kLog2e);                // m = -inf: 0
            m = top;
        }
        if (m > -INFINITY) {
            float part = 0.f;
#pragma unroll
            for (int u = 0; u < kBatch; ++u) part += ex2((v[u] - m) * kLog2e);
            sum += (double)part;
        }
    }
    // The k-th largest of the half-warps' maxima: k elements reach it, so whatever
    // is below is in no result, and few threads have something that is not.
    // (Lists kept during the pass cost more instructions than the pass: 31 million
    // for 576 rows against 9 million.)
    float gm = m;
#pragma unroll
    for (int o = 8; o; o >>= 1) gm = fmaxf(gm, __shfl_xor_sync(kAll, gm, o));
    if ((lane & 15) == 0) s_group[2 * warp + (lane >> 4)] = gm;
    if (t == 0) s_count = 0;
    __syncthreads();
    float bound;
    {
        const float mine = lane < 2 * kScanWarps ? s_group[lane] : -INFINITY;
        int above = 0;
#pragma unroll
        for (int g = 0; g < 2 * kScanWarps; ++g) above += s_group[g] > mine || (s_group[g] == mine && g < lane);
        bound = __shfl_sync(kAll, mine, __ffs(__ballot_sync(kAll, lane < 2 * kScanWarps && above == k - 1)) - 1);
    }
    // the warp's list: lane j < k holds its (j + 1)th best
    float lv = -INFINITY;
    int li = INT_MAX;
    float worst = -INFINITY;            // lane k - 1's entry
    int worst_i = INT_MAX;
    unsigned lanes = __ballot_sync(kAll, m >= bound);
    while (lanes) {
        // the elements of one lane's thread, 128 at a time
        const int src = __ffs(lanes) - 1;
        lanes &= lanes - 1;
        constexpr int kAhead = 4, kStride = 32 * kScanThreads;
        for (int i0 = lo + 32 * warp + src; i0 < hi; i0 += kAhead * kStride) {
            float own[kAhead];
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                const int i = i0 + lane * kScanThreads + u * kStride;
                own[u] = i < hi ? fmaxf(__ldg(x + i), -INFINITY) : -INFINITY;
            }
#pragma unroll 1
            for (int u = 0; u < kAhead && i0 + u * kStride < hi; ++u) {
                const float cand = u == 0 ? own[0] : u == 1 ? own[1] : u == 2 ? own[2] : own[3];
                const int i = i0 + lane * kScanThreads + u * kStride;
                unsigned todo = __ballot_sync(kAll, i < hi && cand >= bound && better(cand, i, worst, worst_i));
                while (todo) {
                    const int at = __ffs(todo) - 1;
                    todo &= todo - 1;
                    const float cv = __shfl_sync(kAll, cand, at);
                    const int ci = __shfl_sync(kAll, i, at);
                    if (!better(cv, ci, worst, worst_i)) continue;
                    const int rank = __popc(__ballot_sync(kAll, lane < k && better(lv, li, cv, ci)));
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
    // the warps' entries side by side, in any order
    {
        const int n = __popc(__ballot_sync(kAll, lane < k && li != INT_MAX));
        int at = 0;
        if (lane == 0 && n) at = atomicAdd(&s_count, n);
        at = __shfl_sync(kAll, at, 0);
        if (lane < n) { s_val[at + lane] = lv; s_idx[at + lane] = li; }
    }
    __syncthreads();
    const size_t at = (size_t)row * slices + slice;
    if (warp == 0) {
        const float wm0 = lane < kScanWarps ? s_max[lane] : -INFINITY;
        float M = wm0;
#pragma unroll
        for (int o = kScanWarps / 2; o; o >>= 1) M = fmaxf(M, __shfl_xor_sync(kAll, M, o));
        double S = wm0 > -INFINITY ? s_sum[lane] * (double)ex2((wm0 - M) * kLog2e) : 0.0;
#pragma unroll
        for (int o = kScanWarps / 2; o; o >>= 1) S += __shfl_xor_sync(kAll, S, o);
        if (lane == 0) {
            out.max[at] = M;
            out.sum[at] = S;
        }
    }
    // each finds its place among all of them
    const int count = s_count;
    for (int e = t; e < max(count, k); e += kScanThreads) {
        int rank = e;                   // fewer than k elements in the slice: no entry
        float v = -INFINITY;
        int i = INT_MAX;
        if (e < count) {
            v = s_val[e];
            i = s_idx[e];
            rank = 0;
            for (int o = 0; o < count; ++o) rank += better(s_val[o], s_idx[o], v, i);
        }
        if (rank < k) {
            out.val[at * k + rank] = v;
            out.idx[at * k + rank] = i;
        }
    }
}

__global__ void __launch_bounds__(kPickThreads)
beam_pick_kernel(Partials in, int slices, int k, int vocab, int eos, const float* __restrict__ scores,
                 const int32_t* __restrict__ done, int32_t* __restrict__ next, int32_t* __restrict__ parent,
                 float* __restrict__ scores_out, int32_t* __restrict__ done_out) {
    __shared__ double s_total[kMaxBeams * kMaxBeams];      // the beams' best, best first; NaN: none
    __shared__ int s_token[kMaxBeams * kMaxBeams];
    __shared__ long long s_flat[kMaxBeams * kMaxBeams];    // beam * vocab + token
    __shared__ float s_best[kMaxBeams * kMaxBeams];
    __shared__ double p_total[kMaxBeams];                  // the kept ones by rank
    __shared__ int p_beam[kMaxBeams], p_token[kMaxBeams];
    __shared__ float s_val[kPickWarps][kMaxSlices * kMaxBeams];
    __shared__ int s_idx[kPickWarps][kMaxSlices * kMaxBeams];
    __shared__ double s_lse[kMaxBeams];
    __shared__ float s_score[kMaxBeams];
    __shared__ int s_done[kMaxBeams];
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
    const size_t row0 = (size_t)blockIdx.x * k;
    pdl_wait();
    if (t < k) {
        s_score[t] = scores[row0 + t];
        s_done[t] = done && done[row0 + t] != 0;
        p_total[t] = (double)-INFINITY;
        p_beam[t] = t;
        p_token[t] = 0;
    }
    // two warps per beam, a lane per slice: one forms the logarithm of the sum of
    // exponentials, the other merges the slices' lists. (What a finished beam's
    // rows hold is not used.)
    for (int b = warp & (kPickWarps - 1); b < k; b += kPickWarps) {
        const size_t at = (row0 + b) * slices + lane;
        if (warp >= kPickWarps) {
            const float m = lane < slices ? in.max[at] : -INFINITY;
            const double part = lane < slices ? in.sum[at] : 0.0;
            float M = m;
#pragma unroll
            for (int o = 16; o; o >>= 1) M = fmaxf(M, __shfl_xor_sync(kAll, M, o));
            double S = m > -INFINITY ? part * (double)ex2((m - M) * kLog2e) : 0.0;
#pragma unroll
            for (int o = 16; o; o >>= 1) S += __shfl_xor_sync(kAll, S, o);
            // a row whose largest logit is infinite has no normaliser
            if (lane == 0) s_lse[b] = M > -INFINITY && M < INFINITY ? (double)M + log(S) : (double)NAN;
            continue;
        }
        for (int e = lane; e < slices * k; e += 32) {
            s_val[warp][e] = in.val[(row0 + b) * slices * k + e];
            s_idx[warp][e] = in.idx[(row0 + b) * slices * k + e];
        }
        __syncwarp();
        int head = 0;
        unsigned key = lane < slices ? order_key(s_val[warp][lane * k]) : 0u;
        int hi = lane < slices ? s_idx[warp][lane * k] : INT_MAX;
        for (int r = 0; r < k; ++r) {
            const unsigned most = __reduce_max_sync(kAll, key);
            const int first = (int)__reduce_min_sync(kAll, key == most ? (unsigned)hi : (unsigned)INT_MAX);
            if (lane == 0) { s_best[b * k + r] = from_order_key(most); s_token[b * k + r] = first; }
            if (key == most && hi == first && hi != INT_MAX) {
                ++head;
                key = head < k ? order_key(s_val[warp][lane * k + head]) : 0u;
                hi = head < k ? s_idx[warp][lane * k + head] : INT_MAX;
            }
        }
        __syncwarp();
    }
    __syncthreads();
    // the candidates' totals
    for (int c = t; c < k * k; c += kPickThreads) {
        const int b = c / k, r = c % k;
        const float score = s_score[b];
        double total = (double)score;
        int token;
        if (s_done[b]) {
            token = r == 0 ? eos : INT_MAX;
        } else if ((double)score - s_lse[b] > (double)-INFINITY) {
            token = s_token[c];
            total += (double)s_best[c] - s_lse[b];
        } else {
            // every candidate ties at -inf, the lowest tokens are its best
            token = r < vocab ? r : INT_MAX;
            total = (double)-INFINITY;
        }
        if (!(total > (double)-INFINITY)) total = (double)-INFINITY;   // NaN counts as -inf
        s_total[c] = token == INT_MAX ? (double)NAN : total;
        s_token[c] = token;
        s_flat[c] = (long long)b * vocab + token;
    }
    __syncthreads();
    // each finds its rank among all (there are always k), a warp for each
    for (int c = warp; c < k * k; c += kPickThreads / 32) {
        const double v = s_total[c];
        if (v != v) continue;
        const long long flat = s_flat[c];
        int rank = 0;
        for (int o0 = 0; o0 < k * k; o0 += 32) {
            const int o = o0 + lane;
            const bool ahead = o < k * k && (s_total[o] > v || (s_total[o] == v && s_flat[o] < flat));
            rank += __popc(__ballot_sync(kAll, ahead));
        }
        if (lane == 0 && rank < k) {
            p_total[rank] = v;
            p_beam[rank] = c / k;
            p_token[rank] = s_token[c];
        }
    }
    __syncthreads();
    // a beam's best child stays in its place, the others take the free places in order
    if (warp == 0) {
        const int b = lane < k ? p_beam[lane] : kMaxBeams + lane;
        const bool heir = __ffs((int)__match_any_sync(kAll, b)) - 1 == lane;
        const unsigned taken = __reduce_or_sync(kAll, lane < k ? 1u << b : 0u);
        const unsigned others = __ballot_sync(kAll, lane < k && !heir);
        const bool was = lane < k && s_done[b];
        if (lane < k) {
            unsigned left = ~taken;                         // the free places, lowest first
            for (int o = __popc(others & ((1u << lane) - 1)); o > 0; --o) left &= left - 1;
            const int place = heir ? b : __ffs((int)left) - 1;
            const int tok = p_token[lane];
            next[row0 + place] = tok;
            parent[row0 + place] = (int)row0 + b;
            scores_out[row0 + place] = (float)p_total[lane];
            if (done_out) done_out[row0 + place] = was || tok == eos;
        }
    }
}

// Slices of the vocabulary per row: one wave of CTAs (576 rows of 50257: 37.5 us;
// two, three and four waves 39.8, 42.3 and 44.8), each of at least one load of
// its threads (2048 logits), at most a lane each of the warp that joins them.
int slices_of(int n_req, int beams, int vocab, int sms) {
    const long long rows = (long long)n_req * beams;
    const int most = (vocab + kScanThreads * kBatch - 1) / (kScanThreads * kBatch);
    long long n = (long long)kScanResident * sms / rows;
    if (n > most) n = most;
    if (n > kMaxSlices) n = kMaxSlices;
    return n < 1 ? 1 : (int)n;
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
    if (beams > kMaxBeams || n_req > kOpsMaxSeqs || vocab > kMaxVocab) return MODEL_ERR_CAPACITY;
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
    TIE_OP_CU(launch_pdl(beam_pick_kernel, dim3((unsigned)n_req), dim3(kPickThreads), 0, st, p, slices, beams, vocab, eos_id, scores,
                         done, next, parent, scores_out, done_out));
    op_launches += 2;
    return MODEL_OK;
}
