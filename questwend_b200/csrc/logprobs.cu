// Log probabilities of given tokens, the entropy of each row's distribution and its most probable tokens, from 32-bit logits in
// one pass over them.
//
//     lp(t) = x_t - m - ln S,   S = sum exp(x - m),   H = ln S - U / S,   U = sum exp(x - m) (x - m),   m = max x
//
// A block takes a segment of a row, LP_SEG logits, and holds it in registers: the segment's maximum, sums and largest logits come
// from there, and memory is read once.  A segment leaves (m, S, U) and its `top` largest as a sorted list; a second kernel joins a
// row's segments (sums relative to the largest m, lists by merging).  Segments are cut by the row alone, so a row's result
// does not depend on how many rows there are.
// Of equal logits the one with the lower id is larger.  A NaN is no candidate for the list and makes the row's numbers NaN.
#include "common.cuh"

#define LP_THREADS 256
#define LP_PER_THREAD 32
#define LP_SEG (LP_THREADS * LP_PER_THREAD)
#define LP_MAX_TOP 64

// Larger logits first, of equal ones the lower id (id < 0: nothing).
__device__ __forceinline__ bool lp_before(float a, int ia, float b, int ib) { return ib < 0 ? ia >= 0 : (ia >= 0 && (a > b || (a == b && ia < ib))); }

__device__ __forceinline__ void lp_warp_best(float& v, int& i) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const float ov = __shfl_xor_sync(0xffffffffu, v, o);
        const int oi = __shfl_xor_sync(0xffffffffu, i, o);
        if (lp_before(ov, oi, v, i)) { v = ov; i = oi; }
    }
}

__global__ void __launch_bounds__(LP_THREADS)
lp_segments_kernel(const float* __restrict__ logits, float* __restrict__ sums, float* __restrict__ best, int* __restrict__ best_id, int V,
                   int segs, int top) {
    pdl_wait();
    pdl_launch_dependents();
    __shared__ float scratch[32], win_v[LP_THREADS / 32];
    __shared__ int win_i[LP_THREADS / 32];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const long long row = blockIdx.y;
    const int seg = blockIdx.x, first = seg * LP_SEG;
    const float* x = logits + row * V;
    float v[LP_PER_THREAD];
    float m = -INFINITY;
#pragma unroll
    for (int e = 0; e < LP_PER_THREAD; ++e) {
        const int i = first + e * LP_THREADS + tid;
        v[e] = i < V ? x[i] : -INFINITY;
        m = fmaxf(m, v[e]);
    }
    m = warp_max(m);
    if (lane == 0) scratch[warp] = m;
    __syncthreads();
    for (int w = 0; w < LP_THREADS / 32; ++w) m = fmaxf(m, scratch[w]);
    float S = 0.f, U = 0.f;
#pragma unroll
    for (int e = 0; e < LP_PER_THREAD; ++e) {
        const float d = v[e] - m, p = v[e] == -INFINITY ? 0.f : __expf(d);
        S += p;
        if (p > 0.f) U += p * d;
    }
    S = block_sum(S, scratch);
    U = block_sum(U, scratch);
    const long long at = row * segs + seg;
    if (tid == 0) {
        sums[at * 3] = m;
        sums[at * 3 + 1] = S;
        sums[at * 3 + 2] = U;
    }
    // the `top` largest, one after the other: everyone's largest that is behind the last one found
    float last = INFINITY;
    int last_i = -1;
    for (int k = 0; k < top; ++k) {
        float bv = -INFINITY;
        int bi = -1;
#pragma unroll
        for (int e = 0; e < LP_PER_THREAD; ++e) {
            const int i = first + e * LP_THREADS + tid;
            const bool open = i < V && v[e] == v[e] && (last_i < 0 || lp_before(last, last_i, v[e], i));
            if (open && lp_before(v[e], i, bv, bi)) { bv = v[e]; bi = i; }
        }
        lp_warp_best(bv, bi);
        __syncthreads();
        if (lane == 0) { win_v[warp] = bv; win_i[warp] = bi; }
        __syncthreads();
        bv = win_v[0];
        bi = win_i[0];
        for (int w = 1; w < LP_THREADS / 32; ++w)
            if (lp_before(win_v[w], win_i[w], bv, bi)) { bv = win_v[w]; bi = win_i[w]; }
        if (tid == 0) { best[at * top + k] = bv; best_id[at * top + k] = bi; }
        if (bi < 0) {
            for (int r = k + 1 + tid; r < top; r += LP_THREADS) { best[at * top + r] = -INFINITY; best_id[at * top + r] = -1; }
            break;
        }
        last = bv;
        last_i = bi;
    }
}

// One warp a row joins its segments.
__global__ void __launch_bounds__(128)
lp_join_kernel(const float* __restrict__ logits, const int* __restrict__ tokens, const float* __restrict__ sums, const float* __restrict__ best,
               const int* __restrict__ best_id, float* __restrict__ logprob, float* __restrict__ entropy, int* __restrict__ top_ids,
               float* __restrict__ top_lps, int rows, int V, int segs, int top) {
    pdl_wait();
    pdl_launch_dependents();
    const int lane = threadIdx.x & 31;
    const long long row = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
    if (row >= rows) return;
    const float* mine = sums + row * segs * 3;
    float m = -INFINITY;
    for (int s = lane; s < segs; s += 32) m = fmaxf(m, mine[s * 3]);
    m = warp_max(m);
    float S = 0.f, U = 0.f;
    for (int s = lane; s < segs; s += 32) {
        const float ms = mine[s * 3], Ss = mine[s * 3 + 1], Us = mine[s * 3 + 2];
        if (Ss != 0.f) {                                    // a segment of nothing but -infinity adds nothing
            const float f = expf(ms - m);
            S += Ss * f;
            U += (Us + Ss * (ms - m)) * f;
        }
    }
    S = warp_sum(S);
    U = warp_sum(U);
    const float lnS = logf(S);
    if (lane == 0) {
        const int t = tokens[row];
        logprob[row] = (t >= 0 && t < V) ? (logits[row * V + t] - m) - lnS : __uint_as_float(0x7fffffffu);
        entropy[row] = lnS - U / S;
    }
    float last = INFINITY;
    int last_i = -1;
    for (int k = 0; k < top; ++k) {
        float bv = -INFINITY;
        int bi = -1;
        for (int s = lane; s < segs; s += 32) {
            const float* lv = best + (row * segs + s) * top;
            const int* li = best_id + (row * segs + s) * top;
            for (int r = 0; r < top; ++r) {                 // the first of the list that is behind the last one found
                if (li[r] < 0) break;
                if (last_i < 0 || lp_before(last, last_i, lv[r], li[r])) {
                    if (lp_before(lv[r], li[r], bv, bi)) { bv = lv[r]; bi = li[r]; }
                    break;
                }
            }
        }
        lp_warp_best(bv, bi);
        if (lane == 0) {
            top_ids[row * top + k] = bi;
            top_lps[row * top + k] = bi < 0 ? __uint_as_float(0x7fffffffu) : (bv - m) - lnS;
        }
        if (bi >= 0) { last = bv; last_i = bi; }
    }
}

extern "C" int qwb_logprobs_segments(int V) { return (int)(((long long)V + LP_SEG - 1) / LP_SEG); }

// scratch: rows x segments x (3 + top) floats, then rows x segments x top ints
extern "C" int qwb_logprobs(const float* logits, const int* tokens, float* logprob, float* entropy, int* top_ids, float* top_lps, float* scratch,
                            int rows, int V, int top, cudaStream_t stream) {
    if (rows <= 0) return 0;
    if (V <= 0 || V > 2000000000 || top < 0 || top > LP_MAX_TOP || top > V)
        return qwb_fail(QWB_ERR_ARG, "token_logprobs: 0 to %d alternatives of a vocabulary of at least as many: top=%d V=%d", LP_MAX_TOP, top, V);
    if (rows > 65535) return qwb_fail(QWB_ERR_ARG, "token_logprobs: at most 65535 rows in a call, not %d", rows);
    const int segs = qwb_logprobs_segments(V);
    float* best = scratch + (size_t)rows * segs * 3;
    int* best_id = reinterpret_cast<int*>(best + (size_t)rows * segs * top);
    qwb_launch(lp_segments_kernel, dim3(segs, rows), LP_THREADS, 0, stream, logits, scratch, best, best_id, V, segs, top);
    qwb_launch(lp_join_kernel, dim3((rows + 3) / 4), 128, 0, stream, logits, tokens, scratch, best, best_id, logprob, entropy, top_ids, top_lps, rows, V,
               segs, top);
    return qwb_check_launch("token_logprobs");
}
