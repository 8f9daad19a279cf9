// Log probabilities of given tokens, the entropy of each row's distribution and its most probable tokens, from 32-bit logits in
// one pass over them.
//
//     lp(t) = x_t - m - ln S,   S = sum exp(x - m),   H = ln S - U / S,   U = sum exp(x - m) (x - m),   m = max x
//
// A block takes a segment of a row, LP_SEG logits, a thread 64 of them in pieces of 16 with the next piece's loads on their way;
// it keeps a reference (a largest logit so far, or up to 8 below it), S and U relative to that, and its largest logit.  Logits are
// bounded by memory as long as a logit costs few instructions: maximum, difference, exp2 of a product, two sums are 7.
// A segment leaves (m, S, U) and each thread's largest logit, a 64th of what it read; a second kernel joins a row's sums and finds its
// `top` largest from these maxima, with a look at the few threads' logits that can be among them.  (A sorted list from every
// segment, found in its block while the others wait at the memory, took 407 us for 2,048 rows of 151,936 logits and a top of 20, where
// the sums alone take 183.)  Segments are cut by the row alone, so a row's result does not depend on how many rows there are.
// Of equal logits the one with the lower id is larger.  A NaN is no candidate for the list and makes the row's numbers NaN.
#include "common.cuh"

#include <limits.h>

#define LP_THREADS 256
#define LP_PIECE 16             // logits of a thread at a time
#define LP_PER_THREAD 64
#define LP_SEG (LP_THREADS * LP_PER_THREAD)
#define LP_MAX_TOP 64
#define LP_JOIN_THREADS 128      // of a row's end: all of 2,048 rows' ends are on the chip at once
#define LP_HELD 8               // maxima of a thread of the joining kernel that it keeps in registers: 65,536 logits' worth
#define LP_CLUSTER 16           // segments of a row that can be a cluster: 262,144 logits
#define LP_GATHER 512           // candidates of a row that shared memory holds

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

// Numbers in their order as whole ones (-0 and 0 are one; no NaN).
__device__ __forceinline__ int lp_key(float x) {
    const int b = __float_as_int(x + 0.f);
    return b < 0 ? b ^ 0x7fffffff : b;
}

// VEC: rows begin at a multiple of 16 bytes and hold a multiple of 4 logits.  A thread then holds 4 neighbouring logits of every 1,024.
template <bool VEC>
__device__ __forceinline__ int lp_index(int e, int tid) { return VEC ? (e >> 2) * (4 * LP_THREADS) + 4 * tid + (e & 3) : e * LP_THREADS + tid; }

__device__ __forceinline__ float lp_exp(float d) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(d * 1.4426950408889634f));
    return y;
}
// Sums relative to `from` as sums relative to `to`, which is not below it.  The clamp: nothing times -infinity is nothing.
__device__ __forceinline__ void lp_raise(float& S, float& U, float from, float to) {
    const float d = from - to, f = lp_exp(d);
    U = (U + S * fmaxf(d, -1e30f)) * f;
    S *= f;
}
#define LP_LOWEST -3.4028234663852886e38f       // a reference when there is none: -infinity itself would leave -infinity minus -infinity

// The end of a row, by one block.  The `top` largest: a thread takes its share of the maxima; each warp's (top / warps, rounded up)-th largest
// of its threads' largest, and the lowest of these, the bar, is at most the row's top-th largest logit, and few maxima are at or above it
// (with random logits about twice `top`); the top-th largest of those is a higher bar.  The 64 logits of the threads that reach it are read
// again and what is at or above the bar gathered in shared memory; each one's rank is how many stand before it.  Where more are there
// than fit (equal logits, orders that put the largest into few threads, fewer logits above -infinity than the bar needs) the list is found one by
// one, a pass over the row each: of 151,936 equal logits a top of 5 / 20 takes 279 / 945 us for 8 rows where random ones take 11 / 12, 1,763 / 6,174 for
// 256 (43 / 51), 2,101 / 7,092 for 2,048 (199 / 211); with 100 tokens left a top of 20 is as fast as ever, one of 64 takes 2.9 ms for 8 rows, 19 for 256.
//   held: the thread's maxima of the first segments; more: those of all segments, for the ones behind (null: there are none)
template <bool VEC, int HELD, int THREADS>
__device__ __forceinline__ void lp_finish(const float* x, int token, float m, float S, float U, const float (&held)[HELD], const float* more, float* logprob,
                                          float* entropy, int* top_ids, float* top_lps, int V, int segs, int top) {
    constexpr int WARPS = THREADS / 32;
    __shared__ float warp_t[WARPS], found_v[LP_GATHER];
    __shared__ int found_i[LP_GATHER], holders[LP_GATHER], picked[LP_GATHER], n_found, n_holders, n_picked;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int shares = segs * (LP_THREADS / THREADS);           // maxima of a thread
    const float lnS = logf(S);
    if (tid == 0) {
        *logprob = (token >= 0 && token < V) ? (x[token] - m) - lnS : __uint_as_float(0x7fffffffu);
        *entropy = lnS - U / S;
        n_found = n_holders = n_picked = 0;
    }
    if (!top) return;
    float largest = -INFINITY;
#pragma unroll
    for (int j = 0; j < HELD; ++j) largest = fmaxf(largest, held[j]);
    for (int j = HELD; j < shares; ++j) largest = fmaxf(largest, __ldcg(more + j * THREADS + tid));
    int left = lp_key(largest), kth = __reduce_max_sync(0xffffffffu, left);
    for (int k = 1; k < (top + WARPS - 1) / WARPS; ++k) {                               // take the warp's largest out, look again
        const unsigned at = __ballot_sync(0xffffffffu, left == kth);
        if (lane == __ffs(at) - 1) left = INT_MIN;
        kth = __reduce_max_sync(0xffffffffu, left);
    }
    if (lane == 0) warp_t[warp] = kth == INT_MIN ? -INFINITY : __int_as_float(kth < 0 ? kth ^ 0x7fffffff : kth);
    __syncthreads();
    float bar = warp_t[0];
#pragma unroll
    for (int w = 1; w < WARPS; ++w) bar = fminf(bar, warp_t[w]);
    if (largest >= bar) {
        auto hold = [&](int j, float y) {
            const int at = atomicAdd(&n_holders, 1);
            if (at < LP_GATHER) {
                holders[at] = j;
                found_v[at] = y;
            }
        };
#pragma unroll
        for (int j = 0; j < HELD; ++j)
            if (j < shares && held[j] >= bar) hold(j * THREADS + tid, held[j]);
        for (int j = HELD; j < shares; ++j) {
            const float y = __ldcg(more + j * THREADS + tid);
            if (y >= bar) hold(j * THREADS + tid, y);
        }
    }
    __syncthreads();
    // the top-th largest of the maxima found is a higher bar, with about half as many at or above it
    const int n_held = min(n_holders, LP_GATHER);
    for (int i = tid; i < n_held; i += THREADS) {
        const float a = found_v[i];
        int above = 0, same = 0;
        for (int j = 0; j < n_held; ++j) {
            above += found_v[j] > a;
            same += found_v[j] == a;
        }
        if (above < top && top <= above + same) warp_t[0] = a;          // whoever writes, writes the same number
    }
    __syncthreads();
    if (n_holders <= LP_GATHER) bar = warp_t[0];
    for (int i = tid; i < n_held; i += THREADS)
        if (found_v[i] >= bar) picked[atomicAdd(&n_picked, 1)] = holders[i];
    __syncthreads();
    // 64 logits of each, all threads side by side
    const int looks = n_picked * LP_PER_THREAD;
#pragma unroll 4
    for (int j = tid; j < looks; j += THREADS) {
        const int who = picked[j / LP_PER_THREAD], i = who / LP_THREADS * LP_SEG + lp_index<VEC>(j % LP_PER_THREAD, who % LP_THREADS);
        const float y = i < V ? x[i] : -INFINITY;
        if (y >= bar && i < V) {
            const int at = atomicAdd(&n_found, 1);
            if (at < LP_GATHER) {
                found_v[at] = y;
                found_i[at] = i;
            }
        }
    }
    __syncthreads();
    const int n = n_found;
    auto leave = [&](int rank, float a, int ia) {
        top_ids[rank] = ia;
        top_lps[rank] = ia < 0 ? __uint_as_float(0x7fffffffu) : (a - m) - lnS;
    };
    if (n <= LP_GATHER && n_holders <= LP_GATHER) {
        for (int i = tid; i < n; i += THREADS) {
            const float a = found_v[i];
            const int ia = found_i[i];
            int rank = 0;
            for (int j = 0; j < n; ++j) rank += lp_before(found_v[j], found_i[j], a, ia);
            if (rank < top) leave(rank, a, ia);
        }
        for (int i = n + tid; i < top; i += THREADS) leave(i, -INFINITY, -1);
        return;
    }
    // one after the other: everyone's largest that is behind the last one found
    float last = INFINITY;
    int last_i = -1;
    for (int k = 0; k < top; ++k) {
        float bv = -INFINITY;
        int bi = -1;
        for (int i = tid; i < V; i += THREADS) {
            const float y = x[i];
            const bool open = y == y && (k == 0 || lp_before(last, last_i, y, i));
            if (open && lp_before(y, i, bv, bi)) { bv = y; bi = i; }
        }
        lp_warp_best(bv, bi);
        __syncthreads();
        if (lane == 0) { found_v[warp] = bv; found_i[warp] = bi; }
        __syncthreads();
        bv = found_v[0];
        bi = found_i[0];
        for (int w = 1; w < WARPS; ++w)
            if (lp_before(found_v[w], found_i[w], bv, bi)) { bv = found_v[w]; bi = found_i[w]; }
        if (bi < 0) {                                               // no logit is left that is a number
            for (int i = k + tid; i < top; i += THREADS) leave(i, -INFINITY, -1);
            return;
        }
        if (tid == 0) leave(k, bv, bi);
        last = bv;
        last_i = bi;
    }
}

__device__ __forceinline__ float lp_remote(const float* mine, int rank) {      // this address of the cluster's `rank`th block
    uint32_t at;
    float v;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"((uint32_t)__cvta_generic_to_shared(mine)), "r"(rank));
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
    return v;
}
__device__ __forceinline__ void lp_cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// CLUSTER: a row's segments are the blocks of a cluster; the first of them takes the others' results from their shared memory and ends the
// row.  Else the results go to `sums` and `maxima` for the joining kernel.
template <bool VEC, bool CLUSTER>
__global__ void __launch_bounds__(LP_THREADS, 4)
lp_segments_kernel(const float* __restrict__ logits, float* __restrict__ sums, float* __restrict__ maxima, const int* __restrict__ tokens,
                   float* __restrict__ logprob, float* __restrict__ entropy, int* __restrict__ top_ids, float* __restrict__ top_lps, int V, int segs,
                   int top) {
    pdl_wait();
    pdl_launch_dependents();
    constexpr int WARPS = LP_THREADS / 32;
    __shared__ float warp_m[WARPS], warp_s[WARPS], warp_u[WARPS], block_sums[3], block_maxima[CLUSTER ? LP_THREADS : 1];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const long long row = blockIdx.y;
    const int seg = blockIdx.x, first = seg * LP_SEG, here = min(V - first, LP_SEG);
    const float* x = logits + row * V + first;
    const bool whole = VEC && here == LP_SEG;
    auto load = [&](float (&v)[LP_PIECE], int e0) {
        if (whole) {
#pragma unroll
            for (int e = 0; e < LP_PIECE; e += 4) {
                const float4 y = *reinterpret_cast<const float4*>(x + lp_index<VEC>(e0 + e, tid));
                v[e] = y.x; v[e + 1] = y.y; v[e + 2] = y.z; v[e + 3] = y.w;
            }
        } else {
#pragma unroll
            for (int e = 0; e < LP_PIECE; ++e) v[e] = lp_index<VEC>(e0 + e, tid) < here ? x[lp_index<VEC>(e0 + e, tid)] : -INFINITY;
        }
    };
    float mine = -INFINITY, ref = LP_LOWEST, S = 0.f, U = 0.f, v[2][LP_PIECE];
    load(v[0], 0);
#pragma unroll
    for (int p = 0; p < LP_PER_THREAD / LP_PIECE; ++p) {
        if (p + 1 < LP_PER_THREAD / LP_PIECE) load(v[(p + 1) & 1], (p + 1) * LP_PIECE);
        const float (&y)[LP_PIECE] = v[p & 1];
#pragma unroll
        for (int e = 0; e < LP_PIECE; ++e) mine = fmaxf(mine, y[e]);
        if (mine > ref + 8.f) {
            lp_raise(S, U, ref, mine);
            ref = mine;
        }
        float s0 = 0.f, s1 = 0.f, u0 = 0.f, u1 = 0.f;
#pragma unroll
        for (int e = 0; e < LP_PIECE; e += 2) {
            const float d0 = y[e] - ref, d1 = y[e + 1] - ref, p0 = lp_exp(d0), p1 = lp_exp(d1);
            s0 += p0;
            s1 += p1;
            u0 = fmaf(p0, fmaxf(d0, -1e30f), u0);                   // 0 times -infinity is 0 here
            u1 = fmaf(p1, fmaxf(d1, -1e30f), u1);
        }
        S += s0 + s1;
        U += u0 + u1;
    }
    const long long at = row * segs + seg;
    if (!CLUSTER && maxima) maxima[at * LP_THREADS + tid] = mine;
    const float most = warp_max(mine);
    if (lane == 0) warp_m[warp] = most;
    __syncthreads();
    float m = ref;                                                  // the lowest number where there is nothing but -infinity
#pragma unroll
    for (int w = 0; w < WARPS; ++w) m = fmaxf(m, warp_m[w]);
    lp_raise(S, U, ref, m);
    S = warp_sum(S);
    U = warp_sum(U);
    if (lane == 0) { warp_s[warp] = S; warp_u[warp] = U; }
    __syncthreads();
    if (tid == 0) {
        m = LP_LOWEST;
        S = U = 0.f;
        for (int w = 0; w < WARPS; ++w) {
            m = fmaxf(m, warp_m[w]);
            S += warp_s[w];
            U += warp_u[w];
        }
        if (!CLUSTER) {
            sums[at * 3] = m;
            sums[at * 3 + 1] = S;
            sums[at * 3 + 2] = U;
        } else {
            block_sums[0] = m;
            block_sums[1] = S;
            block_sums[2] = U;
        }
    }
    if (CLUSTER) {
        block_maxima[tid] = mine;
        lp_cluster_sync();
        float held[LP_CLUSTER], Ss = 0.f, Us = 0.f;
        m = LP_LOWEST;
        if (seg == 0) {
#pragma unroll
            for (int j = 0; j < LP_CLUSTER; ++j) held[j] = top && j < segs ? lp_remote(block_maxima + tid, j) : -INFINITY;
            if (lane < segs) {
                m = lp_remote(block_sums, lane);
                Ss = lp_remote(block_sums + 1, lane);
                Us = lp_remote(block_sums + 2, lane);
            }
        }
        lp_cluster_sync();                                          // nobody leaves while its shared memory is read
        if (seg != 0) return;
        const float all = warp_max(m);
        if (lane < segs) lp_raise(Ss, Us, m, all);
        S = warp_sum(Ss);
        U = warp_sum(Us);
        lp_finish<VEC, LP_CLUSTER, LP_THREADS>(logits + row * V, tokens[row], all, S, U, held, nullptr, logprob + row, entropy + row, top_ids + row * top,
                                               top_lps + row * top, V, segs, top);
    }
}

// A block a row: the segments' sums, then the row's end.  Its reads wait for one another, so it wants all rows' blocks on the chip at once
// and the first of them there before the segments' last: 2,048 rows of 151,936 logits with a top of 5 / 20 / 64 take 204 / 215 / 252 us with
// blocks of 256 threads and 1,024 candidates, 211 / 228 / 282 with half the threads, 201 / 211 / 247 with half the candidates too (16 blocks
// an SM), 213 / 232 / - with 64 threads.
template <bool VEC>
__global__ void __launch_bounds__(LP_JOIN_THREADS, 2048 / LP_JOIN_THREADS)
lp_join_kernel(const float* __restrict__ logits, const int* __restrict__ tokens, const float* sums, const float* maxima,
               float* __restrict__ logprob, float* __restrict__ entropy, int* __restrict__ top_ids, float* __restrict__ top_lps, int V, int segs,
               int top) {
    pdl_wait();
    pdl_launch_dependents();
    const int tid = threadIdx.x, lane = tid & 31;
    const long long row = blockIdx.x;
    const float* mine = sums + row * segs * 3;
    const float* at_most = maxima + row * segs * LP_THREADS;
    float held[LP_HELD];                    // this thread's share of the maxima, the first of them in registers
#pragma unroll
    for (int j = 0; j < LP_HELD; ++j)
        held[j] = top && j < segs * (LP_THREADS / LP_JOIN_THREADS) ? __ldcg(at_most + j * LP_JOIN_THREADS + tid) : -INFINITY;
    // every warp has the sums: the same additions in the same order
    float m = LP_LOWEST;
    for (int s = lane; s < segs; s += 32) m = fmaxf(m, __ldcg(mine + s * 3));
    m = warp_max(m);
    float S = 0.f, U = 0.f;
    for (int s = lane; s < segs; s += 32) {
        float Ss = __ldcg(mine + s * 3 + 1), Us = __ldcg(mine + s * 3 + 2);
        lp_raise(Ss, Us, __ldcg(mine + s * 3), m);
        S += Ss;
        U += Us;
    }
    S = warp_sum(S);
    U = warp_sum(U);
    lp_finish<VEC, LP_HELD, LP_JOIN_THREADS>(logits + row * V, tokens[row], m, S, U, held, at_most, logprob + row, entropy + row, top_ids + row * top,
                                             top_lps + row * top, V, segs, top);
}


// Segments of a row.
extern "C" int qwb_logprobs_segments(int V) { return (int)(((long long)V + LP_SEG - 1) / LP_SEG); }

// Floats of scratch memory of a call for each of its rows; 0: none, its rows go as clusters, while these are all on the chip at once (4 blocks an SM).  8 rows of
// 151,936 logits with a top of 5: 8.2 us on the device by a second kernel, 7.2 so, and 3 us less on the host.
extern "C" int qwb_logprobs_scratch(int rows, int V, int top) {
    const int segs = qwb_logprobs_segments(V);
    return segs <= LP_CLUSTER && (long long)rows * segs <= 148 * 4 ? 0 : segs * (top ? 3 + LP_THREADS : 3);
}

// scratch: as qwb_logprobs_scratch says, or as much as it would with more rows
extern "C" int qwb_logprobs(const float* logits, const int* tokens, float* logprob, float* entropy, int* top_ids, float* top_lps, float* scratch,
                            int rows, int V, int top, cudaStream_t stream) {
    if (rows <= 0) return 0;
    if (V <= 0 || V > 2000000000 || top < 0 || top > LP_MAX_TOP || top > V)
        return qwb_fail(QWB_ERR_ARG, "token_logprobs: 0 to %d alternatives of a vocabulary of at least as many: top=%d V=%d", LP_MAX_TOP, top, V);
    if (rows > 65535) return qwb_fail(QWB_ERR_ARG, "token_logprobs: at most 65535 rows in a call, not %d", rows);
    const int segs = qwb_logprobs_segments(V);
    const bool vec = V % 4 == 0 && (uintptr_t)logits % 16 == 0;
    if (!scratch) {
        if (segs > LP_CLUSTER) return qwb_fail(QWB_ERR_ARG, "token_logprobs: no scratch for %d segments", segs);
        auto kernel = vec ? lp_segments_kernel<true, true> : lp_segments_kernel<false, true>;
        if (segs > 8) {                                             // more than 8 blocks have to be allowed, once a device
            static bool allowed[2][64];
            int device = 0;
            cudaError_t e = cudaGetDevice(&device);
            if (e == cudaSuccess && (device < 0 || device >= 64 || !allowed[vec][device])) {
                e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
                if (e == cudaSuccess && device >= 0 && device < 64) allowed[vec][device] = true;
            }
            if (e != cudaSuccess) return qwb_fail(QWB_ERR_CUDA, "token_logprobs: %s", cudaGetErrorString(e));
        }
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(segs, rows);
        cfg.blockDim = dim3(LP_THREADS);
        cfg.stream = stream;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = segs;
        attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, logits, (float*)nullptr, (float*)nullptr, tokens, logprob, entropy, top_ids, top_lps, V, segs, top);
        if (e != cudaSuccess) return qwb_fail(QWB_ERR_CUDA, "token_logprobs: %s", cudaGetErrorString(e));
        return qwb_check_launch("token_logprobs");
    }
    float* maxima = top ? scratch + (size_t)rows * segs * 3 : nullptr;
    qwb_launch(vec ? lp_segments_kernel<true, false> : lp_segments_kernel<false, false>, dim3(segs, rows), LP_THREADS, 0, stream, logits, scratch, maxima, tokens,
               logprob, entropy, top_ids, top_lps, V, segs, top);
    qwb_launch_link(1, 1, vec ? lp_join_kernel<true> : lp_join_kernel<false>, dim3(rows), LP_JOIN_THREADS, 0, stream, logits, tokens, scratch, maxima,
                    logprob, entropy, top_ids, top_lps, V, segs, top);
    return qwb_check_launch("token_logprobs");
}
