// A step's tables from its sequences' lengths, in one launch: where each sequence's new tokens begin and what it holds behind
// the step, each token's sequence, position and row of the pool, and the sequences' pages as a table with one row a sequence.
//
// What bounds it: 12 bytes a token and 4 a table entry written; a step's call is a few microseconds of latency.  So nothing
// waits for another block: every block of tokens adds up the sequences' counts by itself (a scan of B numbers in shared memory)
// and finds each token's sequence by bisection there; blocks of table entries need no sums at all.
#include "common.cuh"

#define ST_THREADS 256
#define ST_MAX_SEQS 58000       // counts that a block's shared memory holds
#define ST_PER_THREAD 4         // tokens, and table entries, of a thread

__global__ void __launch_bounds__(ST_THREADS)
step_tables_kernel(const int* __restrict__ pages, const int* __restrict__ page_start, const int* __restrict__ pos0,
                   const int* __restrict__ n_new, int* __restrict__ cu_out, int* __restrict__ seq_len, int* __restrict__ tok_seq,
                   int* __restrict__ tok_pos, int* __restrict__ slot_map, int* __restrict__ table, int P, int B, int T, int width,
                   int page_size, int token_blocks) {
    pdl_wait();
    pdl_launch_dependents();
    extern __shared__ int cu[];                                         // [B + 1]
    __shared__ int warp_sums[ST_THREADS / 32];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if ((int)blockIdx.x >= token_blocks) {                              // entries of the page table
        const long long n = (long long)B * width, i0 = (long long)(blockIdx.x - token_blocks) * (ST_THREADS * ST_PER_THREAD);
#pragma unroll
        for (int e = 0; e < ST_PER_THREAD; ++e) {
            const long long i = i0 + e * ST_THREADS + tid;
            if (i >= n) return;
            const int b = (int)(i / width), j = (int)(i - (long long)b * width);
            const long long first = page_start[b], at = first + j;
            table[i] = (first >= 0 && at < page_start[b + 1] && at < P) ? pages[at] : 0;
        }
        return;
    }
    // sums of the counts: a thread's share, the warps' sums, everything in whole numbers
    const int share = (B + ST_THREADS - 1) / ST_THREADS, b0 = min(tid * share, B), b1 = min(b0 + share, B);
    int own = 0;
    for (int b = b0; b < b1; ++b) own += max(n_new[b], 0);
    int upto = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += v;
    }
    if (lane == 31) warp_sums[warp] = upto;
    __syncthreads();
    int before = upto - own;
    for (int w = 0; w < warp; ++w) before += warp_sums[w];
    for (int b = b0; b < b1; ++b) {
        cu[b] = before;
        before += max(n_new[b], 0);
        if (b == B - 1) cu[B] = before;
    }
    __syncthreads();
    if (blockIdx.x == 0) {
        for (int b = tid; b <= B; b += ST_THREADS) {
            cu_out[b] = cu[b];
            if (b < B) seq_len[b] = pos0[b] + cu[b + 1] - cu[b];
        }
    }
#pragma unroll
    for (int e = 0; e < ST_PER_THREAD; ++e) {
        const int t = blockIdx.x * (ST_THREADS * ST_PER_THREAD) + e * ST_THREADS + tid;
        if (t >= T) return;
        int seq = -1, pos = -1, slot = -1;
        if (t < cu[B]) {
            int lo = 0, hi = B;                                         // cu[lo] <= t < cu[hi]
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if (cu[mid] <= t) lo = mid; else hi = mid;
            }
            seq = lo;
            pos = pos0[lo] + t - cu[lo];
            const long long first = page_start[lo], at = first + pos / page_size;
            if (pos >= 0 && first >= 0 && at < page_start[lo + 1] && at < P) slot = pages[at] * page_size + pos % page_size;
        }
        tok_seq[t] = seq;
        tok_pos[t] = pos;
        slot_map[t] = slot;
    }
}

extern "C" int qwb_step_tables(const int* pages, const int* page_start, const int* pos0, const int* n_new, int* cu, int* seq_len,
                               int* tok_seq, int* tok_pos, int* slot_map, int* table, int P, int B, int T, int width, int page_size,
                               int tokens, cudaStream_t stream) {
    if (B <= 0 || B > ST_MAX_SEQS || T < 0 || width < 0 || P < 0 || page_size <= 0)
        return qwb_fail(QWB_ERR_ARG, "step_tables: 1 to %d sequences, no negative sizes: B=%d T=%d width=%d pages=%d", ST_MAX_SEQS, B, T, width, P);
    const int per_block = ST_THREADS * ST_PER_THREAD;
    const int token_blocks = tokens ? (T > 0 ? (T - 1) / per_block + 1 : 1) : 0;
    const long long table_blocks = ((long long)B * width + per_block - 1) / per_block;
    if (token_blocks + table_blocks > 2147483647ll) return qwb_fail(QWB_ERR_ARG, "step_tables: a table of %d x %d is too large", B, width);
    if (token_blocks + table_blocks == 0) return 0;
    const size_t smem = (B + 1) * sizeof(int);
    if (smem > 48 * 1024) {
        const cudaError_t e = cudaFuncSetAttribute(step_tables_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e != cudaSuccess) return qwb_fail(QWB_ERR_CUDA, "step_tables: %s", cudaGetErrorString(e));
    }
    qwb_launch(step_tables_kernel, dim3((unsigned)(token_blocks + table_blocks)), ST_THREADS, smem, stream, pages, page_start, pos0, n_new,
               cu, seq_len, tok_seq, tok_pos, slot_map, table, P, B, T, width, page_size, token_blocks);
    return qwb_check_launch("step_tables");
}
