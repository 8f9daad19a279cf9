// Attention over the cache in 4 bits (kv4.cuh), causal, grouped heads, with an optional window.
//
// Few new tokens a sequence, bfloat16, heads of 64 or 128 (kv4_attn_rows_kernel): a decode step.  What it has to do is read the
// cache, 144 bytes a token and head of 128, for 4 x 128 multiply-adds a query head: on mma.sync, whose products are far from the limit
// here (a group of 4 heads fills half of the 8 columns), so that the time is loads and the way from codes to bfloat16.
//   * A block takes a key/value head and a run of a sequence's pages; its two warps take 32 keys of every page each, with their
//     own copies (cp.async into a ring of their own), maxima, sums and outputs, and meet at the run's end in shared memory.  Nothing in
//     between waits for another warp.
//   * The 16-row operand of both products is the cache's, the 8 columns are (token, query head) pairs:
//     S^T = K Q^T and O^T = V^T P^T, so that 4 query heads take half of an mma and not a quarter.
//   * Which number of a row sits where in an mma's inner dimension is free as long as both operands agree.  A lane therefore takes
//     32 neighbouring numbers of a key (one 16-byte load, one group, one step), and of a value its 16 numbers of 4 keys; codes come out
//     of a 32-bit word two at a time, in the places where their shifts leave them.
//   * A code c becomes the bfloat16 128 + c by one and-or (its 7 bits behind the point hold c) and c s by one fused multiply-add.  The
//     zero points are taken off as sums: of the scores by one more mma, whose inner dimension holds z s of a lane's group and the sum of the
//     query's numbers there (in three bfloat16 parts), of the outputs by a row of z s in the mma that adds up the weights.  (What the two sums have in
//     common is lost from their difference: an output is off by up to 2^-23 of its group's 15 steps, also where it is much smaller itself.)
//   * The scores' columns are the next product's inner dimension: P^T's operand is two 8 x 8 transpositions (movmatrix).
//   * A run's softmax is relative to a reference that is raised, and O rescaled, only where a score passes it by 2^8: most pages vote once
//     and exchange no maxima.  The weights' sum is one more mma with rows of ones, over
//     the weights as they are rounded for the product.
// Runs are cut by the sequence's own length (kv4_runs), never by what else is in the batch.  Up to 16 of them are the blocks of a cluster, which
// read each other's results from shared memory; more leave them in scratch memory for a second kernel.  Both join them in the same order,
// so that which way it went cannot be told from the result (qwb_kv4_plan says which, with times).
//
// The plain kernel: any head size that is a multiple of 32, queries in 32 bits or bfloat16.  A block takes a (token, query head),
// its four warps every fourth key; a lane holds the numbers lane, lane + 32, ... of the query, of the sums and of a key, so a
// group of 32 is a step of the loop over them.  Each warp keeps a running maximum, sum and output; they meet in shared memory.
#include "attention_pieces.h"
#include "kv4.cuh"

#include <math.h>

#define KP_WARPS 4

template <typename T>
__global__ void __launch_bounds__(KP_WARPS * 32)
kv4_attn_plain_kernel(const T* __restrict__ q, const unsigned char* __restrict__ pool, const int* __restrict__ page_table,
                      const int* __restrict__ tok_seq, const int* __restrict__ tok_pos, T* __restrict__ out, int B, int pool_pages,
                      int Hq, int Hkv, int hd, int table_width, float scale, int window) {
    pdl_wait();
    pdl_launch_dependents();
    __shared__ float part[KP_WARPS][KV4_MAX_DIM + 2];
    const int t = blockIdx.x, h = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int groups = hd / KV4_GROUP, kvh = h / (Hq / Hkv);
    const int b = tok_seq[t], pos = tok_pos[t];
    float qv[KV4_MAX_DIM / 32], acc[KV4_MAX_DIM / 32];
#pragma unroll
    for (int g = 0; g < KV4_MAX_DIM / 32; ++g) {
        qv[g] = g < groups ? to_f32(q[((size_t)t * Hq + h) * hd + g * 32 + lane]) : 0.f;
        acc[g] = 0.f;
    }
    float m = -INFINITY, l = 0.f;
    const int first = window > 0 ? max(0, pos - window + 1) : 0;
    if (b >= 0 && b < B) {
        for (int j = first + warp; j <= pos; j += KP_WARPS) {
            if (j / KV4_PAGE >= table_width) break;
            const long long page = page_table[(size_t)b * table_width + j / KV4_PAGE];
            if (page < 0 || page >= pool_pages) continue;
            const int row = j % KV4_PAGE;
            const unsigned char* k = pool + ((size_t)page * Hkv + kvh) * kv4_page_bytes(hd);
            const unsigned char* v = k + kv4_half_bytes(hd);
            const uint16_t* kw = reinterpret_cast<const uint16_t*>(k + kv4_code_bytes(hd)) + row * groups;
            const uint16_t* vw = reinterpret_cast<const uint16_t*>(v + kv4_code_bytes(hd)) + row * groups;
            float s = 0.f;
#pragma unroll
            for (int g = 0; g < KV4_MAX_DIM / 32; ++g) {
                if (g >= groups) break;
                const uint32_t code = (k[row * (hd / 2) + g * 16 + lane / 2] >> (4 * (lane & 1))) & 15u;
                s += qv[g] * (((float)code - kv4_zero(kw[g])) * kv4_step(kw[g]));
            }
            s = warp_sum(s) * scale;
            const float m_new = fmaxf(m, s);
            const float keep = expf(m - m_new), p = expf(s - m_new);
            l = l * keep + p;
#pragma unroll
            for (int g = 0; g < KV4_MAX_DIM / 32; ++g) {
                if (g >= groups) break;
                const uint32_t code = (v[row * (hd / 2) + g * 16 + lane / 2] >> (4 * (lane & 1))) & 15u;
                acc[g] = acc[g] * keep + p * (((float)code - kv4_zero(vw[g])) * kv4_step(vw[g]));
            }
            m = m_new;
        }
    }
    bool broken = false;                    // a value that is not finite makes all of the head NaN
#pragma unroll
    for (int g = 0; g < KV4_MAX_DIM / 32; ++g)
        if (g < groups) {
            part[warp][g * 32 + lane] = acc[g];
            broken |= acc[g] != acc[g];
        }
    if (__any_sync(0xffffffffu, broken)) l = __uint_as_float(0x7fffffffu);
    if (lane == 0) { part[warp][KV4_MAX_DIM] = m; part[warp][KV4_MAX_DIM + 1] = l; }
    __syncthreads();
    float top = -INFINITY, total = 0.f, f[KP_WARPS];
    for (int w = 0; w < KP_WARPS; ++w) top = fmaxf(top, part[w][KV4_MAX_DIM]);
    for (int w = 0; w < KP_WARPS; ++w) {
        f[w] = part[w][KV4_MAX_DIM + 1] == 0.f ? 0.f : expf(part[w][KV4_MAX_DIM] - top);
        total += f[w] * part[w][KV4_MAX_DIM + 1];
    }
    for (int d = threadIdx.x; d < hd; d += KP_WARPS * 32) {
        float o = 0.f;
        for (int w = 0; w < KP_WARPS; ++w)
            if (f[w] != 0.f) o += f[w] * part[w][d];
        out[((size_t)t * Hq + h) * hd + d] = from_f32<T>(total == 0.f ? 0.f : o / total);      // a row that sees nothing: zeros
    }
}

extern "C" int qwb_kv4_attn_plain(const void* q, const unsigned char* pool, const int* page_table, const int* tok_seq, const int* tok_pos,
                                  void* out, int dtype, int T, int B, int pool_pages, int Hq, int Hkv, int hd, int table_width,
                                  float scale, int window, cudaStream_t stream) {
    if (T <= 0) return 0;
    if (Hkv <= 0 || Hq <= 0 || Hq % Hkv || Hq > 65535 || hd <= 0 || hd % KV4_GROUP || hd > KV4_MAX_DIM || table_width <= 0 || window < 0 || !(scale > 0.f))
        return qwb_fail(QWB_ERR_ARG, "kv4_attention: bad sizes Hq=%d Hkv=%d hd=%d width=%d window=%d scale=%g", Hq, Hkv, hd, table_width, window, (double)scale);
    if (dtype == QWB_DT_F32)
        qwb_launch(kv4_attn_plain_kernel<float>, dim3(T, Hq), KP_WARPS * 32, 0, stream, (const float*)q, pool, page_table, tok_seq, tok_pos, (float*)out,
                   B, pool_pages, Hq, Hkv, hd, table_width, scale, window);
    else if (dtype == QWB_DT_BF16)
        qwb_launch(kv4_attn_plain_kernel<bf16>, dim3(T, Hq), KP_WARPS * 32, 0, stream, (const bf16*)q, pool, page_table, tok_seq, tok_pos, (bf16*)out,
                   B, pool_pages, Hq, Hkv, hd, table_width, scale, window);
    else
        return qwb_fail(QWB_ERR_ARG, "kv4_attention: unknown dtype %d", dtype);
    return qwb_check_launch("kv4_attention");
}

// ----------------------------------------------------------------------------- few new tokens: mma.sync
#define KD_WARPS 2
#define KD_KEYS 32              // keys of a page that a warp takes: two tiles of the mma's 16 rows
#define KD_STAGES 2             // pages of a warp's ring: 8 x 4,096 tokens 15.0 us, with three 16.0
#define KD_RUNS 16              // a sequence's pages are cut into about so many runs ...
#define KD_RUN_PAGES 8          // ... of at most this many pages
#define KD_RAISE 8.f            // a run's reference is raised where a score passes it by 2^8

// The pages that a sequence's new tokens see, and how they are cut.
struct Kv4Runs { int first, count, per_run, runs; };
__host__ __device__ __forceinline__ Kv4Runs kv4_runs(int pos0, int len, int window, int table_width) {
    Kv4Runs r;
    const int low = window > 0 && pos0 - window + 1 > 0 ? pos0 - window + 1 : 0;
    r.first = low / KV4_PAGE;
    const int last = (len - 1) / KV4_PAGE < table_width - 1 ? (len - 1) / KV4_PAGE : table_width - 1;
    r.count = len > 0 && last >= r.first ? last - r.first + 1 : 0;
    const int even = (r.count + KD_RUNS - 1) / KD_RUNS;
    r.per_run = even < 1 ? 1 : (even > KD_RUN_PAGES ? KD_RUN_PAGES : even);
    r.runs = (r.count + r.per_run - 1) / r.per_run;
    return r;
}

__device__ __forceinline__ void kd_copy16(void* dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void kd_mma(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t kd_transpose(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ uint32_t kd_pack(float lo, float hi) {
    __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&v);
}
__device__ __forceinline__ float kd_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
template <int HD>
struct KdTile {                                             // a warp's keys of a page and head
    static constexpr int CODES = KD_KEYS * HD / 2, WORDS = KD_KEYS * HD / 16, HALF = CODES + WORDS, BYTES = 2 * HALF;
};
#define KD_CLUSTER 16           // blocks of the largest cluster
template <int HD, int NT>
struct KdSmem {
    static constexpr int RING = KD_WARPS * KD_STAGES * KdTile<HD>::BYTES;
    static constexpr int COL = HD + 4;                      // floats of a column of outputs: two columns are 8 banks apart
    static constexpr int JOIN = KD_WARPS * 8 * NT * (COL + 2) * 4;
    static constexpr int DONE = 8 * NT * (COL + 2) * 4;     // the block's own outputs, maxima and sums, behind its warps'
    static constexpr int BYTES = RING > JOIN + DONE ? RING : JOIN + DONE;
};

// The join of a row's runs: relative to the largest maximum, in four sums of every fourth run, which are then added.
__device__ __forceinline__ float kd_share(float m, float l, float top) { return l == 0.f ? 0.f : m == top ? 1.f : kd_exp2(m - top); }
__device__ __forceinline__ float kd_four(const float (&x)[4]) { return (x[0] + x[1]) + (x[2] + x[3]); }
__device__ __forceinline__ float2 kd_remote2(uint32_t at) {
    float2 v;
    asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(at) : "memory");
    return v;
}
__device__ __forceinline__ float kd_remote(uint32_t at) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
    return v;
}
__device__ __forceinline__ uint32_t kd_of_block(uint32_t mine, int rank) {                     // an address of this block's shared memory, in the cluster's `rank`th
    uint32_t at;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(mine), "r"(rank));
    return at;
}
__device__ __forceinline__ void kd_cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// NT: tiles of 8 columns of a block.  CLUSTER: the runs of a tile are the blocks of a cluster.  part: [rows, max_runs, HD] outputs, then [rows, max_runs, 2] maxima (of scores times log2 e) and sums
// of the runs of sequences that have more than one; a row is (token, query head), of the key/value heads from kv0 on that the launch has blocks for.
// ROOM: blocks an SM that registers leave room for.  With 8 columns 7, as many as shared memory does: 32 x 16,384 tokens 114 us, 116 with 8, 120 with 6.  With
// 16 columns 5 (168 registers, some of them spilled), and 4 where no more are launched than so fit at once: 4 new tokens of one sequence of 8,192
// 15.6 us instead of 17.7, of four sequences, 1,000 blocks, 33.4 instead of 30.1.
template <int HD, int NT, bool CLUSTER, int ROOM>
__global__ void __launch_bounds__(KD_WARPS * 32, ROOM)
kv4_attn_rows_kernel(const bf16* __restrict__ q, const unsigned char* __restrict__ pool, const int* __restrict__ page_table,
                     const int* __restrict__ cu_seqlens, const int* __restrict__ pos0, bf16* __restrict__ out, float* __restrict__ part_o,
                     float* __restrict__ part_ml, int T, int B, int pool_pages, int G, int Hkv, int table_width, float scale_log2, int window,
                     int tiles, int max_runs, int kv0) {
    pdl_wait();
    pdl_launch_dependents();
    using Tile = KdTile<HD>;
    using Smem = KdSmem<HD, NT>;
    extern __shared__ __align__(128) unsigned char smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3;
    int run, tile;
    if (CLUSTER) {
        tile = blockIdx.x / max_runs;                       // max_runs: the cluster's blocks
        run = blockIdx.x - tile * max_runs;
    } else {
        run = tiles == 1 ? blockIdx.x : blockIdx.x / tiles;
        tile = blockIdx.x - run * tiles;
    }
    const int kvh = kv0 + blockIdx.y, b = blockIdx.z;
    const int Hq = Hkv * G;
    const float one_in_g = 1.f / (float)G;
    auto by_g = [&](int x) { return (int)(((float)x + 0.5f) * one_in_g); };             // x / G: exact for x below 2^20 (the launcher's bound)
    const int t0 = cu_seqlens[b], t1 = cu_seqlens[b + 1], p0 = pos0[b], used = max(cu_seqlens[B], 0);
    if (used < T) {                                         // tokens behind the last sequence's: zeros
        const long long me = (((long long)b * gridDim.y + blockIdx.y) * gridDim.x + blockIdx.x) * (KD_WARPS * 32) + threadIdx.x;
        const long long all = (long long)gridDim.x * gridDim.y * gridDim.z * (KD_WARPS * 32), end = (long long)T * Hq * (HD / 8);
        for (long long i = (long long)used * Hq * (HD / 8) + me; i < end; i += all) reinterpret_cast<uint4*>(out)[i] = make_uint4(0, 0, 0, 0);
    }
    const int n_new = min(t1, T) - t0, col0 = tile * 8 * NT, cols = n_new * G;
    if (t0 < 0 || n_new <= 0 || col0 >= cols) return;
    const int len = p0 + n_new;
    const Kv4Runs cut = kv4_runs(p0, len, window, table_width);
    const int runs = min(cut.runs, max_runs);               // a sequence beyond max_len: cut off there, never written beyond the scratch
    if (!CLUSTER && run >= runs && run > 0) return;         // (a block of a cluster stays for its barriers, without pages)
    const int first_page = cut.first + run * cut.per_run, n_pages = max(min(cut.per_run, cut.count - run * cut.per_run), 0);
    const int* table = page_table + (size_t)b * table_width + first_page;
    int my_page = -1;                                       // lane i: the run's i-th page
    if (lane < n_pages) my_page = table[lane];
    if (my_page >= pool_pages) my_page = -1;

    unsigned char* ring = smem + (size_t)warp * KD_STAGES * Tile::BYTES;
    int slot_in = 0, slot_out = 0;
    auto ask = [&](int i) {                                 // the warp's 32 keys of the run's i-th page
        const int page = __shfl_sync(0xffffffffu, my_page, i & 31);
        if (i < n_pages && page >= 0) {
            unsigned char* dst = ring + slot_in * Tile::BYTES;
            const unsigned char* src = pool + ((size_t)page * Hkv + kvh) * kv4_page_bytes(HD) + warp * Tile::CODES;
            constexpr int WORDS_AT = kv4_code_bytes(HD);
#pragma unroll
            for (int o = 0; o < Tile::CODES; o += 512) {
                kd_copy16(dst + o + lane * 16, src + o + lane * 16);
                kd_copy16(dst + Tile::HALF + o + lane * 16, src + kv4_half_bytes(HD) + o + lane * 16);
            }
            constexpr int PIECES = Tile::WORDS / 16;
            if (lane < 2 * PIECES) {
                const int half = lane / PIECES, at = (lane % PIECES) * 16;
                kd_copy16(dst + half * Tile::HALF + Tile::CODES + at, src + half * kv4_half_bytes(HD) + WORDS_AT - warp * Tile::CODES + warp * Tile::WORDS + at);
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
        slot_in = slot_in == KD_STAGES - 1 ? 0 : slot_in + 1;
    };
#pragma unroll
    for (int i = 0; i < KD_STAGES - 1; ++i) ask(i);

    // this block's columns: their last and first key; the queries, in the order in which a lane holds the keys' numbers
    int last_key[NT][2], first_key[NT][2];
    uint32_t qf[NT][HD / 16][2], qz[NT][2];                 // qz: minus the sum of a lane's numbers of the query, in three parts
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int col = min(col0 + n * 8 + 2 * c + e, cols - 1);
            last_key[n][e] = p0 + by_g(col);
            first_key[n][e] = window > 0 ? last_key[n][e] - window + 1 : 0;
        }
        const int col = col0 + n * 8 + r, tok = by_g(col);
        const bool live = col < cols;
        const bf16* src = q + ((size_t)(t0 + tok) * Hq + kvh * G + col - tok * G) * HD + c * (HD / 4);
        float sum = 0.f;
#pragma unroll
        for (int w = 0; w < HD / 32; ++w) {
            uint4 v = make_uint4(0, 0, 0, 0);
            if (live) v = *reinterpret_cast<const uint4*>(src + 8 * w);
            qf[n][2 * w][0] = __byte_perm(v.x, v.z, 0x5410);            // numbers 0 and 4, 1 and 5, 2 and 6, 3 and 7 of 8
            qf[n][2 * w][1] = __byte_perm(v.x, v.z, 0x7632);
            qf[n][2 * w + 1][0] = __byte_perm(v.y, v.w, 0x5410);
            qf[n][2 * w + 1][1] = __byte_perm(v.y, v.w, 0x7632);
            const uint32_t x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) sum += __uint_as_float(x[i] << 16) + __uint_as_float(x[i] & 0xffff0000u);
        }
        const float hi = __bfloat162float(__float2bfloat16_rn(sum)), mid = __bfloat162float(__float2bfloat16_rn(sum - hi));
        qz[n][0] = kd_pack(-hi, -mid);
        qz[n][1] = kd_pack(hi + mid - sum, 0.f);
    }
    const int see_all_from = window > 0 ? p0 + by_g(min(col0 + 8 * NT, cols) - 1) - window + 1 : 0;    // keys below may be hidden from a column,
    const int see_all_to = p0 + by_g(col0);                                                       // keys above as well

    // outputs; the weights' sums (0, 1: from rows of ones) and what the zero points add to a lane's outputs (2, 3); the reference of the raw scores, what passes it by 2^8, and -reference in the
    // exponent's units (0 while there is no reference: a weight of a hidden key is then 2^-infinity)
    float o[NT][HD / 16][4], l[NT][4], m[NT][2], over[NT][2], shift[NT][2];
    const float raise = KD_RAISE / scale_log2;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int i = 0; i < HD / 16; ++i) o[n][i][0] = o[n][i][1] = o[n][i][2] = o[n][i][3] = 0.f;
        l[n][0] = l[n][1] = l[n][2] = l[n][3] = 0.f;
        m[n][0] = m[n][1] = over[n][0] = over[n][1] = -INFINITY;
        shift[n][0] = shift[n][1] = 0.f;
    }
    // row r of a tile is key `key_r` of the 16, row r + 8 the key 8 behind it: of the keys that one load takes from shared memory then
    // never two lie in the same banks
    const int key_r = (r & 1) ? 4 + ((r >> 1) ^ 1) : r >> 1;
    const int vk0 = c, vk1 = 4 + (c ^ 1);                   // a lane's four keys of a value tile: rows 2c, 2c + 1 and the ones 8 behind
    constexpr int TILES = KD_KEYS / 16, GROUPS = HD / KV4_GROUP;

    for (int i = 0; i < n_pages; ++i) {
        ask(i + KD_STAGES - 1);
        asm volatile("cp.async.wait_group %0;" ::"n"(KD_STAGES - 1) : "memory");
        __syncwarp();
        const unsigned char* kt = ring + slot_out * Tile::BYTES;
        slot_out = slot_out == KD_STAGES - 1 ? 0 : slot_out + 1;
        const unsigned char* vt = kt + Tile::HALF;
        const uint16_t* kw = reinterpret_cast<const uint16_t*>(kt + Tile::CODES);
        const uint16_t* vw = reinterpret_cast<const uint16_t*>(vt + Tile::CODES);
        const int base = (first_page + i) * KV4_PAGE + warp * KD_KEYS;
        const bool there = __shfl_sync(0xffffffffu, my_page, i) >= 0;
        if (there && base < len) {
            // S^T = K Q^T
            float s[TILES][NT][4];
#pragma unroll
            for (int t = 0; t < TILES; ++t) {
#pragma unroll
                for (int n = 0; n < NT; ++n) s[t][n][0] = s[t][n][1] = s[t][n][2] = s[t][n][3] = 0.f;
                constexpr int LW = HD / 32;                 // 32-bit words of codes of a lane's numbers of a key
                uint32_t ka[LW], kb[LW];
                const unsigned char* pa = kt + (16 * t + key_r) * (HD / 2) + c * (HD / 8);
                const unsigned char* pb = pa + 8 * (HD / 2);
                if constexpr (LW == 4) {
                    const uint4 va = *reinterpret_cast<const uint4*>(pa), vb = *reinterpret_cast<const uint4*>(pb);
                    ka[0] = va.x; ka[1] = va.y; ka[2] = va.z; ka[3] = va.w;
                    kb[0] = vb.x; kb[1] = vb.y; kb[2] = vb.z; kb[3] = vb.w;
                } else {
                    const uint2 va = *reinterpret_cast<const uint2*>(pa), vb = *reinterpret_cast<const uint2*>(pb);
                    ka[0] = va.x; ka[1] = va.y;
                    kb[0] = vb.x; kb[1] = vb.y;
                }
                const uint16_t* words = kw + (16 * t + key_r) * GROUPS + c * (HD / 4) / KV4_GROUP;
                const uint32_t wa = words[0] * 0x10001u, wb = words[8 * GROUPS] * 0x10001u;
                const uint32_t sa = wa & 0xfff0fff0u, sb = wb & 0xfff0fff0u, fa = kv4_off(sa), fb = kv4_off(sb);
                const uint32_t za = kv4_scaled(wa, sa, fa), zb = kv4_scaled(wb, sb, fb);
#pragma unroll
                for (int n = 0; n < NT; ++n) kd_mma(s[t][n], za, zb, za, zb, qz[n][0], qz[n][1]);
#pragma unroll
                for (int k = 0; k < HD / 16; ++k) {
                    const int sh = 8 * (k & 1);
                    const uint32_t a0 = kv4_scaled(ka[k / 2] >> sh, sa, fa), a1 = kv4_scaled(kb[k / 2] >> sh, sb, fb);
                    const uint32_t a2 = kv4_scaled(ka[k / 2] >> (sh + 4), sa, fa), a3 = kv4_scaled(kb[k / 2] >> (sh + 4), sb, fb);
#pragma unroll
                    for (int n = 0; n < NT; ++n) kd_mma(s[t][n], a0, a1, a2, a3, qf[n][k][0], qf[n][k][1]);
                }
            }
            const bool part_hidden = base + KD_KEYS - 1 > see_all_to || base < see_all_from;        // the same for the warp
            if (part_hidden) {
                // a hidden key counts for nothing whatever it holds: its weight is 0, and a value that is not finite is taken as 0 below and
                // gives those that see it a score of NaN instead
#pragma unroll
                for (int t = 0; t < TILES; ++t)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const int row = 16 * t + key_r + 8 * h, key = base + row;
                        bool bad = false;
#pragma unroll
                        for (int g = 0; g < GROUPS; ++g) bad |= kv4_is_nan(vw[row * GROUPS + g]);
#pragma unroll
                        for (int n = 0; n < NT; ++n)
#pragma unroll
                            for (int e = 0; e < 2; ++e) {
                                if (bad) s[t][n][2 * h + e] = __uint_as_float(0x7fffffffu);
                                if (key > last_key[n][e] || key < first_key[n][e]) s[t][n][2 * h + e] = -INFINITY;
                            }
                    }
            }
            bool raised = false;
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float top = fmaxf(s[0][n][e], s[0][n][e + 2]);
#pragma unroll
                    for (int t = 1; t < TILES; ++t) top = fmaxf(top, fmaxf(s[t][n][e], s[t][n][e + 2]));
                    raised |= top > over[n][e];
                }
            if (__any_sync(0xffffffffu, raised)) {
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    float f[2];
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float top = fmaxf(s[0][n][e], s[0][n][e + 2]);
#pragma unroll
                        for (int t = 1; t < TILES; ++t) top = fmaxf(top, fmaxf(s[t][n][e], s[t][n][e + 2]));
                        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
                        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
                        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
                        const float up = fmaxf(m[n][e], top);
                        f[e] = up == m[n][e] ? 1.f : m[n][e] == -INFINITY ? 0.f : kd_exp2((m[n][e] - up) * scale_log2);
                        m[n][e] = up;
                        over[n][e] = up + raise;
                        shift[n][e] = up == -INFINITY ? 0.f : -up * scale_log2;
                    }
#pragma unroll
                    for (int k = 0; k <= HD / 16; ++k) {
                        float* x = k < HD / 16 ? o[n][k] : l[n];
                        x[0] *= f[0];
                        x[1] *= f[1];
                        x[2] *= f[0];
                        x[3] *= f[1];
                    }
                }
            }
#pragma unroll
            for (int t = 0; t < TILES; ++t) {
                // P = 2^(S - reference)
                uint32_t pb[NT][2];
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    float p[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) p[e] = kd_exp2(fmaf(s[t][n][e], scale_log2, shift[n][e & 1]));
                    pb[n][0] = kd_transpose(kd_pack(p[0], p[1]));
                    pb[n][1] = kd_transpose(kd_pack(p[2], p[3]));
                }
                // O^T += V^T P^T
                const uint16_t* words = vw + r * (HD / 8) / KV4_GROUP;
                const int row0 = 16 * t + vk0, row1 = 16 * t + vk1;
                uint32_t w0 = words[row0 * GROUPS], w1 = words[row1 * GROUPS], w2 = words[(row0 + 8) * GROUPS], w3 = words[(row1 + 8) * GROUPS];
                if (part_hidden) {
                    if (base + row0 >= len || kv4_is_nan(w0)) w0 = 0;
                    if (base + row1 >= len || kv4_is_nan(w1)) w1 = 0;
                    if (base + row0 + 8 >= len || kv4_is_nan(w2)) w2 = 0;
                    if (base + row1 + 8 >= len || kv4_is_nan(w3)) w3 = 0;
                }
                const uint32_t w01 = __byte_perm(w0, w1, 0x5410), w23 = __byte_perm(w2, w3, 0x5410);
                const uint32_t s01 = w01 & 0xfff0fff0u, s23 = w23 & 0xfff0fff0u, f01 = kv4_off(s01), f23 = kv4_off(s23);
                const uint32_t z01 = kv4_scaled(w01, s01, f01), z23 = kv4_scaled(w23, s23, f23);
#pragma unroll
                for (int n = 0; n < NT; ++n) kd_mma(l[n], 0x3f803f80u, z01, 0x3f803f80u, z23, pb[n][0], pb[n][1]);
                constexpr int VW = HD / 64;                 // words of codes of a lane's numbers of a value
                uint32_t v0[VW], v1[VW], v2[VW], v3[VW];
                const unsigned char* pv = vt + r * (HD / 16);
                if constexpr (VW == 2) {
                    const uint2 x0 = *reinterpret_cast<const uint2*>(pv + row0 * (HD / 2)), x1 = *reinterpret_cast<const uint2*>(pv + row1 * (HD / 2));
                    const uint2 x2 = *reinterpret_cast<const uint2*>(pv + (row0 + 8) * (HD / 2)), x3 = *reinterpret_cast<const uint2*>(pv + (row1 + 8) * (HD / 2));
                    v0[0] = x0.x; v0[1] = x0.y; v1[0] = x1.x; v1[1] = x1.y; v2[0] = x2.x; v2[1] = x2.y; v3[0] = x3.x; v3[1] = x3.y;
                } else {
                    v0[0] = *reinterpret_cast<const uint32_t*>(pv + row0 * (HD / 2));
                    v1[0] = *reinterpret_cast<const uint32_t*>(pv + row1 * (HD / 2));
                    v2[0] = *reinterpret_cast<const uint32_t*>(pv + (row0 + 8) * (HD / 2));
                    v3[0] = *reinterpret_cast<const uint32_t*>(pv + (row1 + 8) * (HD / 2));
                }
#pragma unroll
                for (int w = 0; w < VW; ++w) {
                    const uint32_t lo01 = __byte_perm(v0[w], v1[w], 0x5410), hi01 = __byte_perm(v0[w], v1[w], 0x7632);
                    const uint32_t lo23 = __byte_perm(v2[w], v3[w], 0x5410), hi23 = __byte_perm(v2[w], v3[w], 0x7632);
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const uint32_t a0 = kv4_scaled(lo01 >> (4 * j), s01, f01), a1 = kv4_scaled(hi01 >> (4 * j), s01, f01);
                        const uint32_t a2 = kv4_scaled(lo23 >> (4 * j), s23, f23), a3 = kv4_scaled(hi23 >> (4 * j), s23, f23);
#pragma unroll
                        for (int n = 0; n < NT; ++n) kd_mma(o[n][4 * w + j], a0, a1, a2, a3, pb[n][0], pb[n][1]);
                    }
                }
            }
        }
        __syncwarp();                                       // the slot is asked for again
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();                                        // the ring's memory holds the warps' results from here on

    // outputs of a column in the order [mma][upper or lower 8 rows][row]: number row * HD / 8 + 8 (mma / 4) + 4 half + mma % 4
    float* join_o = reinterpret_cast<float*>(smem);
    float* join_ml = join_o + KD_WARPS * 8 * NT * Smem::COL;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int col = n * 8 + 2 * c + e;
            float* dst = join_o + (warp * 8 * NT + col) * Smem::COL + r;
#pragma unroll
            for (int k = 0; k < HD / 16; ++k) {
                dst[16 * k] = o[n][k][e] - l[n][e + 2];
                dst[16 * k + 8] = o[n][k][e + 2] - l[n][e + 2];
            }
            if (r == 0) {
                join_ml[(warp * 8 * NT + col) * 2] = m[n][e] == -INFINITY ? -INFINITY : m[n][e] * scale_log2;
                join_ml[(warp * 8 * NT + col) * 2 + 1] = l[n][e];
            }
        }
    }
    __syncthreads();
    // a warp every second column, a lane four neighbouring places of it (with heads of 64 two)
    constexpr int E = HD / 32;
    float* done_o = join_ml + KD_WARPS * 8 * NT * 2;
    float* done_ml = done_o + 8 * NT * Smem::COL;
    for (int col = warp; col < 8 * NT; col += KD_WARPS) {
        if (col0 + col >= cols) break;
        float mw[KD_WARPS], lw[KD_WARPS], y[E] = {}, top = -INFINITY, total = 0.f;
#pragma unroll
        for (int w = 0; w < KD_WARPS; ++w) {
            mw[w] = join_ml[(w * 8 * NT + col) * 2];
            lw[w] = join_ml[(w * 8 * NT + col) * 2 + 1];
            top = fmaxf(top, mw[w]);
        }
#pragma unroll
        for (int w = 0; w < KD_WARPS; ++w) {
            const float f = kd_share(mw[w], lw[w], top);
            const float* src = join_o + (w * 8 * NT + col) * Smem::COL + lane * E;
            total += f * lw[w];
            if (lw[w] != 0.f) {
#pragma unroll
                for (int e = 0; e < E; ++e) y[e] += f * src[e];
            }
        }
        // a value that is not finite makes all of the head NaN, wherever in its page it lies (masked tiles have it so by the score)
        bool broken = false;
#pragma unroll
        for (int e = 0; e < E; ++e) broken |= y[e] != y[e];
        if (__any_sync(0xffffffffu, broken)) total = __uint_as_float(0x7fffffffu);
        const int tok = by_g(col0 + col);
        const size_t row = (size_t)(t0 + tok) * Hq + kvh * G + col0 + col - tok * G;
        if (CLUSTER ? max_runs == 1 : runs <= 1) {
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const int at = lane * E + e, mma = at / 16, half = (at >> 3) & 1, d = (at & 7) * (HD / 8) + 8 * (mma >> 2) + 4 * half + (mma & 3);
                out[row * HD + d] = from_f32<bf16>(total == 0.f ? 0.f : y[e] / total);
            }
        } else {
            const size_t part = ((size_t)(t0 + tok) * gridDim.y + blockIdx.y) * G + col0 + col - tok * G;         // the row among those of the heads of this launch
            float* dst = CLUSTER ? done_o + col * Smem::COL + lane * E : part_o + (part * max_runs + run) * HD + lane * E;
            if constexpr (E == 4) *reinterpret_cast<float4*>(dst) = make_float4(y[0], y[1], y[2], y[3]);
            else *reinterpret_cast<float2*>(dst) = make_float2(y[0], y[1]);
            if (lane == 0) *reinterpret_cast<float2*>(CLUSTER ? done_ml + 2 * col : part_ml + (part * max_runs + run) * 2) = make_float2(top, total);
        }
    }
    if (CLUSTER && max_runs > 1) {
        kd_cluster_sync();
        // 32 places of a column at a time, all warps of the cluster side by side
        const uint32_t o_at = (uint32_t)__cvta_generic_to_shared(done_o), ml_at = (uint32_t)__cvta_generic_to_shared(done_ml);
        const int n_runs = max(runs, 1), live = min(8 * NT, cols - col0);
        for (int piece = run * KD_WARPS + warp; piece < live * E; piece += max_runs * KD_WARPS) {
            const int col = piece / E, at = (piece % E) * 32 + lane;
            float2 ml = make_float2(-INFINITY, 0.f);
            if (lane < n_runs) ml = kd_remote2(kd_of_block(ml_at + 8 * col, lane));
            float v[KD_CLUSTER];
#pragma unroll
            for (int i = 0; i < KD_CLUSTER; ++i) v[i] = i < n_runs ? kd_remote(kd_of_block(o_at + 4 * (col * Smem::COL + at), i)) : 0.f;
            const float f = kd_share(ml.x, ml.y, warp_max(ml.x)), fl = f * ml.y;
            float sum[4] = {}, y[4] = {};
#pragma unroll
            for (int i = 0; i < KD_CLUSTER; ++i) {
                const float fi = __shfl_sync(0xffffffffu, f, i), l_i = __shfl_sync(0xffffffffu, ml.y, i);
                if (l_i != 0.f) {
                    sum[i & 3] += __shfl_sync(0xffffffffu, fl, i);
                    y[i & 3] = fmaf(fi, v[i], y[i & 3]);
                }
            }
            const float total = kd_four(sum);
            const int tok = by_g(col0 + col), mma = at / 16, half = (at >> 3) & 1, d = (at & 7) * (HD / 8) + 8 * (mma >> 2) + 4 * half + (mma & 3);
            out[((size_t)(t0 + tok) * Hq + kvh * G + col0 + col - tok * G) * HD + d] = from_f32<bf16>(total == 0.f ? 0.f : kd_four(y) / total);
        }
        kd_cluster_sync();                                  // nobody leaves while its shared memory is read
    }
}

// Joins the runs of a row: a block a row, a warp every fourth run, all loads on their way together.  What says how many runs there are was
// there before the attention's blocks began, so it is read while the last of them still run (the kernel starts under their tail).
#define KJ_WARPS 4              // the four sums
template <int HD>
__global__ void __launch_bounds__(KJ_WARPS * 32)
kv4_attn_join_kernel(const float* part_o, const float* part_ml, const int* cu_seqlens, const int* pos0, const int* tok_seq, bf16* __restrict__ out, int T, int B,
                     int Hq, int head0, int heads, int table_width, int window, int max_runs) {
    __shared__ float join_o[KJ_WARPS][HD], join_l[KJ_WARPS];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, t = blockIdx.x / heads;
    const size_t row = blockIdx.x, to = (size_t)t * Hq + head0 + (blockIdx.x - t * heads);
    const int b = __ldcg(tok_seq + t);
    int runs = 0;
    if (b >= 0 && b < B) {
        const int t0 = __ldcg(cu_seqlens + b), t1 = __ldcg(cu_seqlens + b + 1), p0 = __ldcg(pos0 + b);
        runs = min(kv4_runs(p0, p0 + min(t1, T) - t0, window, table_width).runs, max_runs);
    }
    pdl_wait();
    pdl_launch_dependents();
    if (runs <= 1) return;
    constexpr int E = HD / 32;
    const float* mls = part_ml + row * max_runs * 2;
    float top = -INFINITY;
    for (int i = lane; i < runs; i += 32) top = fmaxf(top, __ldcg(mls + 2 * i));
    top = warp_max(top);
    float sum = 0.f, y[E] = {};
#pragma unroll 4
    for (int i = warp; i < runs; i += KJ_WARPS) {           // this warp's of the four sums
        const float2 x = __ldcg(reinterpret_cast<const float2*>(mls + 2 * i));
        float v[E];
        const float* src = part_o + (row * max_runs + i) * HD + lane * E;
        if constexpr (E == 4) *reinterpret_cast<float4*>(v) = __ldcg(reinterpret_cast<const float4*>(src));
        else *reinterpret_cast<float2*>(v) = __ldcg(reinterpret_cast<const float2*>(src));
        const float f = kd_share(x.x, x.y, top), fl = f * x.y;
        if (x.y != 0.f) {                                   // (0: a run that the row sees nothing of)
            sum += fl;
#pragma unroll
            for (int e = 0; e < E; ++e) y[e] = fmaf(f, v[e], y[e]);
        }
    }
#pragma unroll
    for (int e = 0; e < E; ++e) join_o[warp][lane * E + e] = y[e];
    if (lane == 0) join_l[warp] = sum;
    __syncthreads();
    for (int at = threadIdx.x; at < HD; at += KJ_WARPS * 32) {
        const float l[4] = {join_l[0], join_l[1], join_l[2], join_l[3]}, o[4] = {join_o[0][at], join_o[1][at], join_o[2][at], join_o[3][at]};
        const float total = kd_four(l);
        const int mma = at / 16, half = (at >> 3) & 1, d = (at & 7) * (HD / 8) + 8 * (mma >> 2) + 4 * half + (mma & 3);
        out[to * HD + d] = from_f32<bf16>(total == 0.f ? 0.f : kd_four(o) / total);
    }
}

// The most runs of a sequence of up to max_len tokens of which it brings up to max_new.
static long long kv4_max_runs(long long max_len, int max_new, int window, int table_width) {
    long long pages = (max_len + KV4_PAGE - 1) / KV4_PAGE;
    if (window > 0 && ((long long)window + max_new) / KV4_PAGE + 2 < pages) pages = ((long long)window + max_new) / KV4_PAGE + 2;
    if (pages > table_width) pages = table_width;
    if (pages <= KD_RUNS) return pages < 1 ? 1 : pages;
    const long long even = (pages + KD_RUN_PAGES - 1) / KD_RUN_PAGES;
    return even > KD_RUNS ? even : KD_RUNS;
}
static int kv4_columns(int max_new, int G) { return (long long)max_new * G > 8 ? 16 : 8; }      // of a block
static int kv4_cluster_size(long long runs) {
    int size = 1;
    while (size < runs) size *= 2;
    return size;
}

// Whether a step that brings more than a few tokens is faster with its pages read as bfloat16 once and the tcgen05 prompt kernel.  That kernel
// reaches six times the rate, but the pages go through memory twice more; as rows every run of every 16 columns is a block, with a start and an
// end that cost as much as 3.5 pages.  Both in microseconds, from measurements (32 query and 8 key heads of 128, as rows / read, with 8, 32 and 128
// new tokens a sequence): one sequence of 1,000 tokens 11 / 19, 15 / 18, 38 / 18; of 8,192 16 / 34, 40 / 32, 121 / 44; of 60,000 68 / 119, 205 / 121, 769 / 186;
// 8 of 8,192 66 / 91, 219 / 151, 743 / 212; a whole prompt of 128 15 / 9, of 900 262 / 24.  Steps of unequal sequences: a prompt of 4,096 beside 63 single
// tokens behind 4,095 10,711 / 864, of 512 1,187 / 470, of 2,048 beside 31 behind 16,383 5,070 / 999, of 512 beside 7 behind 4,095 232 / 105, of 128 beside 15
// 95 / 124.  (The rule is wrong for 300 new tokens beside 31 single ones, all behind 8,000: 608 / 497, goes as rows.)
// tokens, listed: the step's tokens and its sequences' pages (which say more of unequal sequences than the most of each).
static bool kv4_read_is_faster(int max_len, int max_new, int window, int table_width, int B, int Hq, int Hkv, int hd, int tokens, int listed) {
    const int G = Hq / Hkv;
    if (G > 64 || listed <= 0 || (long long)max_new * G <= 16) return false;
    if (max_new > max_len) max_new = max_len;
    long long mean_len = (long long)listed * KV4_PAGE / B;
    if (mean_len > max_len) mean_len = max_len;
    const Kv4Runs cut = kv4_runs(mean_len > max_new ? (int)(mean_len - max_new) : 0, (int)mean_len, window, table_width);
    const double columns = (double)tokens * G / 16.0 + 0.5 * B;
    const double rows = 5.0 + columns * Hkv * cut.runs * (cut.per_run + 3.5) / (hd == 128 ? 400.0 : 580.0);
    return 4.0 + at_pieces(tokens, B, max_new, max_len, Hq, Hkv, hd, window).us + (double)listed * Hkv * (hd == 128 ? 0.0065 : 0.0045) < rows;
}

// Whether a step is more than the rows kernel's grid, or its division by the group, takes: one whose longest prompt is of 2^20 / group tokens, for instance.
static bool kv4_rows_refuse(int T, int B, int max_new, int Hq, int Hkv, long long max_runs) {
    const int columns = kv4_columns(max_new, Hq / Hkv);
    const long long tiles = ((long long)max_new * (Hq / Hkv) + columns - 1) / columns;
    return tiles * columns >= 1 << 20 || tiles * max_runs > 2147483647ll || Hkv > 65535 || B > 65535 || (long long)T * Hq > 2147483647ll;
}

// How a call goes: the most runs of a sequence, times 8, plus 4 if it cannot go as rows, plus 2 if its runs are joined by scratch memory and a second
// kernel, plus 1 if reading the pages first is faster.  Up to 16 runs go as clusters, up to 64 of these and while they are all on the chip at once (7 blocks an SM, 4 with
// 16 columns): a second launch and a kernel's start less, 8.0 and 7.0 us for one sequence of 2,048 tokens, 15.0 and 13.6 for 16,384; 8 sequences
// of 4,096, 1,024 blocks, are even.  Beyond that a cluster waits for 16 free places, and many small ones start slowly: 64 sequences of 1,000 take 66.8
// us against 36.6, 4 of 8,192 with 6 new tokens 45.7 against 30.9, one prompt of 128, 256 clusters of 2, 26 against 16.
extern "C" int qwb_kv4_plan(int max_len, int max_new, int window, int table_width, int B, int Hq, int Hkv, int hd, int tokens, int listed) {
    if (B <= 0 || Hkv <= 0 || Hq < Hkv) return 8 + 4;                   // nothing that could go as rows
    const long long runs = kv4_max_runs(max_len, max_new, window, table_width);
    const int columns = kv4_columns(max_new, Hq / Hkv);
    const long long tiles = ((long long)max_new * (Hq / Hkv) + columns - 1) / columns;
    const bool clusters = runs <= KD_CLUSTER && tiles * Hkv * B <= 64 && tiles * kv4_cluster_size(runs) * Hkv * B <= 148 * (columns == 8 ? 7 : 4);
    const bool refused = kv4_rows_refuse(tokens, B, max_new, Hq, Hkv, runs), read = kv4_read_is_faster(max_len, max_new, window, table_width, B, Hq, Hkv, hd, tokens, listed);
    return (int)(8 * runs) + (refused ? 4 : 0) + (runs > 1 && !clusters ? 2 : 0) + (read ? 1 : 0);
}

template <int HD, int NT>
static int kv4_launch_rows(const bf16* q, const unsigned char* pool, const int* page_table, const int* cu, const int* pos0, const int* tok_seq, bf16* out,
                           float* scratch, int T, int B, int pool_pages, int max_new, int Hq, int Hkv, int table_width, float scale, int window, int max_runs,
                           int heads, cudaStream_t stream) {
    using Smem = KdSmem<HD, NT>;
    static_assert(Smem::BYTES <= 48 * 1024, "more needs an attribute of the kernel");
    const long long tiles = ((long long)max_new * (Hq / Hkv) + 8 * NT - 1) / (8 * NT);
    if (kv4_rows_refuse(T, B, max_new, Hq, Hkv, max_runs))
        return qwb_fail(QWB_ERR_ARG, "kv4_attention: %d sequences of up to %d new tokens, %d heads: too many blocks as rows", B, max_new, Hq);
    const float log2_scale = scale * 1.4426950408889634f;
    if (!scratch) {
        auto kernel = kv4_attn_rows_kernel<HD, NT, true, NT == 1 ? 7 : 4>;
        const int size = kv4_cluster_size(max_runs);
        if (size > 8) {                                     // more than 8 blocks have to be allowed, once a device
            static bool allowed[64];
            int device = 0;
            cudaError_t e = cudaGetDevice(&device);
            if (e == cudaSuccess && (device < 0 || device >= 64 || !allowed[device])) {
                e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
                if (e == cudaSuccess && device >= 0 && device < 64) allowed[device] = true;
            }
            if (e != cudaSuccess) return qwb_fail(QWB_ERR_CUDA, "kv4_attention: %s", cudaGetErrorString(e));
        }
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3((unsigned)(tiles * size), Hkv, B);
        cfg.blockDim = dim3(KD_WARPS * 32);
        cfg.dynamicSmemBytes = Smem::BYTES;
        cfg.stream = stream;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = size;
        attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, q, pool, page_table, cu, pos0, out, (float*)nullptr, (float*)nullptr, T, B, pool_pages, Hq / Hkv, Hkv,
                                                 table_width, log2_scale, window, (int)tiles, size, 0);
        if (e != cudaSuccess) return qwb_fail(QWB_ERR_CUDA, "kv4_attention: %s", cudaGetErrorString(e));
        return qwb_check_launch("kv4_attention");
    }
    const int G = Hq / Hkv;
    float* part_ml = scratch + (size_t)T * heads * G * max_runs * HD;
    auto kernel = tiles * max_runs * Hkv * B <= 148 * 4 ? kv4_attn_rows_kernel<HD, NT, false, NT == 1 ? 7 : 4> : kv4_attn_rows_kernel<HD, NT, false, NT == 1 ? 7 : 5>;
    for (int kv0 = 0; kv0 < Hkv; kv0 += heads) {            // `heads` key/value heads at a time share the scratch memory
        const int n = heads < Hkv - kv0 ? heads : Hkv - kv0;
        qwb_launch(kernel, dim3((unsigned)(tiles * max_runs), n, B), KD_WARPS * 32, Smem::BYTES, stream, q, pool, page_table, cu, pos0, out,
                   scratch, part_ml, T, B, pool_pages, G, Hkv, table_width, log2_scale, window, (int)tiles, max_runs, kv0);
        qwb_launch_early(kv4_attn_join_kernel<HD>, dim3((unsigned)((long long)T * n * G)), KJ_WARPS * 32, 0, stream, scratch, part_ml, cu, pos0, tok_seq, out, T, B, Hq,
                         kv0 * G, n * G, table_width, window, max_runs);
    }
    return qwb_check_launch("kv4_attention");
}

// max_runs, and whether there is scratch memory: as qwb_kv4_plan says, or with scratch memory anyway.  With it `heads` key/value heads go at a time (others: all
// of them), and it holds T * heads * (Hq / Hkv) * max_runs * (hd + 2) floats.
extern "C" int qwb_kv4_attn_rows(const void* q, const unsigned char* pool, const int* page_table, const int* cu, const int* pos0, const int* tok_seq,
                                 void* out, float* scratch, int T, int B, int pool_pages, int max_new, int Hq, int Hkv, int hd, int table_width, float scale,
                                 int window, int max_runs, int heads, cudaStream_t stream) {
    if (T <= 0) return 0;
    if (heads <= 0 || heads > Hkv) return qwb_fail(QWB_ERR_ARG, "kv4_attention: %d of %d key/value heads at a time", heads, Hkv);
    if (Hkv <= 0 || Hq <= 0 || Hq % Hkv || (hd != 64 && hd != 128) || table_width <= 0 || window < 0 || max_new <= 0 || max_runs <= 0 || B <= 0 || !(scale > 0.f))
        return qwb_fail(QWB_ERR_ARG, "kv4_attention: heads of 64 or 128 only, a scale above 0: Hq=%d Hkv=%d hd=%d width=%d window=%d scale=%g", Hq, Hkv, hd, table_width, window,
                        (double)scale);
    if (max_runs > KD_CLUSTER && !scratch) return qwb_fail(QWB_ERR_ARG, "kv4_attention: no scratch for %d runs", max_runs);
    if ((uintptr_t)q % 16 || (uintptr_t)pool % 16) return qwb_fail(QWB_ERR_ARG, "kv4_attention: q and the pool must start at a multiple of 16 bytes");
    const int columns = kv4_columns(max_new, Hq / Hkv);
#define KV4_ROWS(HD, NT) kv4_launch_rows<HD, NT>((const bf16*)q, pool, page_table, cu, pos0, tok_seq, (bf16*)out, scratch, T, B, pool_pages, max_new, Hq, Hkv, \
                                                 table_width, scale, window, max_runs, heads, stream)
    if (hd == 128) return columns == 16 ? KV4_ROWS(128, 2) : KV4_ROWS(128, 1);
    return columns == 16 ? KV4_ROWS(64, 2) : KV4_ROWS(64, 1);
#undef KV4_ROWS
}
