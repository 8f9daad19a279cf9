// Attention over the cache in 4 bits (kv4.cuh), causal, grouped heads, with an optional window.
//
// The plain kernel: any head size that is a multiple of 32, queries in 32 bits or bfloat16.  A block takes a (token, query head),
// its four warps every fourth key; a lane holds the numbers lane, lane + 32, ... of the query, of the sums and of a key, so a
// group of 32 is a step of the loop over them.  Each warp keeps a running maximum, sum and output; they meet in shared memory.
#include "kv4.cuh"

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
            if (page < 0 || page >= pool_pages) break;
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
#pragma unroll
    for (int g = 0; g < KV4_MAX_DIM / 32; ++g)
        if (g < groups) part[warp][g * 32 + lane] = acc[g];
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
    if (Hkv <= 0 || Hq <= 0 || Hq % Hkv || Hq > 65535 || hd <= 0 || hd % KV4_GROUP || hd > KV4_MAX_DIM || table_width <= 0 || window < 0)
        return qwb_fail(QWB_ERR_ARG, "kv4_attention: bad sizes Hq=%d Hkv=%d hd=%d width=%d window=%d", Hq, Hkv, hd, table_width, window);
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
