// The write into the cache in 4 bits, and its pages back as bfloat16 or 32-bit numbers.
#include "kv4.cuh"

// The code of a number of a group with step s > 0 and zero point z.  The quotient's rounding to 32 bits can put a number on the
// wrong side of the border between two codes; x - (c + 1/2) s in 64 bits tells (ties go to the even quotient, as rint has it).
__device__ __forceinline__ int kv4_code(double x, float s, float z) {
    float c = rintf((float)x / s);
    const double r = fma(-(double)c, (double)s, x), half = 0.5 * (double)s;
    if (r > half || (r == half && ((int)c & 1))) c += 1.f;
    else if (r < -half || (r == -half && ((int)c & 1))) c -= 1.f;
    return (int)fminf(fmaxf(c + z, 0.f), 15.f);
}

// Step and zero point of a group from its lowest and highest number (0 among them): the word, and both as floats.
__device__ __forceinline__ uint32_t kv4_word(double lo, double hi, bool finite, float& s, float& z) {
    const double t = (hi - lo) / 15.0;
    const long long up = __double_as_longlong(t) + (1ll << 48);                         // to 4 significant bits: 3 of the 52 behind the point stay
    const double step = __longlong_as_double(up & ~((1ll << 49) - 1));
    s = z = 0.f;
    if (!finite || !(step < 1.329227995784916e36)) return 0x7fc0u;
    if (step < 1.1754943508222875e-38) return 0u;
    s = (float)step;
    z = (float)fmin(rint(-lo / step), 15.0);
    return (__float_as_uint(s) >> 16) | (uint32_t)z;
}

// One warp a (token, head): queries, then key heads, then value heads, in the order of the fused projection's columns.  Keys
// and values go through 64 bits: the norm, the rotation and the choice of the codes are the formula's whatever the order of
// the sums, and a code is a choice, not a number that could be off by a little.  Queries are made in 32 bits, as for the cache in
// 16 bits.
#define KS_WARPS 4
template <typename TQ>
__global__ void __launch_bounds__(KS_WARPS * 32)
kv4_store_kernel(const float* __restrict__ qkv, const float* __restrict__ q_weight, const float* __restrict__ k_weight,
                 const float* __restrict__ cos_t, const float* __restrict__ sin_t, const int* __restrict__ slot_map,
                 TQ* __restrict__ q_out, unsigned char* __restrict__ pool, long long n_rows, int Hq, int Hkv, int hd, int rot,
                 float eps, int store_kv) {
    pdl_wait();
    pdl_launch_dependents();
    __shared__ double rows[KS_WARPS][KV4_MAX_DIM];
    const int t = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int head = blockIdx.y * KS_WARPS + warp, n_heads = Hq + 2 * Hkv;
    if (head >= n_heads) return;
    const bool is_q = head < Hq, is_k = !is_q && head < Hq + Hkv;
    const float* src = qkv + ((size_t)t * n_heads + head) * hd;
    const int half = rot >> 1;
    const float* c = cos_t + (size_t)t * half;
    const float* sn = sin_t + (size_t)t * half;
    if (is_q) {
        float scale = 1.f;
        if (q_weight) {
            float ss = 0.f;
            for (int i = lane; i < hd; i += 32) ss += src[i] * src[i];
            scale = 1.f / sqrtf(warp_sum(ss) / (float)hd + eps);
        }
        TQ* dst = q_out + ((size_t)t * Hq + head) * hd;
        for (int i = lane; i < half; i += 32) {
            float a = src[i] * scale, b = src[i + half] * scale;
            if (q_weight) { a *= q_weight[i]; b *= q_weight[i + half]; }
            dst[i] = from_f32<TQ>(a * c[i] - b * sn[i]);
            dst[i + half] = from_f32<TQ>(a * sn[i] + b * c[i]);
        }
        for (int i = rot + lane; i < hd; i += 32) dst[i] = from_f32<TQ>(q_weight ? src[i] * scale * q_weight[i] : src[i]);
        return;
    }
    const long long slot = slot_map[t];
    if (!store_kv || slot < 0 || slot >= n_rows) return;            // a token that has no place (behind the last sequence)
    double* row = rows[warp];
    if (is_k) {
        double scale = 1.0;
        if (k_weight) {
            double ss = 0.0;
            for (int i = lane; i < hd; i += 32) ss += (double)src[i] * src[i];
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
            scale = 1.0 / sqrt(ss / hd + (double)eps);
        }
        for (int i = lane; i < half; i += 32) {
            double a = src[i] * scale, b = src[i + half] * scale;
            if (k_weight) { a *= k_weight[i]; b *= k_weight[i + half]; }
            row[i] = a * c[i] - b * sn[i];
            row[i + half] = a * sn[i] + b * c[i];
        }
        for (int i = rot + lane; i < hd; i += 32) row[i] = k_weight ? src[i] * scale * k_weight[i] : (double)src[i];
    } else {
        for (int i = lane; i < hd; i += 32) row[i] = src[i];
    }
    __syncwarp();
    const int kvh = is_k ? head - Hq : head - Hq - Hkv, at = (int)(slot % KV4_PAGE);
    unsigned char* base = pool + ((size_t)(slot / KV4_PAGE) * Hkv + kvh) * kv4_page_bytes(hd) + (is_k ? 0 : kv4_half_bytes(hd));
    for (int g = 0; g < hd / KV4_GROUP; ++g) {
        const double x = row[g * KV4_GROUP + lane];
        const bool finite = __all_sync(0xffffffffu, fabs(x) <= 3.4028234663852886e38);
        double lo = fmin(x, 0.0), hi = fmax(x, 0.0);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            lo = fmin(lo, __shfl_xor_sync(0xffffffffu, lo, o));
            hi = fmax(hi, __shfl_xor_sync(0xffffffffu, hi, o));
        }
        float s, z;
        const uint32_t word = kv4_word(lo, hi, finite, s, z);
        const int code = s > 0.f ? kv4_code(x, s, z) : 0;
        const int next = __shfl_down_sync(0xffffffffu, code, 1);
        if (!(lane & 1)) base[(size_t)at * (hd / 2) + (g * KV4_GROUP + lane) / 2] = (unsigned char)(code | (next << 4));
        if (lane == 0) reinterpret_cast<uint16_t*>(base + kv4_code_bytes(hd))[at * (hd / KV4_GROUP) + g] = (uint16_t)word;
    }
}

// The same for heads of 64 and 128 turned over all their numbers (or not at all), the common case.  HD / 8 lanes take a head: lane L of them
// holds the numbers 4L..4L+3 and HD/2 + 4L..: a number and its rotation partner lie in one lane, and each of its two fours in the group of
// 8 neighbouring lanes, so that norm and group cost three or four exchanges.  What bounds it is memory: 4 bytes read and (queries) 2 or (keys
// and values) 9/16 written a number.  So the choices are made in 32 bits where these leave no doubt: a number whose quotient by the step lies
// nearer to the border of two codes than its error can be, or a step nearer to the border of two roundings (about one head in 220), sends
// its head through 64 bits.  A step of 4,096 tokens of 32 + 2 x 8 heads: a warp a head 130 us, with 64 bits for
// every key 45, so 34 with the next head on its way in registers and 29 (4.8 TB/s) with two by cp.async; what is left is latency and 3.5 waves
// of blocks: 16,384 tokens run at 5.7 TB/s.
//
// Errors of a key in 32 bits, u = 2^-24: the sum of squares 8 + 4 additions, the mean and eps 1, halved by the root; the inverse root
// 4 (2 units of 2^-23): 11 u; times the weight and the number 2 u; the rotation's products and sum 2 u: of p c - r s it is 15 u (|p c| + |r s|)
// < 2^-20 (|p| + |r|) times the largest of |c|, |s| and 1; the largest of that in the 8 lanes is taken for both of their groups.
struct Kv4Choice { uint32_t codes, word; bool sure; };

__device__ __forceinline__ float kv4_max_nan(float a, float b) {
    float y;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
    return y;
}

// Four numbers of a lane in a group of 8 lanes' 32, each off by at most `off` (the same for the group): codes (the first in the lowest bits) and the
// group's word.  A number plus 3 x 2^22 is rounded to a whole one by the addition, and whole ones add up to the packed codes as floats: roundings
// and conversions as such have a fraction of the rate.  Codes are kept in range as sixteenths, whose lower end is an instruction's own.
__device__ __forceinline__ Kv4Choice kv4_four(const float (&x)[4], float off, unsigned mask) {
    float lo = 0.f, hi = 0.f;                                       // hi: a NaN stays one, and t below with it
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        lo = fminf(lo, x[i]);
        hi = kv4_max_nan(hi, x[i]);
    }
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) {
        lo = fminf(lo, __shfl_xor_sync(mask, lo, o));
        hi = kv4_max_nan(hi, __shfl_xor_sync(mask, hi, o));
    }
    Kv4Choice y;
    y.codes = y.word = 0;
    const float t = (hi - lo) * (1.f / 15.f);
    if (t == 0.f && off == 0.f) { y.sure = true; return y; }
    // t is off by 2 off / 15 and by less than 3 of its last places: is it that near to the border of two steps?  (Very small, very large and no
    // numbers: decided in 64 bits.)
    const int bits = __float_as_int(t), border = abs((bits & 0xfffff) - 0x80000);
    const float s = __int_as_float((bits + 0x80000) & ~0xfffff), whole = 12582912.f;
    float inv;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(s));
    const float z0 = fmaf(-lo, inv, whole) - whole, z = fminf(z0, 15.f);
    const float from = fmaf(z, 0.0625f, -0.0625f * whole);          // (z - whole) / 16, exact
    float far = fabsf(fmaf(-z0, s, -lo)), packed = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float v = fmaf(x[i], inv, whole), c = v - whole;
        far = fmaxf(far, fabsf(fmaf(-c, s, x[i])));
        packed = fmaf(fminf(__saturatef(fmaf(v, 0.0625f, from)), 0.9375f), (float)(16 << (4 * i)), packed);
    }
    y.sure = t > 1e-36f && t < 1e36f && (float)(border - 3) * (t * 5.9604644775390625e-8f) > 0.14f * off && far + off < 0.499996f * s;
    y.codes = __float_as_uint(packed + 8388608.f) & 0xffffu;
    y.word = (__float_as_uint(s) >> 16) | (__float_as_uint(z + 8388608.f) & 15u);
    return y;
}
// The same in 64 bits, for both fours of a lane and from the projection's numbers on (weight and cosines null: as they are).
template <int HD>
__device__ __noinline__ uint4 kv4_head_exactly(const float* src, const float* weight, const float* cos_t, const float* sin_t, int L, float eps, unsigned mask) {
    double x[8], scale = 1.0;
    if (weight) {
        double ss = 0.0;
        for (int i = 0; i < 4; ++i) ss += (double)src[4 * L + i] * src[4 * L + i] + (double)src[HD / 2 + 4 * L + i] * src[HD / 2 + 4 * L + i];
        for (int o = 1; o < HD / 8; o <<= 1) ss += __shfl_xor_sync(mask, ss, o);
        scale = 1.0 / sqrt(ss / HD + (double)eps);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        double a = src[4 * L + i], b = src[HD / 2 + 4 * L + i];
        if (weight) {
            a *= scale * weight[4 * L + i];
            b *= scale * weight[HD / 2 + 4 * L + i];
        }
        const double c = cos_t ? (double)cos_t[4 * L + i] : 1.0, sn = cos_t ? (double)sin_t[4 * L + i] : 0.0;
        x[i] = cos_t ? a * c - b * sn : a;
        x[4 + i] = cos_t ? a * sn + b * c : b;
    }
    uint32_t out[4];
#pragma unroll
    for (int g = 0; g < 2; ++g) {
        double lo = 0.0, hi = 0.0;
        int finite = 1;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            finite &= fabs(x[4 * g + i]) <= 3.4028234663852886e38;
            lo = fmin(lo, x[4 * g + i]);
            hi = fmax(hi, x[4 * g + i]);
        }
        for (int o = 1; o < 8; o <<= 1) {
            lo = fmin(lo, __shfl_xor_sync(mask, lo, o));
            hi = fmax(hi, __shfl_xor_sync(mask, hi, o));
            finite &= __shfl_xor_sync(mask, finite, o);
        }
        float s, z;
        out[2 * g + 1] = kv4_word(lo, hi, finite, s, z);
        out[2 * g] = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (s > 0.f) out[2 * g] |= (uint32_t)kv4_code(x[4 * g + i], s, z) << (4 * i);
    }
    return make_uint4(out[0], out[1], out[2], out[3]);
}

template <typename TQ> __device__ __forceinline__ void kv4_put4(TQ* p, float a, float b, float c, float d);
template <> __device__ __forceinline__ void kv4_put4<float>(float* p, float a, float b, float c, float d) { *reinterpret_cast<float4*>(p) = make_float4(a, b, c, d); }
template <> __device__ __forceinline__ void kv4_put4<bf16>(bf16* p, float a, float b, float c, float d) {
    __nv_bfloat162 v[2] = {__floats2bfloat162_rn(a, b), __floats2bfloat162_rn(c, d)};
    *reinterpret_cast<uint2*>(p) = *reinterpret_cast<uint2*>(v);
}

__device__ __forceinline__ void kv4_copy16(void* dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src) : "memory");
}
#define KF_STAGES 3                 // heads in a warp's ring, two of them on their way: 4,096 tokens 29 us; one on its way 32, three 30, five 34
#define KF_BLOCKS 1184              // as many are wanted of a call
template <typename TQ, int HD>
__global__ void __launch_bounds__(KS_WARPS * 32, 8)
kv4_store_fast_kernel(const float* __restrict__ qkv, const float* __restrict__ q_weight, const float* __restrict__ k_weight,
                      const float* __restrict__ cos_t, const float* __restrict__ sin_t, const int* __restrict__ slot_map,
                      TQ* __restrict__ q_out, unsigned char* __restrict__ pool, long long n_rows, int Hq, int Hkv, float eps, int store_kv) {
    pdl_wait();
    pdl_launch_dependents();
    constexpr int LANES = HD / 8, HEADS = 32 / LANES;               // heads of a warp
    const int t = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, L = lane % LANES, of = lane / LANES;
    const unsigned mask = HD == 128 ? 0xffffu << (16 * of) : 0xffu << (8 * of);
    const int n_all = Hq + 2 * Hkv, n_heads = store_kv ? n_all : Hq;
    const float4* row = reinterpret_cast<const float4*>(qkv + (size_t)t * n_all * HD);
    // a lane's numbers of the next heads are on their way into its own places
    __shared__ float4 ring[KS_WARPS][KF_STAGES][2][32];
    const int step = gridDim.y * KS_WARPS * HEADS;
    int head = (blockIdx.y * KS_WARPS + warp) * HEADS + of, slot_in = 0, slot_out = 0;
    auto ask = [&](int h) {
        if (h < n_heads) {
            kv4_copy16(&ring[warp][slot_in][0][lane], row + (size_t)h * (HD / 4) + L);
            kv4_copy16(&ring[warp][slot_in][1][lane], row + (size_t)h * (HD / 4) + HD / 8 + L);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
        slot_in = slot_in == KF_STAGES - 1 ? 0 : slot_in + 1;
    };
#pragma unroll
    for (int i = 0; i < KF_STAGES - 1; ++i) ask(head + i * step);
    float c[4] = {1.f, 1.f, 1.f, 1.f}, sn[4] = {}, turn = 1.f;
    if (cos_t) {
        *reinterpret_cast<float4*>(c) = reinterpret_cast<const float4*>(cos_t + (size_t)t * (HD / 2))[L];
        *reinterpret_cast<float4*>(sn) = reinterpret_cast<const float4*>(sin_t + (size_t)t * (HD / 2))[L];
#pragma unroll
        for (int i = 0; i < 4; ++i) turn = fmaxf(turn, fmaxf(fabsf(c[i]), fabsf(sn[i])));
    }
    const int slot = slot_map[t], at = slot % KV4_PAGE;
    const bool has_place = slot >= 0 && slot < n_rows;
    unsigned char* page = pool + (has_place ? (size_t)(slot / KV4_PAGE) * Hkv * kv4_page_bytes(HD) : 0);
    for (; head < n_heads; head += step) {
        ask(head + (KF_STAGES - 1) * step);
        asm volatile("cp.async.wait_group %0;" ::"n"(KF_STAGES - 1) : "memory");
        float a[4], b[4];
        *reinterpret_cast<float4*>(a) = ring[warp][slot_out][0][lane];
        *reinterpret_cast<float4*>(b) = ring[warp][slot_out][1][lane];
        slot_out = slot_out == KF_STAGES - 1 ? 0 : slot_out + 1;
        if (head < Hq) {
            if (q_weight) {
                float ss = 0.f, w[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) ss = fmaf(a[i], a[i], fmaf(b[i], b[i], ss));
#pragma unroll
                for (int o = 1; o < LANES; o <<= 1) ss += __shfl_xor_sync(mask, ss, o);
                const float scale = rsqrtf(ss * (1.f / HD) + eps);
                *reinterpret_cast<float4*>(w) = reinterpret_cast<const float4*>(q_weight)[L];
#pragma unroll
                for (int i = 0; i < 4; ++i) a[i] *= scale * w[i];
                *reinterpret_cast<float4*>(w) = reinterpret_cast<const float4*>(q_weight)[HD / 8 + L];
#pragma unroll
                for (int i = 0; i < 4; ++i) b[i] *= scale * w[i];
            }
            float x[4], y[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                x[i] = a[i] * c[i] - b[i] * sn[i];
                y[i] = a[i] * sn[i] + b[i] * c[i];
            }
            TQ* dst = q_out + ((size_t)t * Hq + head) * HD + 4 * L;
            kv4_put4<TQ>(dst, x[0], x[1], x[2], x[3]);
            kv4_put4<TQ>(dst + HD / 2, y[0], y[1], y[2], y[3]);
            continue;
        }
        if (!has_place) continue;
        const bool is_k = head < Hq + Hkv;
        const int kvh = head - Hq - (is_k ? 0 : Hkv);
        unsigned char* base = page + (size_t)kvh * kv4_page_bytes(HD) + (is_k ? 0 : kv4_half_bytes(HD));
        const bool turned = is_k && (k_weight || cos_t);
        float w[4] = {1.f, 1.f, 1.f, 1.f}, u[4] = {1.f, 1.f, 1.f, 1.f}, x[4], y[4], off = 0.f;
        bool in_range = true;
        if (turned) {
            float scale = 1.f;
            if (k_weight) {
                float ss = 0.f;
#pragma unroll
                for (int i = 0; i < 4; ++i) ss = fmaf(a[i], a[i], fmaf(b[i], b[i], ss));
#pragma unroll
                for (int o = 1; o < LANES; o <<= 1) ss += __shfl_xor_sync(mask, ss, o);
                const float mean = ss * (1.f / HD) + eps;
                in_range = mean > 1e-30f && mean < 1e30f;           // else squares were lost or are too large: decided in 64 bits
                scale = rsqrtf(mean);
                *reinterpret_cast<float4*>(w) = reinterpret_cast<const float4*>(k_weight)[L];
                *reinterpret_cast<float4*>(u) = reinterpret_cast<const float4*>(k_weight)[HD / 8 + L];
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float p = a[i] * (scale * w[i]), r = b[i] * (scale * u[i]);
                x[i] = p * c[i] - r * sn[i];
                y[i] = p * sn[i] + r * c[i];
                off = fmaxf(off, fabsf(p) + fabsf(r));
            }
            off *= turn * 9.5367431640625e-7f;
#pragma unroll
            for (int o = 1; o < 8; o <<= 1) off = fmaxf(off, __shfl_xor_sync(mask, off, o));
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                x[i] = a[i];
                y[i] = b[i];
            }
        }
        Kv4Choice lo = kv4_four(x, off, mask), hi = kv4_four(y, off, mask);
        if (__any_sync(mask, !(in_range && lo.sure && hi.sure))) {
            const uint4 g = kv4_head_exactly<HD>(reinterpret_cast<const float*>(row) + (size_t)head * HD, turned ? k_weight : nullptr,
                                                 turned && cos_t ? cos_t + (size_t)t * (HD / 2) : nullptr, turned && cos_t ? sin_t + (size_t)t * (HD / 2) : nullptr,
                                                 L, eps, mask);
            lo.codes = g.x;
            lo.word = g.y;
            hi.codes = g.z;
            hi.word = g.w;
        }
        uint16_t* codes = reinterpret_cast<uint16_t*>(base + (size_t)at * (HD / 2));
        codes[L] = (uint16_t)lo.codes;
        codes[HD / 8 + L] = (uint16_t)hi.codes;
        if ((L & 7) == 0) {
            uint16_t* words = reinterpret_cast<uint16_t*>(base + kv4_code_bytes(HD)) + at * (HD / KV4_GROUP);
            words[L / 8] = (uint16_t)lo.word;
            words[HD / 64 + L / 8] = (uint16_t)hi.word;
        }
    }
}

template <typename TQ, int HD>
static void kv4_launch_store(const float* qkv, const float* q_weight, const float* k_weight, const float* cos_t, const float* sin_t, const int* slot_map,
                             void* q_out, unsigned char* pool, long long n_rows, int T, int Hq, int Hkv, float eps, int store_kv, cudaStream_t stream) {
    const int per_block = KS_WARPS * (256 / HD), heads = store_kv ? Hq + 2 * Hkv : Hq, most = (heads + per_block - 1) / per_block;
    int share = (KF_BLOCKS + T - 1) / T;                            // few tokens: several blocks share a token's heads
    if (share > most) share = most;
    qwb_launch(kv4_store_fast_kernel<TQ, HD>, dim3(T, share), KS_WARPS * 32, 0, stream, qkv, q_weight, k_weight, cos_t, sin_t, slot_map, (TQ*)q_out, pool, n_rows,
               Hq, Hkv, eps, store_kv);
}

extern "C" int qwb_kv4_store(const float* qkv, const float* q_weight, const float* k_weight, const float* cos_t, const float* sin_t,
                             const int* slot_map, void* q_out, int q_dtype, unsigned char* pool, int n_pages, int T, int Hq,
                             int Hkv, int hd, int rot, float eps, int store_kv, cudaStream_t stream) {
    if (T <= 0) return 0;
    if (Hq <= 0 || Hkv <= 0 || hd <= 0 || hd % KV4_GROUP || hd > KV4_MAX_DIM || rot < 0 || rot > hd || (rot & 1) || n_pages <= 0)
        return qwb_fail(QWB_ERR_ARG, "kv4_store: bad sizes Hq=%d Hkv=%d hd=%d rot=%d pages=%d", Hq, Hkv, hd, rot, n_pages);
    dim3 grid(T, (Hq + 2 * Hkv + KS_WARPS - 1) / KS_WARPS);
    if (grid.y > 65535) return qwb_fail(QWB_ERR_ARG, "kv4_store: too many heads (%d)", Hq + 2 * Hkv);
    const bool fast = (hd == 64 || hd == 128) && (rot == 0 || rot == hd) && (uintptr_t)qkv % 16 == 0 && (uintptr_t)q_out % 16 == 0 &&
                      (uintptr_t)cos_t % 16 == 0 && (uintptr_t)sin_t % 16 == 0 && (uintptr_t)q_weight % 16 == 0 && (uintptr_t)k_weight % 16 == 0 &&
                      (uintptr_t)pool % 2 == 0;
    if (fast && (q_dtype == QWB_DT_F32 || q_dtype == QWB_DT_BF16)) {
        auto launch = q_dtype == QWB_DT_F32 ? (hd == 128 ? kv4_launch_store<float, 128> : kv4_launch_store<float, 64>)
                                            : (hd == 128 ? kv4_launch_store<bf16, 128> : kv4_launch_store<bf16, 64>);
        launch(qkv, q_weight, k_weight, rot ? cos_t : nullptr, rot ? sin_t : nullptr, slot_map, q_out, pool, (long long)n_pages * KV4_PAGE, T, Hq, Hkv, eps,
               store_kv, stream);
        return qwb_check_launch("kv4_store");
    }
    if (q_dtype == QWB_DT_F32)
        qwb_launch(kv4_store_kernel<float>, grid, KS_WARPS * 32, 0, stream, qkv, q_weight, k_weight, cos_t, sin_t, slot_map, (float*)q_out, pool,
                   (long long)n_pages * KV4_PAGE, Hq, Hkv, hd, rot, eps, store_kv);
    else if (q_dtype == QWB_DT_BF16)
        qwb_launch(kv4_store_kernel<bf16>, grid, KS_WARPS * 32, 0, stream, qkv, q_weight, k_weight, cos_t, sin_t, slot_map, (bf16*)q_out, pool,
                   (long long)n_pages * KV4_PAGE, Hq, Hkv, hd, rot, eps, store_kv);
    else
        return qwb_fail(QWB_ERR_ARG, "kv4_store: unknown dtype %d", q_dtype);
    return qwb_check_launch("kv4_store");
}

// Pages of a step's sequences, one after the other, as plain pages [P, heads, 64, hd] of keys and of values (of the pool's heads from head0 on); rows behind a
// sequence's last token are zeros.  A block takes a (page, head), a thread 8 numbers at a time (one 32-bit word of codes).
// `marked`: a token one of whose values is not finite has values of zero and keys of NaN here, so that a kernel that multiplies
// what a query does not see by 0 gives NaN to the queries that see it only.
// The blocks also write the table that names these pages: [B, width], page_start[b] + j or 0 where a sequence has none (with `marked` -1, there and where
// the pool does not have the page: the kernel that takes the table then sees nothing of it); and with `rows_out` they set rows of
// `row_bytes` (a multiple of 16) behind row `rows_used` of `rows` there to zero (what no sequence of a padded step writes).
struct Kv4ReadArgs {
    const unsigned char* pool;
    const int *pages, *page_start, *seq_len, *rows_used;
    int* table;
    uint4* rows_out;
    int B, width, pool_pages, Hkv, head0, hd, marked, rows, row_bytes;
};
// The table and the rows; then what this block's page holds: its bytes of this head, and how many rows of it live.
__device__ __forceinline__ const unsigned char* kv4_read_begin(const Kv4ReadArgs& a, int hd, int& live) {
    const int entry = blockIdx.x, head = a.head0 + blockIdx.y;
    const long long me = ((long long)blockIdx.y * gridDim.x + entry) * blockDim.x + threadIdx.x, all = (long long)gridDim.x * gridDim.y * blockDim.x;
    for (long long i = me; i < (long long)a.B * a.width; i += all) {
        const int b = (int)(i / a.width), j = (int)(i - (long long)b * a.width), at = a.page_start[b] + j;
        const bool listed = at >= 0 && at < a.page_start[b + 1] && at < (int)gridDim.x;
        int entry = listed ? at : 0;
        if (a.marked) {
            const int page = listed ? a.pages[at] : -1;
            if (page < 0 || page >= a.pool_pages) entry = -1;
        }
        a.table[i] = entry;
    }
    if (a.rows_out) {
        const long long end = (long long)a.rows * (a.row_bytes / 16);
        for (long long i = (long long)max(*a.rows_used, 0) * (a.row_bytes / 16) + me; i < end; i += all) a.rows_out[i] = make_uint4(0, 0, 0, 0);
    }
    // the sequence that holds this entry: the last one that begins at or before it
    int lo = 0, hi = a.B;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (a.page_start[mid] <= entry) lo = mid; else hi = mid;
    }
    const int j = entry - a.page_start[lo];
    const long long page = a.pages[entry];
    live = entry < a.page_start[lo + 1] ? min(max(a.seq_len[lo] - j * KV4_PAGE, 0), KV4_PAGE) : 0;
    if (j < 0 || page < 0 || page >= a.pool_pages) live = 0;
    return a.pool + ((size_t)(live ? page : 0) * a.Hkv + head) * kv4_page_bytes(hd);
}

template <typename T>
__global__ void __launch_bounds__(256)
kv4_read_kernel(const Kv4ReadArgs a, T* __restrict__ k_out, T* __restrict__ v_out) {
    pdl_wait();
    pdl_launch_dependents();
    int live;
    const int hd = a.hd, words = hd / 8, groups = hd / KV4_GROUP;
    const unsigned char* base = kv4_read_begin(a, hd, live);
    const size_t out0 = ((size_t)blockIdx.x * gridDim.y + blockIdx.y) * KV4_PAGE * hd;
    const uint16_t* v_words = reinterpret_cast<const uint16_t*>(base + kv4_half_bytes(hd) + kv4_code_bytes(hd));
    for (int i = threadIdx.x; i < 2 * KV4_PAGE * words; i += 256) {
        const bool is_v = i >= KV4_PAGE * words;
        const int at = is_v ? i - KV4_PAGE * words : i, row = at / words, w = at - row * words;
        const unsigned char* part = base + (is_v ? kv4_half_bytes(hd) : 0);
        T* dst = (is_v ? v_out : k_out) + out0 + (size_t)at * 8;
        uint32_t codes = 0, word = 0;
        float s = 0.f;
        if (row < live) {
            codes = reinterpret_cast<const uint32_t*>(part)[at];
            word = reinterpret_cast<const uint16_t*>(part + kv4_code_bytes(hd))[row * groups + w / 4];
            s = kv4_step(word);
            bool bad = false;
            for (int g = 0; a.marked && g < groups; ++g) bad |= kv4_is_nan(v_words[row * groups + g]);
            if (bad) s = is_v ? 0.f : __uint_as_float(0x7fffffffu);
        }
        const float z = kv4_zero(word);
#pragma unroll
        for (int n = 0; n < 8; ++n) dst[n] = from_f32<T>(((float)((codes >> (4 * n)) & 15u) - z) * s);
    }
}

// bfloat16, heads of 64 and 128: a thread takes the same 8 numbers of every 16th (32nd) row, all its loads on their way before the first
// is used, and two codes at a time, all of it exact: c s - z s.  What bounds it: 32 KB written a page and head of 128 for 9 KB read; 7,500 of them
// 54 us, 5.8 TB/s (one word and its address at a time 82).
// Registers for 8 blocks an SM with heads of 64: with the 39 that it takes by itself three chunks of 900 over it 93.8 us instead of 91.5.
template <int HD>
__global__ void __launch_bounds__(256, HD == 64 ? 8 : 4)
kv4_read_fast_kernel(const Kv4ReadArgs a, bf16* __restrict__ k_out, bf16* __restrict__ v_out) {
    pdl_wait();
    pdl_launch_dependents();
    constexpr int WORDS = HD / 8, ROWS = 256 / WORDS, PASSES = KV4_PAGE / ROWS, HALF = kv4_half_bytes(HD), CODES = kv4_code_bytes(HD);
    int live;
    const unsigned char* base = kv4_read_begin(a, HD, live);
    const int tid = threadIdx.x, w = tid % WORDS, r0 = tid / WORDS, g = w / 4;
    const unsigned twice = (2 * g) | (2 * g + 1) << 4 | (2 * g) << 8 | (2 * g + 1) << 12;          // selects the group's word twice
    uint32_t codes[2][PASSES];
    uint2 words[2][PASSES];
#pragma unroll
    for (int p = 0; p < 2; ++p)
#pragma unroll
        for (int i = 0; i < PASSES; ++i) {
            const int row = r0 + i * ROWS;
            codes[p][i] = 0;
            words[p][i] = make_uint2(0, 0);
            if (row < live) {
                codes[p][i] = reinterpret_cast<const uint32_t*>(base + p * HALF)[i * 256 + tid];
                if (HD == 128) words[p][i] = reinterpret_cast<const uint2*>(base + p * HALF + CODES)[row];
                else words[p][i].x = reinterpret_cast<const uint32_t*>(base + p * HALF + CODES)[row];
            }
        }
    const size_t out0 = ((size_t)blockIdx.x * gridDim.y + blockIdx.y) * KV4_PAGE * HD;
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
        const uint2 v = words[1][i];
        const bool bad = a.marked && (__vcmpeq2(v.x & 0x7f807f80u, 0x7f807f80u) | __vcmpeq2(v.y & 0x7f807f80u, 0x7f807f80u));
#pragma unroll
        for (int p = 0; p < 2; ++p) {
            const uint32_t word = __byte_perm(words[p][i].x, words[p][i].y, twice);
            uint32_t step = word & 0xfff0fff0u;
            if (bad) step = p ? 0u : 0x7fc07fc0u;
            const uint32_t off = kv4_off(step), zs = kv4_scaled(word, step, off);
            uint32_t x[4];
#pragma unroll
            for (int n = 0; n < 4; ++n) {
                const uint32_t cs = kv4_scaled(codes[p][i] >> (4 * n), step, off);
                const __nv_bfloat162 d = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&cs), *reinterpret_cast<const __nv_bfloat162*>(&zs));
                x[n] = *reinterpret_cast<const uint32_t*>(&d);
            }
            *reinterpret_cast<uint4*>((p ? v_out : k_out) + out0 + (size_t)(i * 256 + tid) * 8) =
                make_uint4(__byte_perm(x[0], x[1], 0x5410), __byte_perm(x[2], x[3], 0x5410), __byte_perm(x[0], x[1], 0x7632), __byte_perm(x[2], x[3], 0x7632));
        }
    }
}

extern "C" int qwb_kv4_read(const unsigned char* pool, const int* pages, const int* page_start, const int* seq_len, void* k_out,
                            void* v_out, int dtype, int* table, int P, int B, int width, int pool_pages, int Hkv, int head0,
                            int heads, int hd, int marked, void* rows_out, const int* rows_used, int rows, int row_bytes, cudaStream_t stream) {
    if (P <= 0) return 0;
    if (B <= 0 || width <= 0 || Hkv <= 0 || Hkv > 65535 || head0 < 0 || heads <= 0 || heads > Hkv - head0 || hd <= 0 || hd % KV4_GROUP || hd > KV4_MAX_DIM || pool_pages <= 0)
        return qwb_fail(QWB_ERR_ARG, "kv4_read: bad sizes B=%d width=%d Hkv=%d (%d from %d on) hd=%d pages=%d", B, width, Hkv, heads, head0, hd, pool_pages);
    if ((uintptr_t)pool % 16 || (uintptr_t)k_out % 16 || (uintptr_t)v_out % 16)
        return qwb_fail(QWB_ERR_ARG, "kv4_read: pool and outputs must start at a multiple of 16 bytes");
    if (rows_out && ((uintptr_t)rows_out % 16 || row_bytes % 16 || !rows_used))
        return qwb_fail(QWB_ERR_ARG, "kv4_read: rows of %d bytes", row_bytes);
    const Kv4ReadArgs args = {pool, pages, page_start, seq_len, rows_used, table, (uint4*)rows_out, B, width, pool_pages, Hkv, head0, hd, marked, rows, row_bytes};
    const dim3 grid(P, heads);
    // early: its blocks wait at their beginning, its launch does not; one token's write and read 4.7 -> 4.1 us
    if (dtype == QWB_DT_F32) qwb_launch_early(kv4_read_kernel<float>, grid, 256, 0, stream, args, (float*)k_out, (float*)v_out);
    else if (dtype != QWB_DT_BF16) return qwb_fail(QWB_ERR_ARG, "kv4_read: unknown dtype %d", dtype);
    else if (hd == 128) qwb_launch_early(kv4_read_fast_kernel<128>, grid, 256, 0, stream, args, (bf16*)k_out, (bf16*)v_out);
    else if (hd == 64) qwb_launch_early(kv4_read_fast_kernel<64>, grid, 256, 0, stream, args, (bf16*)k_out, (bf16*)v_out);
    else qwb_launch_early(kv4_read_kernel<bf16>, grid, 256, 0, stream, args, (bf16*)k_out, (bf16*)v_out);
    return qwb_check_launch("kv4_read");
}
