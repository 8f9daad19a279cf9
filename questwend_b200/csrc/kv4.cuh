// The cache in 4 bits: what its bytes mean.
//
// A row is a token's key or value of one key/value head, hd numbers.  It is cut into groups of 32 neighbouring ones; with
// lo = min(x, 0) and hi = max(x, 0) over a group its step is s = (hi - lo) / 15, rounded to 4 significant bits, its zero
// point z = rint(-lo / s) in 0..15, a number's code c = rint(x / s) + z, kept in 0..15, and the number that it stands for
// (c - z) s.  c - z has 4 bits and s has 4, so that number is exact in bfloat16 and in 32 bits: whoever reads the cache, in
// whatever type and order, reads the same numbers.  (Rounding the step
// makes it 2 % larger or smaller on average, and the codes' own rounding, half a step at most, with it; the largest numbers may then lie up to
// 15/16 of a step beyond the last code instead of half a step.)
// A group of zeros, or whose step would lie under 2^-126, has step 0 and stands for zeros.  A group that holds a number that
// is not finite, or whose step would be 2^120 or more (so that 128 s is a number), stands for NaN: whoever sees the token gets NaN for all numbers
// of the head, in every form of the attention, and nothing is lost silently.
//
// A page of 64 tokens and one head: 64 rows of key codes (hd / 2 bytes, the lower half of a byte first), 64 rows of the
// keys' words (hd / 32 of 16 bits: the bits of s as a bfloat16, whose lowest 4 are zero, with z in them), then the values' codes
// and words.  With hd = 128 that is 9,216 bytes where bfloat16 takes 32,768.
#pragma once

#include "common.cuh"

#define KV4_PAGE 64
#define KV4_GROUP 32
#define KV4_MAX_DIM 256

__host__ __device__ constexpr int kv4_code_bytes(int hd) { return KV4_PAGE * hd / 2; }
__host__ __device__ constexpr int kv4_half_bytes(int hd) { return KV4_PAGE * (hd / 2 + hd / 16); }     // keys, or values
__host__ __device__ constexpr int kv4_page_bytes(int hd) { return 2 * kv4_half_bytes(hd); }

__device__ __forceinline__ float kv4_step(uint32_t word) { return __uint_as_float((word & 0xfff0u) << 16); }
__device__ __forceinline__ float kv4_zero(uint32_t word) { return (float)(word & 15u); }
__device__ __forceinline__ bool kv4_is_nan(uint32_t word) { return (word & 0x7f80u) == 0x7f80u; }

// Two codes c, in the lowest four bits of each half of `codes`, as the bfloat16 numbers c s: 128 + c by one and-or, then a fused
// multiply-add that takes 128 s off, exact throughout.  step: s twice; off: -128 s twice.
__device__ __forceinline__ uint32_t kv4_scaled(uint32_t codes, uint32_t step, uint32_t off) {
    uint32_t e;
    asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(e) : "r"(codes), "r"(0x000f000fu), "r"(0x43004300u));        // written as & and |, two instructions
    __nv_bfloat162 v = __hfma2(*reinterpret_cast<__nv_bfloat162*>(&e), *reinterpret_cast<__nv_bfloat162*>(&step), *reinterpret_cast<__nv_bfloat162*>(&off));
    return *reinterpret_cast<uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t kv4_off(uint32_t step) {
    __nv_bfloat162 v = __hmul2(*reinterpret_cast<__nv_bfloat162*>(&step), __floats2bfloat162_rn(-128.f, -128.f));
    return *reinterpret_cast<uint32_t*>(&v);
}
