// Pages of keys and values in 8 bits: what the kernels that write, read and unpack them share.
//
// A page is a row of bytes: [2 (keys, values)][kv heads][page size][head size] in e4m3 (four bits of exponent, three of
// mantissa, no infinity, 0x7f and 0xff are no number), then [2][kv heads] scale bytes, padded to a multiple of 128. The
// scale byte e of a block (one page of one key/value head, keys and values apart) stands for 2^(e - 127), and 0 for 0: a
// block of zeros, or one that nothing was stored to. Scales are powers of two, so that a stored value is exact in
// bfloat16 and raising a block's scale only moves the exponents of what it holds (values that become subnormal are
// rounded once more, by at most half of 2^-9 of the new scale).
#pragma once
#include "common.cuh"

#define KV8_MAX_SCALE 247                            // 448 * 2^(247 - 127) is the first such bound beyond the largest float32

__host__ __device__ inline long kv8_body_bytes(int nkv, int page_size, int d) { return 2L * nkv * page_size * d; }
__host__ __device__ inline long kv8_page_bytes(int nkv, int page_size, int d) {
    return (kv8_body_bytes(nkv, page_size, d) + 2L * nkv + 127) / 128 * 128;
}

// 2^n for -126 <= n <= 127
__device__ __forceinline__ float kv8_power(int n) { return __int_as_float((n + 127) << 23); }
// What a scale byte stands for.
__device__ __forceinline__ float kv8_scale(unsigned e) { return __uint_as_float(e << 23); }

// The smallest scale byte in 1..KV8_MAX_SCALE whose block holds magnitudes up to amax (finite), 448 being e4m3's largest:
// with amax = 1.m * 2^(E - 127) that is E - 8, and one more where 1.m is beyond 1.75. 0 for an amax of 0.
__device__ __forceinline__ int kv8_needed(float amax) {
    const unsigned bits = __float_as_uint(amax);
    if (bits == 0u) return 0;
    int e = (int)(bits >> 23) - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
    if (e < 1) e = 1;
    if (e > KV8_MAX_SCALE) e = KV8_MAX_SCALE;
    return e;
}

// Two floats of at most 448 to e4m3, to nearest even; what is no number stays none. lo in the low byte.
__device__ __forceinline__ unsigned kv8_pack2(float lo, float hi) {
    unsigned short r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;\n" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ unsigned kv8_pack4(float a, float b, float c, float d) { return kv8_pack2(a, b) | (kv8_pack2(c, d) << 16); }

// Two values in e4m3 as a pair of half-precision numbers (every value of e4m3 is one).
__device__ __forceinline__ unsigned kv8_half2(unsigned short two) {
    unsigned r;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;\n" : "=r"(r) : "h"(two));
    return r;
}
__device__ __forceinline__ float2 kv8_unpack2(unsigned short two) {
    const unsigned h = kv8_half2(two);
    float2 f;
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.f32.f16 %0, l;\n\tcvt.f32.f16 %1, h;\n\t}\n" : "=f"(f.x), "=f"(f.y) : "r"(h));
    return f;
}
__device__ __forceinline__ void kv8_unpack4(unsigned word, float (&v)[4]) {
    const float2 a = kv8_unpack2((unsigned short)word), b = kv8_unpack2((unsigned short)(word >> 16));
    v[0] = a.x; v[1] = a.y; v[2] = b.x; v[3] = b.y;
}
