// What the kernels over an 8-bit cache share: its numbers (cache8.cu says what they are) and the arguments of attention.
#pragma once
#include "common.cuh"

namespace vapi {

constexpr int C8_BLOCK = 16;                       // tokens of a head that share a scale
constexpr int C8_MIN_EXP = -110, C8_MAX_EXP = 119; // 448 * 2^119 is the largest bfloat16 of this form; below 2^-119 nothing is kept

struct C8Params {
    long long q_row_stride;
    const unsigned char* codes;
    const signed char* exps;
    const int* block_table; int table_stride;
    const int* cu_q; const int* seqlens_k;
    int nh, nkv, d, page_size, num_pages;
    float scale_log2e;
    int window;
    int settled;                                   // keys before a sequence's own tokens were written by what has ended, whatever still runs
    int* status;
};

// The exponents of the block of keys at `where` and of its values, a byte each.  (From L2: the line may have been read before the
// kernel that wrote this step's blocks had ended.)
__device__ __forceinline__ int c8_scales(const C8Params& p, int where, int per_head) {
    const unsigned char* e = reinterpret_cast<const unsigned char*>(p.exps);
    return (int)__ldcg(e + where) | (int)__ldcg(e + where + p.nkv * per_head) << 8;
}

// 2^e for e in -126 .. 127
__device__ __forceinline__ float c8_power(int e) { return __int_as_float((e + 127) << 23); }

// The smallest e with amax <= 448 * 2^e, within the limits, for a finite amax >= 0: amax = m * 2^x with 1 <= m < 2, 448 = 1.75 * 2^8.
__device__ __forceinline__ int c8_exponent(float amax) {
    const unsigned u = __float_as_uint(amax);
    const int e = (int)(u >> 23) - 127 - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
    return min(max(e, C8_MIN_EXP), C8_MAX_EXP);
}

// The nearest e4m3 number (ties to even), magnitudes above 448 as 448; NaN for what is not finite, so that it is seen again.
__device__ __forceinline__ unsigned char c8_code(float x) {
    unsigned short c;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(c) : "f"(0.f), "f"(x));
    return fabsf(x) < INFINITY ? (unsigned char)(c & 0xff) : (unsigned char)0x7f;
}

// Four codes, x the lowest byte.
__device__ __forceinline__ unsigned c8_codes4(float x, float y, float z, float w) {
    unsigned short lo, hi;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(y), "f"(x));
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(w), "f"(z));
    unsigned c = (unsigned)lo | (unsigned)hi << 16;
    if (!(fmaxf(fmaxf(fabsf(x), fabsf(y)), fmaxf(fabsf(z), fabsf(w))) < INFINITY) || x != x || y != y || z != z || w != w)
        c = (unsigned)c8_code(x) | (unsigned)c8_code(y) << 8 | (unsigned)c8_code(z) << 16 | (unsigned)c8_code(w) << 24;
    return c;
}

// Four codes as two pairs of halves, exactly; the lowest byte in the low half of `lo`.
__device__ __forceinline__ void c8_halves4(unsigned c, unsigned& lo, unsigned& hi) {
    asm("{\n.reg .b16 a, b;\nmov.b32 {a, b}, %2;\ncvt.rn.f16x2.e4m3x2 %0, a;\ncvt.rn.f16x2.e4m3x2 %1, b;\n}" : "=r"(lo), "=r"(hi) : "r"(c));
}
__device__ __forceinline__ float2 c8_pair(unsigned h) {          // two halves as floats
    float2 f;
    asm("{\n.reg .b16 a, b;\nmov.b32 {a, b}, %2;\ncvt.f32.f16 %0, a;\ncvt.f32.f16 %1, b;\n}" : "=f"(f.x), "=f"(f.y) : "r"(h));
    return f;
}

// Four codes as floats.
__device__ __forceinline__ float4 c8_floats(unsigned c) {
    unsigned lo, hi;
    c8_halves4(c, lo, hi);
    const float2 x = c8_pair(lo), y = c8_pair(hi);
    return make_float4(x.x, x.y, y.x, y.y);
}

// Four codes times f, rounded again.
__device__ __forceinline__ unsigned c8_rescale(unsigned c, float f) {
    const float4 v = c8_floats(c);
    return (unsigned)c8_code(v.x * f) | (unsigned)c8_code(v.y * f) << 8 | (unsigned)c8_code(v.z * f) << 16 | (unsigned)c8_code(v.w * f) << 24;
}

}  // namespace vapi
