// hkv_e4m3.cuh -- E4M3 blocks with a power-of-two scale: the arithmetic of the
// 8-bit cache format, shared by the kernels that write, read and attend it.
//
// A block holds values x as codes c with x ~ c * 2^e.  e is the least integer
// with max|x| <= 448 * 2^e over the block's finite values (448 = 1.75 * 2^8, the
// largest E4M3 number), so no code saturates and the rounding to 4 significant
// bits (nearest, ties to even) is the only error: at most 2^-4 of the value down
// to 2^-6 * 2^e, and 2^-10 * 2^e below that.  A power of two makes scaling exact,
// and when e grows because a larger row joins the block, the older codes move by
// an exponent: they keep their values unless they fall below the normal range.
// A value that is not finite is stored as E4M3's NaN and leaves e alone, so it
// poisons its own row and nothing else of its block.
#pragma once

#include <cuda_fp16.h>
#include <stdint.h>

namespace hkv {
namespace dev {

// Exponent of an all-zero block, and the least one: 448 * 2^-100 is far below
// any activation, and 2^100 * 2^-126 still leaves every scale a normal float.
constexpr int kExpMin = -100;

// 2^e, e in [-126, 127].
__device__ __forceinline__ float pow2(int e) { return __int_as_float((e + 127) << 23); }

// The least e with amax <= 448 * 2^e (amax finite, >= 0), at least kExpMin.
__device__ __forceinline__ int block_exponent(float amax) {
    const uint32_t u = __float_as_uint(amax);
    const int e = static_cast<int>(u >> 23) - 127 - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
    return max(e, kExpMin);
}

__device__ __forceinline__ float finite_abs(float x) {
    const float a = fabsf(x);
    return a <= 3.402823466e38f ? a : 0.f;
}

// Two values times inv (a power of two) as codes, lo in the low byte.
__device__ __forceinline__ uint32_t to_codes2(float lo, float hi, float inv) {
    const float nan = __int_as_float(0x7fffffff);
    const float a = fabsf(lo) <= 3.402823466e38f ? lo * inv : nan;
    const float b = fabsf(hi) <= 3.402823466e38f ? hi * inv : nan;
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(b), "f"(a));
    return r;
}
__device__ __forceinline__ uint32_t to_codes4(float4 x, float inv) {
    return to_codes2(x.x, x.y, inv) | (to_codes2(x.z, x.w, inv) << 16);
}

// Two codes (16 bits) as an F16 pair, exact: every E4M3 number is an F16 number.
__device__ __forceinline__ uint32_t codes_to_half2(uint32_t c) {
    uint32_t r;
    asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\t"
        "cvt.rn.f16x2.e4m3x2 %0, lo;\n\t}"
        : "=r"(r)
        : "r"(c));
    return r;
}
__device__ __forceinline__ uint32_t codes_to_half2_hi(uint32_t c) {
    uint32_t r;
    asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\t"
        "cvt.rn.f16x2.e4m3x2 %0, hi;\n\t}"
        : "=r"(r)
        : "r"(c));
    return r;
}
__device__ __forceinline__ float4 codes_to_float4(uint32_t c) {
    const uint32_t lo = codes_to_half2(c), hi = codes_to_half2_hi(c);
    const float2 a = __half22float2(*reinterpret_cast<const __half2 *>(&lo));
    const float2 b = __half22float2(*reinterpret_cast<const __half2 *>(&hi));
    return make_float4(a.x, a.y, b.x, b.y);
}

// Four codes of a block whose exponent grows by d > 0, rounded again.
__device__ __forceinline__ uint32_t rescale_codes4(uint32_t c, int d) {
    return to_codes4(codes_to_float4(c), pow2(max(-d, -126)));
}

}  // namespace dev
}  // namespace hkv
