// The format of the 8-bit key/value pages, shared by the kernels that write and read them.
//
// A block is 16 tokens of one kv head.  Keys lie as [pages][kv heads][page size][D], values transposed within a block as
// [pages][kv heads][page size / 16][D][16]; in both pools a block is 16 * D contiguous bytes and block number
// (page * kv heads + head) * (page size / 16) + (token in page) / 16 starts at byte number * 16 * D.  The scales are
// float [pages][kv heads][page size / 16], indexed by the same block number.
// An element is q * 2^e with q in e4m3 or int8 and 2^e the block's scale: the smallest power of two for which the block's
// largest magnitude fits (448 or 127 times it), e within [-40, 40].  Powers of two because the value of an element is then
// exact in bfloat16 (4 or 7 significant bits), because a block that grows can be encoded again by a shift (exact for e4m3
// but for its subnormals), and because it costs e4m3 no precision; int8 gives away up to one of its bits.
#pragma once
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "common.cuh"

enum { PI_E4M3 = 2, PI_INT8 = 3 };          // dtype codes of the pages, beside PI_F32 and PI_BF16

#define C8_BLOCK 16
#define C8_E_MIN (-40)
#define C8_E_MAX 40

// smallest e with amax <= qmax 2^e: amax = m 2^E with m in [1, 2); 448 = 1.75 * 2^8, 127 = 1.984375 * 2^6.
// amax is not negative and not NaN; subnormals fall to the lower limit as they should.
template <bool E4M3>
__device__ __forceinline__ int c8_exponent(float amax) {
    const unsigned bits = __float_as_uint(amax);
    const int E = (int)(bits >> 23) - 127;
    const unsigned mant = bits & 0x7fffffu;
    const int e = E4M3 ? E - 8 + (mant > 0x600000u ? 1 : 0) : E - 6 + (mant > 0x7e0000u ? 1 : 0);
    return max(C8_E_MIN, min(C8_E_MAX, e));
}

__device__ __forceinline__ float c8_pow2(int e) { return __uint_as_float((unsigned)(e + 127) << 23); }   // |e| < 127

// the exponent of a stored scale; whatever lies there, a number within the limits
__device__ __forceinline__ int c8_scale_exponent(float scale) {
    const int e = (int)((__float_as_uint(scale) >> 23) & 0xffu) - 127;
    return max(C8_E_MIN, min(C8_E_MAX, e));
}

// two values already divided by the scale -> two codes in the low 16 bits, rounded to nearest even and kept within the
// type's largest number.  The values are finite (what is not a number was replaced by zero before).
template <bool E4M3>
__device__ __forceinline__ unsigned c8_encode2(float a, float b) {
    if constexpr (E4M3) {
        return __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
    } else {
        const int x = __float2int_rn(fminf(fmaxf(a, -127.0f), 127.0f)), y = __float2int_rn(fminf(fmaxf(b, -127.0f), 127.0f));
        return (unsigned)(x & 0xff) | ((unsigned)(y & 0xff) << 8);
    }
}

// two codes (the low 16 bits) -> half2, exactly
template <bool E4M3>
__device__ __forceinline__ __half2 c8_decode2(unsigned codes) {
    if constexpr (E4M3) {
        return __half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)codes, __NV_E4M3));
    } else {
        // 0x6400 | u is 1024 + u in half precision; u = code + 128
        const unsigned w = __byte_perm(codes ^ 0x8080u, 0x64646464u, 0x4140);
        return __hsub2(*reinterpret_cast<const __half2*>(&w), __float2half2_rn(1152.0f));
    }
}

// four codes -> two half2 (elements 0, 1 and 2, 3), exactly
template <bool E4M3>
__device__ __forceinline__ void c8_decode4(unsigned codes, unsigned& lo, unsigned& hi) {
    if constexpr (E4M3) {
        const __half2 a = c8_decode2<true>(codes & 0xffffu), b = c8_decode2<true>(codes >> 16);
        lo = *reinterpret_cast<const unsigned*>(&a); hi = *reinterpret_cast<const unsigned*>(&b);
    } else {
        const unsigned u = codes ^ 0x80808080u;
        const unsigned a = __byte_perm(u, 0x64646464u, 0x4140), b = __byte_perm(u, 0x64646464u, 0x4342);
        const __half2 bias = __float2half2_rn(1152.0f);
        const __half2 x = __hsub2(*reinterpret_cast<const __half2*>(&a), bias), y = __hsub2(*reinterpret_cast<const __half2*>(&b), bias);
        lo = *reinterpret_cast<const unsigned*>(&x); hi = *reinterpret_cast<const unsigned*>(&y);
    }
}
