// The paged cache in 8 bits, as its kernels share it.
//
// A layer's keys (and values) are e4m3 numbers [page][kv head][slot][dim] and a float32 scale per (page, kv head): the
// number that a byte stands for is e4m3 * scale.  A scale is a power of two 2^e, -48 <= e <= 48.  So a row that is stored
// again under a larger scale loses nothing above e4m3's subnormals, scores take a page's scale in one exact
// multiplication, and the attention kernels may carry a value page's scale as an integer in the exponent of a weight.
// The range leaves float32 room for what is multiplied with it: weights times 2^(-e) stay finite and, between any two
// pages, above 2^-126 unless they differ by 2^30 besides.
//
// Every e4m3 number is a float16 number (and e4m3 x e4m3-scaled sums are not needed): the attention kernels hand keys and
// values to the tensor cores as float16, exactly, with one conversion per two numbers, and float32 accumulators.
//
// A key row that holds NaN marks a token whose key or value was not finite when it was stored; its values are stored as
// zeros.  Value rows therefore never hold NaN, and a weight of 0 removes a masked token whatever it held.
#pragma once
#include "common.cuh"

#include <cuda_fp16.h>

namespace {

constexpr int Q8_E_MIN = -48, Q8_E_MAX = 48;

// 2^e for the exponents that scales have (and sums of a few)
__device__ __forceinline__ float q8_pow2(int e) { return __int_as_float((e + 127) << 23); }
// the exponent of a scale as stored; powers of two only
__device__ __forceinline__ int q8_exponent(float scale) { return ((__float_as_int(scale) >> 23) & 0xff) - 127; }

// the smallest e in [-48, 48] with m <= 448 * 2^e, from the bits of m >= 0: 448 = 1.75 * 2^8, so a mantissa above
// 1.75 (0x600000) carries into the exponent
__device__ __forceinline__ int q8_exponent_for(int bits) {
    if (bits == 0) return Q8_E_MIN;
    const int e = ((bits + 0x1fffff) >> 23) - 127 - 8;
    return min(max(e, Q8_E_MIN), Q8_E_MAX);
}

// two e4m3 numbers (the low byte first) as two float16
__device__ __forceinline__ uint32_t q8_to_f16x2(uint32_t two) {
    uint32_t r;
    asm("{\n.reg .b16 l;\ncvt.u16.u32 l, %1;\ncvt.rn.f16x2.e4m3x2 %0, l;\n}\n" : "=r"(r) : "r"(two));
    return r;
}
// four e4m3 numbers as two pairs of float16
__device__ __forceinline__ void q8_to_f16x4(uint32_t four, uint32_t& lo, uint32_t& hi) {
    asm("{\n.reg .b16 l, h;\nmov.b32 {l, h}, %2;\ncvt.rn.f16x2.e4m3x2 %0, l;\ncvt.rn.f16x2.e4m3x2 %1, h;\n}\n"
        : "=r"(lo), "=r"(hi) : "r"(four));
}
// the nearest e4m3 numbers, ties to even; beyond +-448 they stay at it, NaN is NaN
__device__ __forceinline__ uint32_t q8_pack2(float lo, float hi) {
    unsigned short r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;\n" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}

__device__ __forceinline__ uint32_t q8_half2(float lo, float hi) {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}

}  // namespace
