// The 8-bit KV cache. A row - one token of one kv head - is D numbers of type e4m3 and one scale 2^e, e in [-14, 7], so that
// value = code * 2^e. e is the smallest one with min(max |x|, 57344) <= 448 * 2^e.
//
// Why powers of two: a code has 4 significant bits, and scaling by 2^e adds none. Every value is then a number of fp16 (from
// 2^-23 up to 448 * 2^7 = 57344) and of bf16, to the bit: what reads the cache may apply the scale in 16 bits and feed the
// tensor cores without a further rounding. A scale of more bits would not make the codes better, e4m3 being a floating type.
// Where the scale is kept in check: rows whose largest number is below 448 * 2^-14 = 0.027 share the scale 2^-14 (steps of
// 2^-23), numbers beyond +-57344 (bf16 and fp32 rows) are stored as +-57344.
//
// Memory: codes [num_blocks][block_size][kv_heads][D]; scales one byte e + 15 (the exponent field of the fp16 number 2^e),
// [num_blocks][kv_heads][block_size rounded up to 16], so that the scales of a head's page are one aligned piece.
#pragma once

#include "common.cuh"

namespace sca_b200 {
namespace fp8 {

constexpr int kMinExponent = -14, kMaxExponent = 7;
constexpr float kLargest = 57344.0f;  // 448 * 2^7

__host__ __device__ constexpr int64_t ScaleRow(int64_t block_size) { return (block_size + 15) / 16 * 16; }

// The exponent for a row whose largest number is `amax` (not NaN, at most kLargest). 448 = 1.75 * 2^8: with amax = f * 2^k it is
// k - 8, and one more where f exceeds 1.75, which the addition carries into the exponent field.
__device__ __forceinline__ int ExponentFor(float amax) {
    const int e = static_cast<int>((__float_as_uint(amax) + 0x1fffffu) >> 23) - 127 - 8;
    return max(kMinExponent, min(kMaxExponent, e));
}
__device__ __forceinline__ float PowerOfTwo(int e) { return __uint_as_float(static_cast<uint32_t>(e + 127) << 23); }
// The scale a byte stands for; two of them as a pair of fp16 numbers.
__device__ __forceinline__ float ScaleOf(uint32_t byte) { return __uint_as_float((byte + 112u) << 23); }
__device__ __forceinline__ uint32_t ScalePair(uint32_t byte0, uint32_t byte1) { return ((byte0 & 31u) << 10) | ((byte1 & 31u) << 26); }

// Two numbers into codes (lo in the low byte): to nearest, ties to even, at most 448 in size; NaN stays NaN.
__device__ __forceinline__ uint32_t Encode2(float lo, float hi) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}
// The codes in the low / high half of a word as a pair of fp16 numbers; exact.
__device__ __forceinline__ uint32_t DecodeLow(uint32_t word) {
    uint32_t r;
    asm("{\n.reg .b16 l, h;\nmov.b32 {l, h}, %1;\ncvt.rn.f16x2.e4m3x2 %0, l;\n}\n" : "=r"(r) : "r"(word));
    return r;
}
__device__ __forceinline__ uint32_t DecodeHigh(uint32_t word) {
    uint32_t r;
    asm("{\n.reg .b16 l, h;\nmov.b32 {l, h}, %1;\ncvt.rn.f16x2.e4m3x2 %0, h;\n}\n" : "=r"(r) : "r"(word));
    return r;
}
__device__ __forceinline__ uint32_t MulHalf2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
__device__ __forceinline__ float2 UnpackHalf2(uint32_t v) {
    const __half2 h = *reinterpret_cast<const __half2*>(&v);
    return __half22float2(h);
}

}  // namespace fp8
}  // namespace sca_b200
