// zkv_fp8.cuh -- what the 8-bit kernels share: e4m3 with an fp32 scale for
// each block of 128 elements.
#pragma once

#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "zkv_common.cuh"

namespace zkv {
namespace fp8 {

constexpr int kBlock = 128;      // elements of a row that share a scale
constexpr float kMax = 448.f;    // largest e4m3 value

static inline int blocks_of(int64_t n) { return (int)((n + kBlock - 1) / kBlock); }
static inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// The scale of a block from the bits of its largest magnitude.  Magnitudes
// are compared as integers, so that a NaN counts as larger than an infinity
// and neither is lost: the block then reads back as NaN.
__device__ __forceinline__ uint32_t magnitude(float x) { return __float_as_uint(x) & 0x7fffffffu; }
__device__ __forceinline__ float scale_of(uint32_t largest) { return __fdiv_rn(__uint_as_float(largest), kMax); }

__device__ __forceinline__ uint32_t e4m3x4(float a, float b, float c, float d) {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
    return lo | (hi << 16);
}

// e4m3 of the fp32 quotient by a block's scale, two roundings as defined, and
// nearly always without a division: x times the reciprocal shrunk and grown
// by 2^-21 encloses the quotient and its rounding (the products are off by
// 3 * 2^-24 at most), rounding is monotone, so where both ends give one code
// the quotient has it; else (that close to the middle of two codes) the
// elements are divided.  A scale of 0 stores zeros.
struct Quotient {
    float scale, low, high;
    bool divide;  // the reciprocal is not an ordinary number

    __device__ __forceinline__ explicit Quotient(float s) {
        const float r = __fdiv_rn(1.f, s);
        scale = s;
        low = r * (1.f - 4.76837158203125e-7f);
        high = r * (1.f + 4.76837158203125e-7f);
        divide = !(s > 1e-30f && s < 1e30f);
    }
    __device__ __forceinline__ uint32_t e4m3(float a, float b, float c, float d) const {
        const uint32_t x = e4m3x4(a * low, b * low, c * low, d * low);
        const uint32_t y = e4m3x4(a * high, b * high, c * high, d * high);
        if (x == y && !divide) return x;
        if (scale == 0.f) return 0u;
        return e4m3x4(__fdiv_rn(a, scale), __fdiv_rn(b, scale), __fdiv_rn(c, scale), __fdiv_rn(d, scale));
    }
};

}  // namespace fp8
}  // namespace zkv
