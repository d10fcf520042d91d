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

// e4m3 of the fp32 quotient by a block's scale, two roundings as defined,
// without a division an element: from the correctly rounded reciprocal r, the
// product q = x r and the remainder x - q s, which is exact in one fused
// operation, q + r (x - q s) is the rounded quotient (P. Markstein,
// "Computation of elementary functions on the IBM RISC System/6000
// processor", IBM J. Res. Dev. 34, 1990).  The division took 16383 x 4096
// elements 53 us, and 50 to 69 where it decided only what two enclosing
// products left open: an element in 16 of every seventh block of bf16 numbers
// is the exact middle of two codes.  A scale of 0 stores zeros.
struct Quotient {
    float lift, scale, r;  // lift: a power of two that keeps a remainder within fp32's range

    __device__ __forceinline__ explicit Quotient(float s) {
        lift = s < 1e-20f ? 18446744073709551616.f : s > 1e20f ? 5.421010862427522e-20f : 1.f;
        scale = s * lift;
        r = scale == 0.f ? 0.f : __fdiv_rn(1.f, scale);
    }
    __device__ __forceinline__ float of(float x) const {
        x *= lift;
        const float q = x * r;
        return copysignf(fmaf(fmaf(-q, scale, x), r, q), x);  // (the remainder of -0 is +0)
    }
    __device__ __forceinline__ uint32_t e4m3(float a, float b, float c, float d) const {
        return e4m3x4(of(a), of(b), of(c), of(d));
    }
};

}  // namespace fp8
}  // namespace zkv
