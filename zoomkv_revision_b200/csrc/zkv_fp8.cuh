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
// is the exact middle of two codes; 40.5 so.  A scale of 0 stores zeros.
struct Quotient {
    float lift, scale, r;  // lift: a power of two that keeps a remainder within fp32's range

    __device__ __forceinline__ explicit Quotient(float s) {
        lift = s < 1e-20f ? 18446744073709551616.f : s > 1e20f ? 5.421010862427522e-20f : 1.f;
        scale = s * lift;
        r = scale == 0.f ? 0.f : __fdiv_rn(1.f, scale);
    }
    // To be called once on what e4m3 is given.
    template <int N>
    __device__ __forceinline__ void prepare(float (&x)[N]) const {
        if (lift != 1.f)
#pragma unroll
            for (int i = 0; i < N; ++i) x[i] *= lift;
    }
    // Two quotients at once: packed products and sums (16383 x 4096 elements 43.8 -> 40.5 us).  The remainder of -0 is +0, so
    // the sign is the element's own.
    __device__ __forceinline__ void of(float& a, float& b) const {
        asm("{\n\t"
            ".reg .b64 x, y, s, q, t;\n\t"
            ".reg .b32 u, v;\n\t"
            "mov.b64 x, {%0, %1};\n\t"
            "mov.b64 y, {%2, %2};\n\t"
            "mov.b64 s, {%3, %3};\n\t"
            "mul.rn.f32x2 q, x, y;\n\t"
            "fma.rn.f32x2 t, q, s, x;\n\t"
            "fma.rn.f32x2 t, t, y, q;\n\t"
            "mov.b64 {u, v}, t;\n\t"
            "copysign.f32 %0, %0, u;\n\t"
            "copysign.f32 %1, %1, v;\n\t}"
            : "+f"(a), "+f"(b)
            : "f"(r), "f"(-scale));
    }
    __device__ __forceinline__ uint32_t e4m3(float a, float b, float c, float d) const {
        of(a, b);
        of(c, d);
        return e4m3x4(a, b, c, d);
    }
};

}  // namespace fp8
}  // namespace zkv
