// zkv_fp8.cu -- rows in 8 bits: e4m3 elements with an fp32 scale for each
// block of 128, from 16-bit rows (zkv_quant_fp8) or from the RMSNorm of a
// residual sum (zkv_rmsnorm_fp8).  The reference has no 8-bit layer; its
// RMSNorm is flashinfer's (model_hub/qwen.py:429-612).
#include <algorithm>

#include "zkv_fp8.cuh"

namespace zkv {
namespace fp8 {

struct RowArgs {
    const uint16_t* x;
    int64_t x_ld;
    const uint16_t* residual;  // NULL: the norm is x's own
    int64_t residual_ld;
    uint16_t* sum;  // x + residual as it is kept
    int64_t sum_ld;
    const uint16_t* w;
    uint8_t* out;
    int64_t out_ld;
    float* scale;
    int64_t scale_token, scale_block;
    int64_t tokens;
    int dim;
    float eps;
};

template <bool kBf16>
__device__ __forceinline__ void to_floats(uint32_t w, float& lo, float& hi) {
    if (kBf16) {
        lo = __uint_as_float(w << 16);
        hi = __uint_as_float(w & 0xffff0000u);
    } else {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
        lo = f.x;
        hi = f.y;
    }
}

template <bool kBf16>
__device__ __forceinline__ uint32_t from_floats(float lo, float hi) {
    if (kBf16) return pack_bf162(lo, hi);
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}

template <bool kBf16>
__device__ __forceinline__ void load16(const uint16_t* p, float (&v)[16]) {
    const uint4 a = reinterpret_cast<const uint4*>(p)[0], b = reinterpret_cast<const uint4*>(p)[1];
    const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
    for (int i = 0; i < 8; ++i) to_floats<kBf16>(w[i], v[2 * i], v[2 * i + 1]);
}

// 16 elements of a thread, m the largest magnitude of them; the 8 threads of a block of 128 find its scale.
__device__ __forceinline__ void store_block(float (&y)[16], uint32_t m, const RowArgs& a, int64_t row, int at, bool in) {
#pragma unroll
    for (int off = 4; off >= 1; off >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, off));
    if (!in) return;
    const float s = scale_of(m);
    const Quotient by(s);
    by.prepare(y);
    uint4 q;
    q.x = by.e4m3(y[0], y[1], y[2], y[3]);
    q.y = by.e4m3(y[4], y[5], y[6], y[7]);
    q.z = by.e4m3(y[8], y[9], y[10], y[11]);
    q.w = by.e4m3(y[12], y[13], y[14], y[15]);
    *reinterpret_cast<uint4*>(a.out + row * a.out_ld + at) = q;
    if (at % kBlock == 0) a.scale[row * a.scale_token + (at / kBlock) * a.scale_block] = s;
}

// Eight threads a block, 16 elements each: a warp reads 1 KB in a row, and one
// 16-byte store a thread writes.  16383 x 4096 bf16: 40 us, 5.1 TB/s (0.78 of
// the copy rate): the issue slots are what it runs out of, with ten
// instructions an element.  Sixteen threads a block of 8 elements, two blocks
// each: 50 us against 37 in the same state with the quotients left out.
constexpr int kQuantThreads = 256;
template <bool kBf16>
__global__ void __launch_bounds__(kQuantThreads) quant_kernel(RowArgs a, int blocks) {
    const int64_t item = (blockIdx.x * (int64_t)kQuantThreads + threadIdx.x) >> 3;
    const int64_t row = item / blocks;
    const int at = (int)(item - row * blocks) * kBlock + (threadIdx.x & 7) * 16;
    const bool in = row < a.tokens && at < a.dim;
    grid_dep_wait();
    grid_dep_launch_next();
    float y[16] = {};
    uint32_t m = 0;
    if (in) {
        const uint4* x = reinterpret_cast<const uint4*>(a.x + row * a.x_ld + at);
        const uint4 p = x[0], q = x[1];
        const uint32_t w[8] = {p.x, p.y, p.z, p.w, q.x, q.y, q.z, q.w};
        // 16-bit magnitudes are ordered as the numbers are, infinities and NaN above: two in one comparison
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            m = __vmaxu2(m, w[i] & 0x7fff7fffu);
            to_floats<kBf16>(w[i], y[2 * i], y[2 * i + 1]);
        }
        float lo, hi;
        to_floats<kBf16>(m, lo, hi);
        m = max(magnitude(lo), magnitude(hi));
    }
    store_block(y, m, a, row, at, in);
}

// kRow threads a row (a power of two, whole warps), kTurns x 16 elements of
// it each, which stay in registers between the sum of squares and the output:
// one pass over the data.  fp32 inside; the sum with the residual is rounded
// to its type first, as it is kept, and the norm is that of the kept sum.
// 16384 x 4096 bf16 with a residual: 79 us, 5.9 TB/s (0.91 of the copy rate;
// 77 with the quotients' remainders left out); 32 x 4096: 2.2 us, the chain of
// a row's loads, its sum and its blocks.
template <bool kBf16, int kRow, int kTurns>
__global__ void __launch_bounds__(kRow < 128 ? 128 : kRow) norm_kernel(RowArgs a) {
    constexpr int kThreads = kRow < 128 ? 128 : kRow;
    constexpr int kWarps = kRow / 32;
    const int64_t row = blockIdx.x * (int64_t)(kThreads / kRow) + threadIdx.x / kRow;
    const int t = threadIdx.x % kRow;
    const bool live = row < a.tokens;
    float x[kTurns][16] = {};
    float ss = 0.f;
    grid_dep_wait();
    grid_dep_launch_next();
#pragma unroll
    for (int j = 0; j < kTurns; ++j) {
        const int at = (j * kRow + t) * 16;
        if (!live || at >= a.dim) continue;
        load16<kBf16>(a.x + row * a.x_ld + at, x[j]);
        if (a.residual) {
            float r[16];
            load16<kBf16>(a.residual + row * a.residual_ld + at, r);
            uint32_t w[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                w[i] = from_floats<kBf16>(x[j][2 * i] + r[2 * i], x[j][2 * i + 1] + r[2 * i + 1]);
                to_floats<kBf16>(w[i], x[j][2 * i], x[j][2 * i + 1]);
            }
            uint4* to = reinterpret_cast<uint4*>(a.sum + row * a.sum_ld + at);
            to[0] = make_uint4(w[0], w[1], w[2], w[3]);
            to[1] = make_uint4(w[4], w[5], w[6], w[7]);
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) ss += x[j][i] * x[j][i];
    }
#pragma unroll
    for (int off = 16; off >= 1; off >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, off);
    if (kWarps > 1) {
        __shared__ float red[kThreads / 32];
        if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = ss;
        __syncthreads();
        ss = 0.f;
        const int first = (threadIdx.x / kRow) * kWarps;
#pragma unroll
        for (int i = 0; i < kWarps; ++i) ss += red[first + i];
    }
    const float inv = rsqrtf(ss / (float)a.dim + a.eps);
#pragma unroll
    for (int j = 0; j < kTurns; ++j) {
        const int at = (j * kRow + t) * 16;
        const bool in = live && at < a.dim;
        if (in) {
            float w[16];
            load16<kBf16>(a.w + at, w);
#pragma unroll
            for (int i = 0; i < 16; ++i) x[j][i] = x[j][i] * inv * w[i];
        }
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < 16; ++i) m = max(m, magnitude(x[j][i]));
        store_block(x[j], m, a, row, at, in);
    }
}

template <bool kBf16, int kRow, int kTurns>
static int launch_norm(const RowArgs& a, cudaStream_t stream) {
    constexpr int kThreads = kRow < 128 ? 128 : kRow, kRows = kThreads / kRow;
    return launch_pdl_kernel(norm_kernel<kBf16, kRow, kTurns>, dim3((unsigned)((a.tokens + kRows - 1) / kRows)),
                             dim3(kThreads), 0, stream, a);
}

template <bool kBf16>
static int norm_of(const RowArgs& a, cudaStream_t stream) {
    if (a.dim <= 512) return launch_norm<kBf16, 32, 1>(a, stream);
    if (a.dim <= 1024) return launch_norm<kBf16, 64, 1>(a, stream);
    if (a.dim <= 2048) return launch_norm<kBf16, 128, 1>(a, stream);
    if (a.dim <= 4096) return launch_norm<kBf16, 256, 1>(a, stream);
    if (a.dim <= 8192) return launch_norm<kBf16, 512, 1>(a, stream);
    if (a.dim <= 16384) return launch_norm<kBf16, 512, 2>(a, stream);
    return launch_norm<kBf16, 512, 4>(a, stream);
}

static int check_rows(const RowArgs& a, int dtype) {
    if (!a.x || !a.out || !a.scale || a.tokens < 0 || a.dim < 1) return ZKV_ERR_ARG;
    if (dtype != ZKV_DT_BF16 && dtype != ZKV_DT_F16) return ZKV_ERR_ARG;
    if (a.scale_token < 1 || a.scale_block < 1 || a.x_ld < a.dim || a.out_ld < a.dim) return ZKV_ERR_ARG;
    if (a.dim % 16) return ZKV_ERR_UNSUPPORTED;
    if (!aligned16(a.x) || !aligned16(a.out) || a.x_ld % 8 || a.out_ld % 16) return ZKV_ERR_ALIGN;
    if (a.tokens > INT32_MAX) return ZKV_ERR_CAPACITY;
    return ZKV_OK;
}

}  // namespace fp8
}  // namespace zkv

using namespace zkv;

extern "C" int zkv_quant_fp8(const void* x, int64_t x_ld, int dtype, int64_t tokens, int dim, void* out, int64_t out_ld,
                             float* scale, int64_t scale_token, int64_t scale_block, void* stream) {
    fp8::RowArgs a = {};
    a.x = (const uint16_t*)x, a.x_ld = x_ld, a.out = (uint8_t*)out, a.out_ld = out_ld;
    a.scale = scale, a.scale_token = scale_token, a.scale_block = scale_block, a.tokens = tokens, a.dim = dim;
    if (const int rc = fp8::check_rows(a, dtype)) return rc;
    const int blocks = fp8::blocks_of(dim);
    const int64_t ctas = (tokens * blocks * 8 + fp8::kQuantThreads - 1) / fp8::kQuantThreads;
    if (ctas > INT32_MAX) return ZKV_ERR_CAPACITY;
    if (tokens == 0) return ZKV_OK;
    return launch_pdl_kernel(dtype == ZKV_DT_BF16 ? fp8::quant_kernel<true> : fp8::quant_kernel<false>, dim3((unsigned)ctas),
                             dim3(fp8::kQuantThreads), 0, (cudaStream_t)stream, a, blocks);
}

extern "C" int zkv_rmsnorm_fp8(const void* x, int64_t x_ld, const void* residual, int64_t residual_ld, void* residual_out,
                               int64_t residual_out_ld, const void* w, int dtype, int64_t tokens, int dim, float eps,
                               void* out, int64_t out_ld, float* scale, int64_t scale_token, int64_t scale_block,
                               void* stream) {
    fp8::RowArgs a = {};
    a.x = (const uint16_t*)x, a.x_ld = x_ld, a.out = (uint8_t*)out, a.out_ld = out_ld;
    a.residual = (const uint16_t*)residual, a.residual_ld = residual_ld;
    a.sum = (uint16_t*)residual_out, a.sum_ld = residual_out_ld;
    a.w = (const uint16_t*)w, a.eps = eps;
    a.scale = scale, a.scale_token = scale_token, a.scale_block = scale_block, a.tokens = tokens, a.dim = dim;
    if (!w || !(eps >= 0.f) || !residual != !residual_out) return ZKV_ERR_ARG;
    if (residual && (residual_ld < dim || residual_out_ld < dim)) return ZKV_ERR_ARG;
    if (const int rc = fp8::check_rows(a, dtype)) return rc;
    if (!fp8::aligned16(w)) return ZKV_ERR_ALIGN;
    if (residual && (!fp8::aligned16(residual) || !fp8::aligned16(residual_out) || residual_ld % 8 || residual_out_ld % 8))
        return ZKV_ERR_ALIGN;
    if (dim > 32768) return ZKV_ERR_CAPACITY;
    if (tokens == 0) return ZKV_OK;
    return dtype == ZKV_DT_BF16 ? fp8::norm_of<true>(a, (cudaStream_t)stream) : fp8::norm_of<false>(a, (cudaStream_t)stream);
}
