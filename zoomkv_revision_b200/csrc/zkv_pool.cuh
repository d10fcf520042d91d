// zkv_pool.cuh -- what the pooled-cache kernels share: host checks of a
// zkv_pool and the status word.
#pragma once

#include "zkv_common.cuh"

namespace zkv {
namespace pool {

// The status word keeps the largest code, so that two failures in one call
// give the same word in any order.
__device__ __forceinline__ void raise_status(int32_t* status, int code) {
    if (status) atomicMax(status, code);
}

// Exclusive sum over the block's threads (blockDim.x a multiple of 32); *total gets the sum.
static __device__ __forceinline__ int64_t block_sum_before(int64_t x, int64_t* sh, int64_t* total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
    int64_t incl = x;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
        const int64_t y = __shfl_up_sync(0xffffffffu, incl, off);
        if (lane >= off) incl += y;
    }
    __syncthreads();  // the previous use of sh
    if (lane == 31) sh[warp] = incl;
    __syncthreads();
    int64_t w = lane < nw ? sh[lane] : 0;
    int64_t wi = w;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
        const int64_t y = __shfl_up_sync(0xffffffffu, wi, off);
        if (lane >= off) wi += y;
    }
    *total = __shfl_sync(0xffffffffu, wi, 31);
    return incl - x + __shfl_sync(0xffffffffu, wi - w, warp);
}

static inline int log2_of(int x) {
    int s = 0;
    while ((1 << s) < x) ++s;
    return s;
}

static inline bool block_size_ok(int s) { return s >= 16 && s <= 1024 && (s & (s - 1)) == 0; }

static inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

static inline int element_bytes(int dtype) { return dtype == ZKV_DT_F8E4M3 ? 1 : 2; }

// The fields that a caller fills; `maps` is zkv_pool_init's.
static inline int check_pool(const zkv_pool* p) {
    if (!p || !p->k || !p->v || p->n_blocks < 1 || p->kv_heads < 1) return ZKV_ERR_ARG;
    if (p->dtype != ZKV_DT_BF16 && p->dtype != ZKV_DT_F16 && p->dtype != ZKV_DT_F8E4M3) return ZKV_ERR_ARG;
    if ((p->k_scale || p->v_scale) && p->dtype != ZKV_DT_F8E4M3) return ZKV_ERR_ARG;
    if (p->head_dim != 64 && p->head_dim != 128 && p->head_dim != 256) return ZKV_ERR_UNSUPPORTED;
    if (!block_size_ok(p->block_size)) return ZKV_ERR_UNSUPPORTED;
    if (p->n_blocks > INT32_MAX) return ZKV_ERR_CAPACITY;
    if (!aligned16(p->k) || !aligned16(p->v)) return ZKV_ERR_ALIGN;
    const int64_t strides[6] = {p->k_block, p->k_token, p->k_head, p->v_block, p->v_token, p->v_head};
    const int per16 = 16 / element_bytes(p->dtype);
    for (int64_t s : strides) {
        if (s < 1) return ZKV_ERR_ARG;
        if (s % per16) return ZKV_ERR_ALIGN;
    }
    return ZKV_OK;
}

}  // namespace pool
}  // namespace zkv
