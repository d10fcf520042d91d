// zkv_pool_decode.cu -- attention of one new token per request over a pooled
// KV cache.
//
//   o = sum_t p_t v_t / sum_t p_t,  p_t = exp(cap(scale q . k_t) - max)
//
// First form: one CTA per (request, kv head, 8 query heads) and 512 tokens;
// each warp runs the softmax over every fourth token with the row's dims over
// its lanes, the warps' and then the splits' partials (m, l, o) are joined.
#include <cuda.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <algorithm>
#include <cstring>

#include "zkv_pool.cuh"

namespace zkv {
namespace pool {

constexpr int kHeads = 8;      // query heads of a row
constexpr int kSplit = 512;    // tokens of a CTA
constexpr int kDecodeWarps = 4;

struct DecodeArgs {
    const uint8_t* q;
    const uint8_t* k;
    const uint8_t* v;
    const float* k_scale;
    const float* v_scale;
    const int32_t* lens;
    const int32_t* table;
    void* out;
    float* lse;
    int32_t* status;
    float* parts;  // [rows][splits][kHeads][D + 2]
    int64_t q_row, q_head, k_block, k_token, k_head, v_block, v_token, v_head;  // bytes
    int64_t table_ld, n_blocks;
    int64_t cap;  // longest length
    int kv_heads, G, chunks, splits, shift, window;
    float scale, softcap;
};

template <int kType>
__device__ __forceinline__ float load_el(const uint8_t* p, int i) {
    if constexpr (kType == ZKV_DT_BF16) return bfbits2f(reinterpret_cast<const uint16_t*>(p)[i]);
    else if constexpr (kType == ZKV_DT_F16) return __half2float(reinterpret_cast<const __half*>(p)[i]);
    else return __half2float(__half(__nv_cvt_fp8_to_halfraw(p[i], __NV_E4M3)));
}

template <int kType>
__device__ __forceinline__ void store_el(void* p, int64_t i, float x) {
    if constexpr (kType == ZKV_DT_BF16) reinterpret_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(x);
    else reinterpret_cast<__half*>(p)[i] = __float2half_rn(x);
}

__device__ __forceinline__ int request_len(const DecodeArgs& a, int b, bool report) {
    const int n = a.lens[b];
    if (n >= 0 && n <= a.cap) return n;
    if (report) raise_status(a.status, ZKV_ERR_RANGE);
    return n < 0 ? 0 : (int)a.cap;
}

template <int kQ, int kPool, int D>
__global__ void __launch_bounds__(kDecodeWarps * 32) pool_decode_kernel(const __grid_constant__ DecodeArgs a) {
    constexpr int E = D / 32;
    __shared__ float s_o[kDecodeWarps][kHeads][D];
    __shared__ float s_ml[kDecodeWarps][kHeads][2];
    const int row = blockIdx.x, split = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int c = row % a.chunks, h = row / a.chunks % a.kv_heads, b = row / (a.chunks * a.kv_heads);
    const int len = request_len(a, b, split == 0 && threadIdx.x == 0);
    const int lo = a.window > 0 && len > a.window ? len - a.window : 0;
    const int t0 = max(lo, split * kSplit), t1 = min((int64_t)len, (int64_t)(split + 1) * kSplit);
    float* part = a.parts + ((int64_t)row * a.splits + split) * kHeads * (D + 2);
    const int n_heads = min(kHeads, a.G - c * kHeads);
    float q[kHeads][E], o[kHeads][E], m[kHeads], l[kHeads];
    for (int g = 0; g < kHeads; ++g) {
        m[g] = -INFINITY;
        l[g] = 0.f;
        for (int e = 0; e < E; ++e) {
            o[g][e] = 0.f;
            q[g][e] = g < n_heads ? load_el<kQ>(a.q + b * a.q_row + (int64_t)(h * a.G + c * kHeads + g) * a.q_head,
                                                lane + 32 * e)
                                  : 0.f;
        }
    }
    const float ks = a.k_scale ? a.k_scale[h] : 1.f, vs = a.v_scale ? a.v_scale[h] : 1.f;
    for (int t = t0 + warp; t < t1; t += kDecodeWarps) {
        const int id = a.table[b * a.table_ld + (t >> a.shift)];
        if (id < 0 || id >= a.n_blocks) {
            if (lane == 0) raise_status(a.status, ZKV_ERR_RANGE);
            continue;
        }
        const int at = t & ((1 << a.shift) - 1);
        const uint8_t* kp = a.k + id * a.k_block + at * a.k_token + h * a.k_head;
        const uint8_t* vp = a.v + id * a.v_block + at * a.v_token + h * a.v_head;
        float k[E], v[E];
        for (int e = 0; e < E; ++e) {
            k[e] = load_el<kPool>(kp, lane + 32 * e);
            v[e] = load_el<kPool>(vp, lane + 32 * e);
        }
        for (int g = 0; g < kHeads; ++g) {
            float x = 0.f;
            for (int e = 0; e < E; ++e) x += q[g][e] * k[e];
            for (int off = 16; off >= 1; off >>= 1) x += __shfl_xor_sync(0xffffffffu, x, off);
            x *= a.scale * ks;
            if (a.softcap > 0.f) x = a.softcap * tanhf(x / a.softcap);
            if (x == -INFINITY) continue;
            const float mn = fmaxf(m[g], x), f = m[g] == -INFINITY ? 0.f : expf(m[g] - mn), p = expf(x - mn);
            l[g] = l[g] * f + p;
            m[g] = mn;
            for (int e = 0; e < E; ++e) o[g][e] = o[g][e] * f + p * v[e];
        }
    }
    for (int g = 0; g < kHeads; ++g) {
        for (int e = 0; e < E; ++e) s_o[warp][g][lane + 32 * e] = o[g][e] * vs;
        if (lane == 0) {
            s_ml[warp][g][0] = m[g];
            s_ml[warp][g][1] = l[g];
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < kHeads * D; i += blockDim.x) {
        const int g = i / D, d = i % D;
        float mm = -INFINITY, ll = 0.f, oo = 0.f;
        for (int w = 0; w < kDecodeWarps; ++w) mm = fmaxf(mm, s_ml[w][g][0]);
        for (int w = 0; w < kDecodeWarps; ++w) {
            const float f = s_ml[w][g][0] == -INFINITY ? 0.f : expf(s_ml[w][g][0] - mm);
            ll += f * s_ml[w][g][1];
            oo += f == 0.f ? 0.f : f * s_o[w][g][d];
        }
        part[g * (D + 2) + d] = oo;
        if (d == 0) {
            part[g * (D + 2) + D] = mm;
            part[g * (D + 2) + D + 1] = ll;
        }
    }
}

template <int kQ, int D>
__global__ void pool_join_kernel(const __grid_constant__ DecodeArgs a) {
    const int row = blockIdx.x, g = blockIdx.y, d = threadIdx.x;
    const int c = row % a.chunks, h = row / a.chunks % a.kv_heads, b = row / (a.chunks * a.kv_heads);
    if (g >= a.G - c * kHeads) return;
    const float* part = a.parts + (int64_t)row * a.splits * kHeads * (D + 2) + g * (D + 2);
    float m = -INFINITY, l = 0.f, o = 0.f;
    for (int s = 0; s < a.splits; ++s) m = fmaxf(m, part[(int64_t)s * kHeads * (D + 2) + D]);
    for (int s = 0; s < a.splits; ++s) {
        const float* p = part + (int64_t)s * kHeads * (D + 2);
        const float f = p[D] == -INFINITY ? 0.f : expf(p[D] - m);
        l += f * p[D + 1];
        if (f != 0.f) o += f * p[d];
    }
    const int64_t head = (int64_t)b * a.kv_heads * a.G + h * a.G + c * kHeads + g;
    store_el<kQ>(a.out, head * D + d, l > 0.f ? o / l : 0.f);
    if (a.lse && d == 0) a.lse[head] = m + logf(l);
}

static int decode_splits(int64_t max_len) { return (int)std::max<int64_t>(1, (max_len + kSplit - 1) / kSplit); }

template <int kQ, int kPool>
static void launch_decode(const DecodeArgs& a, int rows, int D, cudaStream_t st) {
    const dim3 g1(rows, a.splits), g2(rows, std::min(kHeads, a.G));
    switch (D) {
        case 64:
            pool_decode_kernel<kQ, kPool, 64><<<g1, kDecodeWarps * 32, 0, st>>>(a);
            pool_join_kernel<kQ, 64><<<g2, 64, 0, st>>>(a);
            break;
        case 128:
            pool_decode_kernel<kQ, kPool, 128><<<g1, kDecodeWarps * 32, 0, st>>>(a);
            pool_join_kernel<kQ, 128><<<g2, 128, 0, st>>>(a);
            break;
        default:
            pool_decode_kernel<kQ, kPool, 256><<<g1, kDecodeWarps * 32, 0, st>>>(a);
            pool_join_kernel<kQ, 256><<<g2, 256, 0, st>>>(a);
            break;
    }
}

}  // namespace pool
}  // namespace zkv

using namespace zkv;

extern "C" int zkv_pool_init(zkv_pool* p) {
    const int rc = pool::check_pool(p);
    if (rc == ZKV_OK) std::memset(p->maps, 0, sizeof(p->maps));
    return rc;
}

extern "C" size_t zkv_pool_decode_ws_bytes(int batch, int q_heads, int kv_heads, int head_dim, int64_t max_len) {
    if (batch < 0 || q_heads < 1 || kv_heads < 1 || q_heads % kv_heads || head_dim < 1 || max_len < 0) return 0;
    const int chunks = (q_heads / kv_heads + pool::kHeads - 1) / pool::kHeads;
    return (size_t)batch * kv_heads * chunks * pool::decode_splits(max_len) * pool::kHeads * (head_dim + 2) * 4 + 256;
}

extern "C" int zkv_pool_decode(const void* q, int64_t q_row, int64_t q_head, int dtype, const zkv_pool* p,
                               const int32_t* lens, const int32_t* block_table, int64_t table_ld, int width,
                               int batch, int q_heads, float scale, int window, float softcap, int64_t max_len,
                               void* out, float* lse, int32_t* status, void* workspace, size_t ws_bytes,
                               void* stream) {
    const int rc = pool::check_pool(p);
    if (rc != ZKV_OK) return rc;
    if (batch < 0 || width < 0 || table_ld < width || q_heads < 1 || q_heads % p->kv_heads || window < 0 ||
        max_len < 0 || !(softcap >= 0.f) || (dtype != ZKV_DT_BF16 && dtype != ZKV_DT_F16))
        return ZKV_ERR_ARG;
    if (p->dtype != ZKV_DT_F8E4M3 && p->dtype != dtype) return ZKV_ERR_ARG;
    if (batch == 0) return ZKV_OK;
    if (!q || !lens || !out || !workspace || (!block_table && width > 0)) return ZKV_ERR_ARG;
    if (!pool::aligned16(q) || q_row % 8 || q_head % 8 || !pool::aligned16(out)) return ZKV_ERR_ALIGN;
    if ((reinterpret_cast<uintptr_t>(workspace) & 255) != 0) return ZKV_ERR_ALIGN;
    const int64_t room = (int64_t)width * p->block_size;
    const int64_t cap = std::min<int64_t>(max_len > 0 ? std::min(max_len, room) : room, INT32_MAX);
    if (ws_bytes < zkv_pool_decode_ws_bytes(batch, q_heads, p->kv_heads, p->head_dim, cap)) return ZKV_ERR_CAPACITY;
    const int el = pool::element_bytes(p->dtype);
    pool::DecodeArgs a;
    a.q = (const uint8_t*)q, a.k = (const uint8_t*)p->k, a.v = (const uint8_t*)p->v;
    a.k_scale = p->k_scale, a.v_scale = p->v_scale;
    a.lens = lens, a.table = block_table, a.out = out, a.lse = lse, a.status = status;
    a.parts = (float*)workspace;
    a.q_row = q_row * 2, a.q_head = q_head * 2;
    a.k_block = p->k_block * el, a.k_token = p->k_token * el, a.k_head = p->k_head * el;
    a.v_block = p->v_block * el, a.v_token = p->v_token * el, a.v_head = p->v_head * el;
    a.table_ld = table_ld, a.n_blocks = p->n_blocks, a.cap = cap;
    a.kv_heads = p->kv_heads, a.G = q_heads / p->kv_heads, a.chunks = (a.G + pool::kHeads - 1) / pool::kHeads;
    a.splits = pool::decode_splits(cap), a.shift = pool::log2_of(p->block_size), a.window = window;
    a.scale = scale, a.softcap = softcap;
    if (a.splits > 65535) return ZKV_ERR_CAPACITY;
    const int rows = batch * p->kv_heads * a.chunks;
    cudaStream_t st = (cudaStream_t)stream;
    if (p->dtype == ZKV_DT_BF16) pool::launch_decode<ZKV_DT_BF16, ZKV_DT_BF16>(a, rows, p->head_dim, st);
    else if (p->dtype == ZKV_DT_F16) pool::launch_decode<ZKV_DT_F16, ZKV_DT_F16>(a, rows, p->head_dim, st);
    else if (dtype == ZKV_DT_BF16) pool::launch_decode<ZKV_DT_BF16, ZKV_DT_F8E4M3>(a, rows, p->head_dim, st);
    else pool::launch_decode<ZKV_DT_F16, ZKV_DT_F8E4M3>(a, rows, p->head_dim, st);
    return launch_status();
}
