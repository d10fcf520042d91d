// zkv_fp8_gemm.cu -- products of e4m3 rows with e4m3 weights, both with fp32
// scales for blocks of 128 (rows: 1 x 128, weights: 128 x 128), and the gated
// form whose output is e4m3 with block scales again:
//   y[m][n] = sum_b xs[m][b] ws[n / 128][b] sum_{k in block b} x[m][k] w[n][k]
//   a[m][f] = silu(g) u, g and u the two parts' products, stored as blocks
// The scales change with every block of the inner dimension, so each block's
// sum of 128 products (tcgen05, fp32 in tensor memory) is read back, scaled
// and added in fp32 registers.
//
// Features are the matrix rows of the tensor core's tile (128 lanes), tokens
// its columns: a step of few tokens fills the tile all the same, and the
// weights go from memory to the tensor core without passing a register.  What
// bounds such a call is reading the weights once; tiles that are fewer than
// the SMs are cut along the inner dimension over a cluster, whose CTAs add
// their parts through distributed shared memory in the order of their ranks.
#include <cuda.h>

#include <algorithm>
#include <cstring>
#include <mutex>

#include "zkv_fp8.cuh"
#include "zkv_tc.cuh"

namespace zkv {
namespace fp8 {

constexpr int kTile = 128;       // features of a tile
constexpr int kTileBytes = kTile * kBlock;
constexpr int kSmemSM = 228 * 1024, kSmemReserved = 1024;

struct Product {
    const float* x_scale;
    int64_t xs_token, xs_block;
    const float* w_scale;  // [parts * row_blocks][k_blocks]
    int64_t tokens;
    int rows;  // features of a part
    int row_blocks, k_blocks;
    void* out;
    int64_t out_ld;
    int dtype;
    float* out_scale;  // the gated form's
    int64_t os_token, os_block;
    int32_t* status;
};

// kTok tokens and kParts tiles of 128 features a CTA.
template <int kTok, int kParts>
struct Few {
    static constexpr int kCols = kTok * kParts;
    static constexpr int kGroups = kCols > 64 ? 2 : 1;  // warpgroups that take the sums out of tensor memory
    static constexpr int kThreads = 64 + 128 * kGroups;
    static constexpr int kMine = kCols / kGroups;  // columns of a thread
    static constexpr int kBufs = kCols <= 64 ? 4 : 2;
    static constexpr int kTmem = kCols * kBufs;
    // Two CTAs an SM, but for the widest.  CTAs of a cluster wait for one
    // another, so a set of them must never hold tensor memory that another
    // set's CTA waits for on the same SM: at most 256 of 512 columns for a
    // CTA that is not alone, and shared memory of which no third fits.
    static constexpr int kPerSM = kTmem <= 256 ? 2 : 1;
    static constexpr int kStage = kParts * kTileBytes + kTok * kBlock;
    static constexpr int kAhead = 4;  // blocks of scales staged at a time
    static constexpr int kScales = 2 * kAhead * kCols * 4;
    static constexpr int kRoom = kSmemSM / kPerSM - kSmemReserved - 1024 - kScales - 512;
    static constexpr int kStages = kRoom / kStage < 8 ? kRoom / kStage : 8;
    static constexpr int kSmem = 1024 + kStages * kStage + kScales + 512;
    static constexpr int kJoin = kParts == 2 && kTok > 64 ? 64 : kTok;  // tokens joined at a time
    static_assert(kTmem >= 32 && kTmem <= 512 && (kTmem & (kTmem - 1)) == 0, "tensor memory comes in powers of two");
    static_assert(kStages >= 2, "a ring");
    static_assert(kSmem > kSmemSM / 3, "no third CTA on an SM");
    static_assert(kJoin * kParts * kTile * 4 <= kStages * kStage, "the parts are joined in the ring's place");
};

__device__ __forceinline__ void store4(const Product& a, int64_t token, int f, float4 y) {
    const int left = a.rows - f;
    if (left <= 0) return;
    const int64_t at = token * a.out_ld + f;
    if (a.dtype == ZKV_DT_F32) {
        float* to = (float*)a.out + at;
        if (left >= 4 && ((uintptr_t)to & 15) == 0) {
            *reinterpret_cast<float4*>(to) = y;
        } else {
            const float v[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (i < left) to[i] = v[i];
        }
        return;
    }
    uint32_t w[2];
    if (a.dtype == ZKV_DT_BF16) {
        w[0] = pack_bf162(y.x, y.y), w[1] = pack_bf162(y.z, y.w);
    } else {
        const __half2 lo = __floats2half2_rn(y.x, y.y), hi = __floats2half2_rn(y.z, y.w);
        w[0] = *reinterpret_cast<const uint32_t*>(&lo), w[1] = *reinterpret_cast<const uint32_t*>(&hi);
    }
    uint16_t* to = (uint16_t*)a.out + at;
    if (left >= 4 && ((uintptr_t)to & 7) == 0) {
        *reinterpret_cast<uint2*>(to) = make_uint2(w[0], w[1]);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (i < left) to[i] = (uint16_t)(w[i >> 1] >> (16 * (i & 1)));
    }
}

__device__ __forceinline__ float gated(float g, float u) { return g / (1.f + __expf(-g)) * u; }

template <int kTok, int kParts>
__global__ void __launch_bounds__(Few<kTok, kParts>::kThreads)
    few_kernel(const __grid_constant__ CUtensorMap w_map, const __grid_constant__ CUtensorMap x_map, Product a) {
    using C = Few<kTok, kParts>;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t base = (smem_u32(smem_raw) + 1023) & ~1023u;
    const uint32_t scales_at = base + C::kStages * C::kStage;
    const uint32_t bars = scales_at + C::kScales;
    const uint32_t full = bars, empty = full + 8 * C::kStages, sum_full = empty + 8 * C::kStages,
                   sum_empty = sum_full + 8 * C::kBufs, tmem_at = sum_empty + 8 * C::kBufs;
    uint8_t* const generic = smem_raw + (base - smem_u32(smem_raw));
    float* const scales = reinterpret_cast<float*>(generic + C::kStages * C::kStage);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = tc::cluster_rank(), parts = tc::cluster_size();
    const int tile = blockIdx.x / parts;
    const int64_t t0 = (int64_t)blockIdx.y * kTok;
    // this CTA's blocks of the inner dimension
    const int b0 = (int)((int64_t)a.k_blocks * rank / parts), n = (int)((int64_t)a.k_blocks * (rank + 1) / parts) - b0;

    if (threadIdx.x == 0) {
        for (int i = 0; i < C::kStages; ++i) {
            mbar_init(reinterpret_cast<uint64_t*>(generic + (full - base) + 8 * i), 1);
            mbar_init(reinterpret_cast<uint64_t*>(generic + (empty - base) + 8 * i), 1);
        }
        for (int i = 0; i < C::kBufs; ++i) {
            mbar_init(reinterpret_cast<uint64_t*>(generic + (sum_full - base) + 8 * i), 1);
            mbar_init(reinterpret_cast<uint64_t*>(generic + (sum_empty - base) + 8 * i), 4 * C::kGroups);
        }
        mbar_fence_init();
        tc::prefetch_map(&w_map);
        tc::prefetch_map(&x_map);
    }
    if (warp == 1) tc::tmem_alloc(tmem_at, C::kTmem);
    tc::fence_before();
    __syncthreads();
    tc::fence_after();
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(generic + (tmem_at - base));

    float acc[C::kMine];
#pragma unroll
    for (int c = 0; c < C::kMine; ++c) acc[c] = 0.f;

    if (warp == 0) {
        if (lane == 0) {
            int got = 0;
            for (; got < n; ++got) {
                const int s = got % C::kStages, turn = got / C::kStages;
                if (turn > 0 && !tc::wait_for(empty + 8 * s, (turn - 1) & 1, a.status)) break;
                const uint32_t at = base + s * C::kStage, bar = full + 8 * s;
                tc::arrive_expect_tx(bar, C::kStage);
                for (int p = 0; p < kParts; ++p)
                    tc::tma_3d(at + p * kTileBytes, &w_map, (b0 + got) * kBlock, tile * kTile, p, bar);
                tc::tma_2d(at + kParts * kTileBytes, &x_map, (b0 + got) * kBlock, (int)t0, bar);
            }
            // every copy has landed before the CTA ends, whatever became of the others
            for (int i = got > C::kStages ? got - C::kStages : 0; i < got; ++i)
                if (!tc::wait_for(full + 8 * (i % C::kStages), (i / C::kStages) & 1, a.status)) break;
        }
        __syncwarp();
    } else if (warp == 1) {
        if (lane == 0) {
            constexpr uint32_t desc = tc::e4m3_desc(kTile, kTok);
            int done = 0;
            for (; done < n; ++done) {
                const int s = done % C::kStages, b = done % C::kBufs, turn = done / C::kBufs;
                if (!tc::wait_for(full + 8 * s, (done / C::kStages) & 1, a.status)) break;
                if (turn > 0 && !tc::wait_for(sum_empty + 8 * b, (turn - 1) & 1, a.status)) break;
                tc::fence_after();
                const uint32_t at = base + s * C::kStage;
                const uint64_t x = tc::tile_desc(at + kParts * kTileBytes);
#pragma unroll
                for (int p = 0; p < kParts; ++p) {
                    const uint64_t w = tc::tile_desc(at + p * kTileBytes);
#pragma unroll
                    for (int k = 0; k < kBlock / 32; ++k)  // 32 bytes further: 2 of the descriptor's 16
                        tc::mma_e4m3(tmem + b * C::kCols + p * kTok, w + 2 * k, x + 2 * k, desc, k > 0);
                }
                tc::commit(empty + 8 * s);
                tc::commit(sum_full + 8 * b);
            }
            // the last products have ended before tensor memory is given back
            if (done > 0) tc::wait_for(sum_full + 8 * ((done - 1) % C::kBufs), ((done - 1) / C::kBufs) & 1, a.status);
        }
        __syncwarp();
    } else {
        const int e = threadIdx.x - 64, group = (warp - 2) >> 2;
        const uint32_t mine = tmem + ((uint32_t)(warp & 3) << 21) + group * C::kMine;
        const float* ws = a.w_scale + (int64_t)tile * a.k_blocks + b0;
        const int64_t up = (int64_t)a.row_blocks * a.k_blocks;
        constexpr int kEach = (C::kAhead * kTok + C::kThreads - 65) / (C::kThreads - 64);
        // token scales of a few blocks times the weights' scale, one turn ahead in registers, then in shared memory
        float next[kEach][kParts];
        auto fetch = [&](int first) {
#pragma unroll
            for (int j = 0; j < kEach; ++j) {
                const int i = e + j * (C::kThreads - 64), b = first + i / kTok;
                const int64_t t = t0 + i % kTok;
                const bool in = i < C::kAhead * kTok && b < n && t < a.tokens;
                const float x = in ? a.x_scale[t * a.xs_token + (b0 + b) * a.xs_block] : 0.f;
#pragma unroll
                for (int p = 0; p < kParts; ++p) next[j][p] = in ? x * ws[b + p * up] : 0.f;
            }
        };
        fetch(0);
        bool ok = true;  // after a wait that ran out: to the end without another
        for (int kb = 0; kb < n; ++kb) {
            float* const sc = scales + ((kb / C::kAhead) & 1) * C::kAhead * C::kCols;
            if (kb % C::kAhead == 0) {
#pragma unroll
                for (int j = 0; j < kEach; ++j) {
                    const int i = e + j * (C::kThreads - 64);
                    if (i < C::kAhead * kTok)
#pragma unroll
                        for (int p = 0; p < kParts; ++p) sc[(i / kTok) * C::kCols + p * kTok + i % kTok] = next[j][p];
                }
                asm volatile("bar.sync 1, %0;" ::"n"(C::kThreads - 64) : "memory");
                fetch(kb + C::kAhead);
            }
            const float4* by = reinterpret_cast<const float4*>(sc + (kb % C::kAhead) * C::kCols + group * C::kMine);
            const int b = kb % C::kBufs;
            ok = __all_sync(0xffffffffu, ok && tc::wait_for(sum_full + 8 * b, (kb / C::kBufs) & 1, a.status));
            tc::fence_after();
            if (ok) {
#pragma unroll
                for (int c = 0; c < C::kMine; c += 16) {
                    float v[16];
                    tc::ld16(mine + b * C::kCols + c, v);
                    tc::wait_ld();
                    if (c + 16 == C::kMine) {
                        tc::fence_before();
                        if (lane == 0) tc::arrive(sum_empty + 8 * b);
                    }
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float4 s = by[c / 4 + i];
                        acc[c + 4 * i] = fmaf(v[4 * i], s.x, acc[c + 4 * i]);
                        acc[c + 4 * i + 1] = fmaf(v[4 * i + 1], s.y, acc[c + 4 * i + 1]);
                        acc[c + 4 * i + 2] = fmaf(v[4 * i + 2], s.z, acc[c + 4 * i + 2]);
                        acc[c + 4 * i + 3] = fmaf(v[4 * i + 3], s.w, acc[c + 4 * i + 3]);
                    }
                }
            }
        }
        tc::fence_before();
    }
    __syncthreads();
    tc::fence_after();
    if (warp == 1) tc::tmem_free(tmem, C::kTmem);

    // The CTAs' parts, token by token [part][token][feature] in the ring's place; the cluster's CTAs take the tokens in turn.
    float* const join = reinterpret_cast<float*>(generic);
#pragma unroll
    for (int c0 = 0; c0 < kTok; c0 += C::kJoin) {
        if (warp >= 2) {
            const int f = (warp & 3) * 32 + lane, first = (warp - 2) / 4 * C::kMine;
#pragma unroll
            for (int c = 0; c < C::kMine; ++c) {
                const int col = first + c, t = col % kTok - c0;
                if (t >= 0 && t < C::kJoin) join[(col / kTok * C::kJoin + t) * kTile + f] = acc[c];
            }
        }
        if (parts > 1) tc::cluster_sync();
        else __syncthreads();
        for (int t = warp * parts + rank; t < C::kJoin; t += C::kThreads / 32 * parts) {
            const int64_t token = t0 + c0 + t;
            if (token >= a.tokens) break;
            float4 y[kParts];
#pragma unroll
            for (int p = 0; p < kParts; ++p) {
                const uint32_t at = base + ((p * C::kJoin + t) * kTile + lane * 4) * 4;
                y[p] = make_float4(0.f, 0.f, 0.f, 0.f);
                for (uint32_t r = 0; r < parts; ++r) {
                    const float4 v = tc::ld_cluster(tc::in_cta(at, r));
                    y[p].x += v.x, y[p].y += v.y, y[p].z += v.z, y[p].w += v.w;
                }
            }
            const int f = tile * kTile + lane * 4;
            if (kParts == 1) {
                store4(a, token, f, y[0]);
            } else {
                float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
                if (f < a.rows)  // rows are whole 16 bytes
                    v = make_float4(gated(y[0].x, y[kParts - 1].x), gated(y[0].y, y[kParts - 1].y),
                                    gated(y[0].z, y[kParts - 1].z), gated(y[0].w, y[kParts - 1].w));
                const uint32_t m = __reduce_max_sync(
                    0xffffffffu, max(max(magnitude(v.x), magnitude(v.y)), max(magnitude(v.z), magnitude(v.w))));
                const float s = scale_of(m);
                if (f < a.rows)
                    *reinterpret_cast<uint32_t*>((uint8_t*)a.out + token * a.out_ld + f) = e4m3x4(v.x, v.y, v.z, v.w, s);
                if (lane == 0) a.out_scale[token * a.os_token + tile * a.os_block] = s;
            }
        }
        if (parts > 1) tc::cluster_sync();
        else if (c0 + C::kJoin < kTok) __syncthreads();
    }
}

// ------------------------------------------------------------ host
using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                 const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                 CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

static EncodeTiled encode_fn() {
    static EncodeTiled fn = nullptr;
    static std::once_flag once;
    std::call_once(once, [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult qr;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &qr) ==
                cudaSuccess &&
            qr == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<EncodeTiled>(p);
    });
    return fn;
}

// Rows of k bytes, ld apart, in boxes of 128 bytes x `box` rows with the
// 128-byte swizzle; `parts` > 0: so many such matrices after one another.
// What lies past the last row or column reads as zeros.
static bool encode_rows(CUtensorMap* map, const void* at, int64_t k, int64_t rows, int64_t ld, int parts, int box) {
    EncodeTiled fn = encode_fn();
    if (!fn) return false;
    const cuuint64_t dims[3] = {(cuuint64_t)k, (cuuint64_t)rows, (cuuint64_t)std::max(parts, 1)};
    const cuuint64_t strides[2] = {(cuuint64_t)ld, (cuuint64_t)(rows * ld)};
    const cuuint32_t size[3] = {kBlock, (cuuint32_t)box, 1}, es[3] = {1, 1, 1};
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, parts > 0 ? 3 : 2, const_cast<void*>(at), dims, strides, size, es,
              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

static int sm_count() {
    static std::mutex mutex;
    static int count[64] = {};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 0;
    const std::lock_guard<std::mutex> lock(mutex);
    if (!count[dev] && cudaDeviceGetAttribute(&count[dev], cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 0;
    return count[dev];
}

// CTAs of a cluster that share a tile's inner dimension: the number for which the waves of CTAs take the fewest blocks
// after one another, each wave with a fixed cost of about four blocks (filling the ring, joining the parts).
static int parts_of(int64_t tiles, int k_blocks, int places) {
    int best = 1;
    int64_t least = INT64_MAX;
    for (int s = 1; s <= 8 && s <= k_blocks; ++s) {
        const int64_t waves = (tiles * s + places - 1) / places, cost = waves * ((k_blocks + s - 1) / s + 4);
        if (cost < least) least = cost, best = s;
    }
    return best;
}

template <int kTok, int kParts>
static int launch_few(const zkv_fp8_weight* w, const void* x, int64_t x_ld, const Product& a, cudaStream_t stream) {
    using C = Few<kTok, kParts>;
    CUtensorMap x_map;
    if (!encode_rows(&x_map, x, w->k, a.tokens, x_ld, 0, kTok)) return ZKV_ERR_ARG;
    const int sms = sm_count();
    if (!sms) return launch_refused();
    const int64_t wide = (a.tokens + kTok - 1) / kTok;
    if (wide > 65535) return ZKV_ERR_CAPACITY;
    const int parts = parts_of(a.row_blocks * wide, a.k_blocks, sms * C::kPerSM);
    auto kernel = few_kernel<kTok, kParts>;
    if (!raise_smem_limit((const void*)kernel, C::kSmem)) return launch_refused();
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(a.row_blocks * parts), (unsigned)wide, 1);
    cfg.blockDim = dim3(C::kThreads, 1, 1);
    cfg.dynamicSmemBytes = C::kSmem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)parts;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    CUtensorMap w_map;
    memcpy(&w_map, w->map, sizeof w_map);
    if (cudaLaunchKernelEx(&cfg, kernel, w_map, x_map, a) != cudaSuccess) return launch_refused();
    return launch_status();
}

static int check_weight(const zkv_fp8_weight* w) {
    if (!w || !w->w || !w->scale || w->rows < 1 || w->k < 1 || w->ld < w->k) return ZKV_ERR_ARG;
    if (w->parts != 1 && w->parts != 2) return ZKV_ERR_ARG;
    if (w->k % 16 || (w->parts == 2 && w->rows % 16)) return ZKV_ERR_UNSUPPORTED;
    if (!aligned16(w->w) || w->ld % 16) return ZKV_ERR_ALIGN;
    // a tile's coordinates, its scale's index and the tensor map's strides
    if (w->rows > 1 << 30 || w->k > 1 << 24 || w->ld > (int64_t)1 << 32) return ZKV_ERR_CAPACITY;
    return ZKV_OK;
}

// x and the handle, for both entries; fills what they share of `a`.
static int check_call(const void* x, int64_t x_ld, const float* x_scale, int64_t xs_token, int64_t xs_block, int64_t tokens,
                      const zkv_fp8_weight* w, const void* out, int64_t out_ld, int32_t* status, Product* a) {
    if (const int rc = check_weight(w)) return rc;
    if (!x || !x_scale || !out || tokens < 0 || x_ld < w->k || out_ld < w->rows || xs_token < 0 || xs_block < 0)
        return ZKV_ERR_ARG;
    if (!aligned16(x) || x_ld % 16) return ZKV_ERR_ALIGN;
    if (tokens > INT32_MAX || x_ld > (int64_t)1 << 32) return ZKV_ERR_CAPACITY;
    *a = {};
    a->x_scale = x_scale, a->xs_token = xs_token, a->xs_block = xs_block, a->w_scale = w->scale, a->tokens = tokens;
    a->rows = (int)w->rows, a->row_blocks = blocks_of(w->rows), a->k_blocks = blocks_of(w->k);
    a->out = const_cast<void*>(out), a->out_ld = out_ld, a->status = status;
    return ZKV_OK;
}

template <int kParts>
static int launch(const zkv_fp8_weight* w, const void* x, int64_t x_ld, const Product& a, cudaStream_t stream) {
    if (a.tokens <= 16) return launch_few<16, kParts>(w, x, x_ld, a, stream);
    if (a.tokens <= 32) return launch_few<32, kParts>(w, x, x_ld, a, stream);
    if (a.tokens <= 64) return launch_few<64, kParts>(w, x, x_ld, a, stream);
    return launch_few<128, kParts>(w, x, x_ld, a, stream);
}

}  // namespace fp8
}  // namespace zkv

using namespace zkv;

extern "C" int zkv_fp8_weight_init(zkv_fp8_weight* w) {
    if (const int rc = fp8::check_weight(w)) return rc;
    static_assert(sizeof(CUtensorMap) == sizeof w->map, "map");
    CUtensorMap map;
    if (!fp8::encode_rows(&map, w->w, w->k, w->rows, w->ld, w->parts, fp8::kTile)) return ZKV_ERR_ARG;
    memcpy(w->map, &map, sizeof map);
    return ZKV_OK;
}

extern "C" int zkv_fp8_linear(const void* x, int64_t x_ld, const float* x_scale, int64_t xs_token, int64_t xs_block,
                              int64_t tokens, const zkv_fp8_weight* w, void* out, int64_t out_ld, int dtype,
                              int32_t* status, void* stream) {
    fp8::Product a;
    if (const int rc = fp8::check_call(x, x_ld, x_scale, xs_token, xs_block, tokens, w, out, out_ld, status, &a)) return rc;
    if (w->parts != 1 || (dtype != ZKV_DT_BF16 && dtype != ZKV_DT_F16 && dtype != ZKV_DT_F32)) return ZKV_ERR_ARG;
    if (reinterpret_cast<uintptr_t>(out) & (dtype == ZKV_DT_F32 ? 3 : 1)) return ZKV_ERR_ALIGN;
    if (tokens == 0) return ZKV_OK;
    a.dtype = dtype;
    return fp8::launch<1>(w, x, x_ld, a, (cudaStream_t)stream);
}

extern "C" int zkv_fp8_swiglu(const void* x, int64_t x_ld, const float* x_scale, int64_t xs_token, int64_t xs_block,
                              int64_t tokens, const zkv_fp8_weight* w, void* out, int64_t out_ld, float* out_scale,
                              int64_t os_token, int64_t os_block, int32_t* status, void* stream) {
    fp8::Product a;
    if (const int rc = fp8::check_call(x, x_ld, x_scale, xs_token, xs_block, tokens, w, out, out_ld, status, &a)) return rc;
    if (w->parts != 2 || !out_scale || os_token < 1 || os_block < 1) return ZKV_ERR_ARG;
    if (!fp8::aligned16(out) || out_ld % 16) return ZKV_ERR_ALIGN;
    if (tokens == 0) return ZKV_OK;
    a.out_scale = out_scale, a.os_token = os_token, a.os_block = os_block;
    return fp8::launch<2>(w, x, x_ld, a, (cudaStream_t)stream);
}
