// zkv_fp8_gemm.cu -- products of e4m3 rows with e4m3 weights, both with fp32
// scales for blocks of 128 (rows: 1 x 128, weights: 128 x 128), and the gated
// form whose output is e4m3 with block scales again:
//   y[m][n] = sum_b xs[m][b] ws[n / 128][b] sum_{k in block b} x[m][k] w[n][k]
//   a[m][f] = silu(g) u, g and u the two parts' products, stored as blocks
// The scales change with every block of the inner dimension, so each block's
// sum of 128 products (tcgen05, fp32 in tensor memory) is read back, scaled
// and added in fp32 registers.
//
// Up to 64 tokens features are the rows of the tensor core's tile (128 lanes)
// and tokens its columns: a step of few tokens fills the tile all the same,
// and the weights go from memory to the tensor core without passing a
// register.  What bounds such a call is reading the weights once (32 tokens x
// 151936 x 4096: 103 us, 6.2 TB/s), and below some 50 MB of weights the chain
// launch - first copies - products - join (8 tokens x 4096 x 4096: 6.2 us for
// 2.6 of bytes).  Tiles that are fewer than the SMs are cut along the inner
// dimension over a cluster, whose CTAs add their parts through distributed
// shared memory in the order of their ranks.  From 65 tokens on the tokens are
// the rows; long prompts take pairs of CTAs (below).
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
constexpr int kBox = 64;         // features of a copy

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
    // 128 tokens are the rows of the tensor core's tile themselves: a reader then has a token of its own and one scale for
    // all its columns, where with features as rows it loads a scale for each (as many bytes of shared memory as of sums).
    static constexpr bool kTokenRows = kTok == kTile;
    static constexpr int kCols = kTok * kParts;  // columns of tensor memory for a block
    static constexpr int kGroups = kCols >= 128 ? 4 : kCols >= 64 ? 2 : 1;  // warpgroups that take the sums out of tensor memory
    static constexpr int kReaders = 128 * kGroups, kThreads = 96 + kReaders;
    static constexpr int kMine = kCols / kGroups;  // columns of a thread
    static constexpr int kLoad = kMine == 32 ? 32 : 16;  // columns of a load (64 columns: what registers leave room for)
    static constexpr int kBufs = kCols == 256 ? 2 : kCols >= 64 ? 4 : 8;
    static constexpr int kTmem = kCols * kBufs;
    static constexpr int kStage = kParts * kTileBytes + kTok * kBlock;
    static constexpr int kAhead = 4;  // blocks of scales staged at a time
    static constexpr int kScales = 2 * kAhead * kCols * 4;
    static constexpr int kPitch = kTokenRows ? kTile + 4 : kTile;  // floats from token to token where they are joined
    static constexpr int kMost = 12;  // stages of the ring: barriers
    static constexpr int smem(int stages) { return 1024 + stages * kStage + kScales + 512; }
    static constexpr int stages_in(int bytes) {
        return (bytes - smem(0)) / kStage < kMost ? (bytes - smem(0)) / kStage : kMost;
    }
    // The ring takes an SM's shared memory, or half of it, for two CTAs an SM: for one part and up to 32 tokens (151936 x
    // 4096: 8 tokens 97 us, 106 with one; 32 tokens 101 and 119).  More tokens take the registers of one, and two parts'
    // stages are too few in half the memory (8 tokens of 12288 x 4096: 23.3 us, 21.7 with one).
    // The CTAs of a cluster wait for one another, so none may have to wait for tensor memory that a CTA of another cluster
    // holds on its SM: at most two CTAs of this file's kernels fit on an SM (each takes more than a third of its shared
    // memory), with at most half of the tensor memory each; one that takes more of it fits beside none.
    static constexpr bool kHalves = kParts == 1 && kTok <= 32;
    // Even, as the buffers are: a stage is always the same issuing warp's.  A wait for a phase by its parity lets a warp
    // through at once while the phase before, another warp's, has not ended.
    static constexpr int kStages = stages_in((kHalves ? 113 : 227) * 1024) / 2 * 2;
    static_assert(kStages % 2 == 0 && kBufs % 2 == 0, "a stage and a buffer have one issuing warp");
    static_assert(kTmem >= 32 && kTmem <= 512 && (kTmem & (kTmem - 1)) == 0, "tensor memory comes in powers of two");
    static_assert(kTmem <= 256 || smem(kStages) > (227 - 76) * 1024, "alone on its SM");
    static_assert(smem(kStages) > 76 * 1024, "no third CTA on an SM");
    // and the registers are the launch bounds'
    static_assert(!kHalves || (2 * (smem(kStages) + 1024) <= 228 * 1024 && 2 * kTmem <= 512), "two CTAs an SM");
    static_assert(kMine % kLoad == 0, "whole loads");
    static_assert(16 * (kMost + kBufs) + 4 <= 512, "barriers");
    static_assert(kStages >= 2 && kTok * kParts * kPitch * 4 <= kStages * kStage, "the parts are joined in the ring's place");
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

// silu(g) u: g u / (1 + h^2) with h = exp(-|g| / 2) = 2^(-|g| log2(e) / 2), times h^2 where g is below zero, one h on either
// side of u.  So nothing on the way leaves fp32's range while h is in it (|g| < 174) and the result is, and the forms of
// the two instructions that flush subnormal numbers will do: exp(-g) itself overflows at g = -88.7.  h is off by 2^-22 of
// itself and, for its argument's roundings, |g| 2^-24, twice over; the reciprocal by 2^-23 and the five other operations by
// 2^-24 each: a relative error of at most (|g| + 8) 2^-23.
__device__ __forceinline__ float gated(float g, float u) {
    float h, r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(h) : "f"(fabsf(g) * -0.72134752f));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(fmaf(h, h, 1.f)));
    const float below = g < 0.f ? h : 1.f;
    return g * r * below * u * below;
}

template <int kTok, int kParts>
__global__ void __launch_bounds__(Few<kTok, kParts>::kThreads, Few<kTok, kParts>::kHalves ? 2 : 1)
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
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
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
    if (warp == 1) tc::tmem_alloc<C::kTmem>(tmem_at);
    // while the kernel before this one may still run: the first weights on their way into L2
    if (warp == 0 && t0 == 0)
        for (int i = lane; i < 2 * kParts * min(n, C::kStages); i += 32)
            tc::prefetch_3d(&w_map, (b0 + i / (2 * kParts)) * kBlock, tile * kTile + (i & 1) * kBox, i / 2 % kParts);
    tc::fence_before();
    __syncthreads();
    tc::fence_after();
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(generic + (tmem_at - base));
    grid_dep_wait();
    grid_dep_launch_next();

    float acc[C::kMine];
#pragma unroll
    for (int c = 0; c < C::kMine; ++c) acc[c] = 0.f;

    if (warp == 0) {
        int got = 0, s = 0, phase = 1;  // of `empty`: a fresh barrier's last phase counts as over
        for (; got < n; ++got) {
            if (!tc::wait_all(empty + 8 * s, phase, a.status)) break;
            const uint32_t at = base + s * C::kStage, bar = full + 8 * s;
            if (tc::elected()) {
                tc::arrive_expect_tx(bar, C::kStage);
                for (int p = 0; p < 2 * kParts; ++p)
                    tc::tma_3d(at + p * kBox * kBlock, &w_map, (b0 + got) * kBlock, tile * kTile + (p & 1) * kBox, p >> 1, bar);
                tc::tma_2d(at + kParts * kTileBytes, &x_map, (b0 + got) * kBlock, (int)t0, bar);
            }
            __syncwarp();
            if (++s == C::kStages) s = 0, phase ^= 1;
        }
        // every copy has landed before the CTA ends, whatever became of the others
        for (int i = got > C::kStages ? got - C::kStages : 0; i < got; ++i)
            if (!tc::wait_all(full + 8 * (i % C::kStages), (i / C::kStages) & 1, a.status)) break;
    } else if (warp <= 2) {
        // Two warps issue every other block's products: to pass two barriers takes a warp some 400 clocks, to issue 400 more.
        int done = warp - 1;
        for (; done < n; done += 2) {
            const int s = done % C::kStages, b = done % C::kBufs, turn = done / C::kBufs;
            if (turn > 0 && !tc::wait_all(sum_empty + 8 * b, (turn - 1) & 1, a.status)) break;
            if (!tc::wait_all(full + 8 * s, (done / C::kStages) & 1, a.status)) break;
            tc::fence_after();
            const uint32_t at = base + s * C::kStage, d = tmem + b * C::kCols;
            const uint64_t x = tc::tile_desc(at + kParts * kTileBytes);
            if (tc::elected()) {
                if (C::kTokenRows) {
                    constexpr uint32_t desc = tc::e4m3_desc(kTile, kParts * kTile);
                    const uint64_t w = tc::tile_desc(at);
#pragma unroll
                    for (int k = 0; k < kBlock / 32; ++k)  // 32 bytes further: 2 of the descriptor's 16
                        tc::mma_e4m3(d, x + 2 * k, w + 2 * k, desc, k > 0);
                } else {
                    constexpr uint32_t desc = tc::e4m3_desc(kTile, kTok);
#pragma unroll
                    for (int p = 0; p < kParts; ++p) {
                        const uint64_t w = tc::tile_desc(at + p * kTileBytes);
#pragma unroll
                        for (int k = 0; k < kBlock / 32; ++k) tc::mma_e4m3(d + p * kTok, w + 2 * k, x + 2 * k, desc, k > 0);
                    }
                }
                tc::commit(sum_full + 8 * b);
                tc::commit(empty + 8 * s);
            }
            __syncwarp();
        }
        // its last products have ended before tensor memory is given back
        done -= 2;
        if (done >= 0) tc::wait_all(sum_full + 8 * (done % C::kBufs), (done / C::kBufs) & 1, a.status);
    } else {
        const int e = threadIdx.x - 96, group = (warp - 3) >> 2;
        const uint32_t mine = tmem + ((uint32_t)(warp & 3) << 21) + group * C::kMine;
        const float* ws = a.w_scale + (int64_t)tile * a.k_blocks + b0;
        const int64_t up = (int64_t)a.row_blocks * a.k_blocks;
        constexpr int kEach = (C::kAhead * kTok + C::kReaders - 1) / C::kReaders;
        // token scales of a few blocks times the weights' scale, one turn ahead in registers, then in shared memory
        float next[kEach][kParts];
        auto fetch = [&](int first) {
#pragma unroll
            for (int j = 0; j < kEach; ++j) {
                const int i = e + j * C::kReaders, b = first + i / kTok;
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
                    const int i = e + j * C::kReaders;
                    if (i < C::kAhead * kTok)
#pragma unroll
                        for (int p = 0; p < kParts; ++p) sc[(i / kTok) * C::kCols + p * kTok + i % kTok] = next[j][p];
                }
                asm volatile("bar.sync 1, %0;" ::"n"(C::kReaders) : "memory");
                fetch(kb + C::kAhead);
            }
            const float* by = sc + (kb % C::kAhead) * C::kCols +
                              (C::kTokenRows ? group * C::kMine / kTile * kTile + (warp & 3) * 32 + lane : group * C::kMine);
            const float own = *by;  // token rows: this thread's
            const int b = kb % C::kBufs;
            ok = __all_sync(0xffffffffu, ok && tc::wait_for(sum_full + 8 * b, (kb / C::kBufs) & 1, a.status));
            tc::fence_after();
            if (ok) {
#pragma unroll
                for (int c = 0; c < C::kMine; c += C::kLoad) {
                    uint32_t v[C::kLoad];
                    tc::ld(mine + b * C::kCols + c, v);
                    tc::wait_ld(v);
                    if (c + C::kLoad == C::kMine) {
                        tc::fence_before();
                        if (lane == 0) tc::arrive(sum_empty + 8 * b);
                    }
#pragma unroll
                    for (int i = 0; i < C::kLoad; i += 4) {
                        const float4 s = C::kTokenRows ? make_float4(own, own, own, own)
                                                       : *reinterpret_cast<const float4*>(by + c + i);
                        acc[c + i] = fmaf(__uint_as_float(v[i]), s.x, acc[c + i]);
                        acc[c + i + 1] = fmaf(__uint_as_float(v[i + 1]), s.y, acc[c + i + 1]);
                        acc[c + i + 2] = fmaf(__uint_as_float(v[i + 2]), s.z, acc[c + i + 2]);
                        acc[c + i + 3] = fmaf(__uint_as_float(v[i + 3]), s.w, acc[c + i + 3]);
                    }
                }
            }
        }
        tc::fence_before();
    }
    __syncthreads();
    tc::fence_after();
    if (warp == 1) tc::tmem_free<C::kTmem>(tmem);

    // The CTAs' parts, token by token [part][token][feature] in the ring's place; the cluster's CTAs take the tokens in
    // turn, a warp some at a time.
    float* const join = reinterpret_cast<float*>(generic);
    if (warp >= 3) {
        const int row = (warp & 3) * 32 + lane, first = (warp - 3) / 4 * C::kMine;
        if (C::kTokenRows) {
            float* to = join + (first / kTile * kTok + row) * C::kPitch + first % kTile;
#pragma unroll
            for (int c = 0; c < C::kMine; c += 4)
                *reinterpret_cast<float4*>(to + c) = make_float4(acc[c], acc[c + 1], acc[c + 2], acc[c + 3]);
        } else {
#pragma unroll
            for (int c = 0; c < C::kMine; ++c) {
                const int col = first + c;
                join[(col / kTok * kTok + col % kTok) * C::kPitch + row] = acc[c];
            }
        }
    }
    if (parts > 1) tc::cluster_sync();
    else __syncthreads();
    constexpr int kAtOnce = kTok >= 128 && kParts == 2 ? 4 : 2;
    const int turn = C::kThreads / 32 * parts, f = tile * kTile + lane * 4;
    const int most = (int)min((int64_t)kTok, a.tokens - t0);  // tokens of this tile
    for (int t = warp * parts + rank; t < most; t += kAtOnce * turn) {
        float4 y[kAtOnce][kParts];
        auto at = [&](int u, int p) { return (p * kTok + t + u * turn) * C::kPitch + lane * 4; };
        auto have = [&](int u) { return t + u * turn < most; };
#pragma unroll
        for (int u = 0; u < kAtOnce; ++u)
#pragma unroll
            for (int p = 0; p < kParts; ++p)
                y[u][p] = parts == 1 && have(u) ? *reinterpret_cast<const float4*>(join + at(u, p))
                                                : make_float4(0.f, 0.f, 0.f, 0.f);
        for (uint32_t r = 0; parts > 1 && r < parts; ++r) {
            const uint32_t from = tc::in_cta(base, r);
            float4 v[kAtOnce][kParts];
#pragma unroll
            for (int u = 0; u < kAtOnce; ++u)
#pragma unroll
                for (int p = 0; p < kParts; ++p)
                    v[u][p] = have(u) ? tc::ld_cluster(from + at(u, p) * 4) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int u = 0; u < kAtOnce; ++u)
#pragma unroll
                for (int p = 0; p < kParts; ++p)
                    y[u][p].x += v[u][p].x, y[u][p].y += v[u][p].y, y[u][p].z += v[u][p].z, y[u][p].w += v[u][p].w;
        }
        if (kParts == 1) {
#pragma unroll
            for (int u = 0; u < kAtOnce; ++u)
                if (have(u)) store4(a, t0 + t + u * turn, f, y[u][0]);
        } else {
            uint32_t q[kAtOnce];
            float s[kAtOnce];
#pragma unroll
            for (int u = 0; u < kAtOnce; ++u) {
                const float4 g = y[u][0], h = y[u][kParts - 1];
                float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
                if (f < a.rows)  // rows are whole 16 bytes
                    v = make_float4(gated(g.x, h.x), gated(g.y, h.y), gated(g.z, h.z), gated(g.w, h.w));
                s[u] = scale_of(__reduce_max_sync(
                    0xffffffffu, max(max(magnitude(v.x), magnitude(v.y)), max(magnitude(v.z), magnitude(v.w)))));
                const Quotient by(s[u]);
                float e[4] = {v.x, v.y, v.z, v.w};
                by.prepare(e);
                q[u] = by.e4m3(e[0], e[1], e[2], e[3]);
            }
#pragma unroll
            for (int u = 0; u < kAtOnce; ++u) {
                const int64_t to = t0 + t + u * turn;
                if (!have(u)) break;
                if (f < a.rows) *reinterpret_cast<uint32_t*>((uint8_t*)a.out + to * a.out_ld + f) = q[u];
                if (lane == 0) a.out_scale[to * a.os_token + tile * a.os_block] = s[u];
            }
        }
    }
    if (parts > 1) tc::cluster_sync();
}

// ------------------------------------------------------------ many tokens
// Tokens are the matrix rows: 256 of them and 256 features a tile (gated: 128
// of each part), by a pair of CTAs whose tensor cores share the features'
// operand, so that a CTA loads 32 KB for a block of the inner dimension
// instead of 48 (96 bytes a clock at the full rate, more than L2 gives an SM).
// Each block's sums go to tensor memory, and from there, scaled, into fp32
// registers: a thread has one token and 128 features, and both scales are its
// own.  The tensor core would have to wait while a block's sums are read and
// the barriers pass between the two CTAs (some 1100 clocks for the 512 of a
// block), so the tile is multiplied in two halves of 128 features with two
// buffers of tensor memory each, every half by an issuing warp and a
// warpgroup of readers of its own.
// 4096 x 6144 x 4096: 93 us (2.2 PFLOP/s; 78 us with the readers' loop taken
// out of a copy, six waves of tiles for 5.2); in a loop at the power limit 107
// us at 1.49 GHz (92 without the readers).  Sixteen warps of readers with 64
// features each took 105 and 121: more instructions for the same sums.  Packed
// products and sums of two elements changed nothing.
template <bool kGated>
struct Many {
    static constexpr int kTokens = 256, kFeatures = 256;
    // A warpgroup for the copies and products, two of readers, which take the registers that the first gives up:
    // 128 x 72 + 256 x 216 of the 384 x 168 of the launch.
    static constexpr int kReaders = 256, kThreads = 128 + kReaders;
    static constexpr int kStages = 4;
    static constexpr int kStage = 2 * kTileBytes;  // 128 rows of tokens, 128 of features
    // Output staging: two tiles for each warpgroup; gated: one in all, and the sums that warpgroups exchange.
    static constexpr int kOut = (kGated ? 5 : 4) * kTileBytes;
    static constexpr int kTop = kGated ? 1024 : 0;
    // Scales come to shared memory by a warp of their own, four blocks of the inner dimension at a time: the readers pass
    // one barrier for them in four blocks, and none waits for global memory.
    static constexpr int kBatch = 4, kSlots = 2, kSlot = kBatch * 4 * (128 + 2);  // 128 tokens, two of the weights
    static constexpr int kSmem = 1024 + kStages * kStage + kOut + kTop + kSlots * kSlot + 256;
    static_assert(kSmem <= 227 * 1024, "shared memory");
};

struct ManyTiles {
    int m, n;    // tiles of tokens and of features
    int total;   // m * n
    // Eight tiles of tokens by all tiles of features after one another: a wave reads few of either.
    __device__ __forceinline__ void at(int t, int& tm, int& tn) const {
        const int per = 8 * n, g = t / per, first = g * 8, high = min(8, m - first), r = t - g * per;
        tm = first + r % high;
        tn = r / high;
    }
};

__device__ __forceinline__ void group_sync(int group) {
    asm volatile("bar.sync %0, 128;" ::"r"(1 + group) : "memory");
}

__device__ __forceinline__ void readers_sync() { asm volatile("bar.sync 3, 256;" ::: "memory"); }

// 16 bytes of row r of a swizzled tile of 128-byte rows.
__device__ __forceinline__ uint32_t swizzled(uint32_t tile, int r, int chunk) {
    return tile + r * 128 + ((chunk ^ (r & 7)) << 4);
}
__device__ __forceinline__ void st_shared(uint32_t at, uint4 v) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
__device__ __forceinline__ void st_shared1(uint32_t at, uint32_t v) {
    asm volatile("st.shared.b32 [%0], %1;" ::"r"(at), "r"(v) : "memory");
}
template <typename T>
__device__ __forceinline__ T ld_shared(uint32_t at) {
    if (sizeof(T) == 2) {
        uint16_t v;
        asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(at) : "memory");
        return (T)v;
    }
    uint32_t v;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(at) : "memory");
    return (T)v;
}

__device__ __forceinline__ float4 ld_shared4(uint32_t at) {
    float4 v;
    asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(at) : "memory");
    return v;
}

// One swizzled tile of 128 rows to an output whose rows do not start on 16 bytes: by a warpgroup, element by element.
template <typename T>
__device__ __forceinline__ void copy_out(const Product& a, uint32_t tile, int64_t token, int f, int columns) {
    const int warp = (threadIdx.x >> 5) & 3, lane = threadIdx.x & 31;
    for (int r = warp; r < 128; r += 4) {
        if (token + r >= a.tokens) break;
        T* to = (T*)a.out + (token + r) * a.out_ld + f;
        for (int c = lane; c < columns; c += 32) {
            const int byte = c * (int)sizeof(T);
            if (f + c < a.rows) to[c] = ld_shared<T>(swizzled(tile, r, byte >> 4) + (byte & 15));
        }
    }
}

// Whether a row's last features end inside 16 bytes of this tile: a tensor map's store writes those 16 bytes whole.
__device__ __forceinline__ bool cut_short(int rows, int f, int columns, int element) {
    return f + columns > rows && rows * (int64_t)element % 16;
}

template <bool kGated>
__global__ void __launch_bounds__(Many<kGated>::kThreads, 1)
    many_kernel(const __grid_constant__ CUtensorMap w_map, const __grid_constant__ CUtensorMap x_map,
                const __grid_constant__ CUtensorMap out_map, Product a, ManyTiles tiles, bool mapped) {
    using C = Many<kGated>;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t base = (smem_u32(smem_raw) + 1023) & ~1023u;
    uint8_t* const generic = smem_raw + (base - smem_u32(smem_raw));
    const uint32_t out_at = base + C::kStages * C::kStage, top_at = out_at + C::kOut, slots = top_at + C::kTop,
                   bars = slots + C::kSlots * C::kSlot;
    const uint32_t full = bars, empty = full + 8 * C::kStages, sum_full = empty + 8 * C::kStages, sum_empty = sum_full + 32,
                   slot_full = sum_empty + 32, slot_empty = slot_full + 8 * C::kSlots, tmem_at = slot_empty + 8 * C::kSlots;
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const uint32_t rank = tc::cluster_rank();
    const int n = a.k_blocks, pairs = gridDim.x >> 1;

    if (threadIdx.x == 0) {
        auto bar = [&](uint32_t at) { return reinterpret_cast<uint64_t*>(generic + (at - base)); };
        for (int i = 0; i < C::kStages; ++i) {
            mbar_init(bar(full + 8 * i), 1);
            mbar_init(bar(empty + 8 * i), 2);  // both halves
        }
        for (int i = 0; i < 4; ++i) {
            mbar_init(bar(sum_full + 8 * i), 1);
            mbar_init(bar(sum_empty + 8 * i), 8);  // a half's 4 warps of readers, of both CTAs
        }
        for (int i = 0; i < C::kSlots; ++i) {
            mbar_init(bar(slot_full + 8 * i), 32);
            mbar_init(bar(slot_empty + 8 * i), C::kReaders / 32);
        }
        mbar_fence_init();
        tc::prefetch_map(&w_map);
        tc::prefetch_map(&x_map);
    }
    if (warp == 1) tc::tmem_alloc_pair(tmem_at, 512);
    tc::fence_before();
    __syncthreads();
    tc::cluster_sync();  // both CTAs' barriers
    tc::fence_after();
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(generic + (tmem_at - base));
    grid_dep_wait();
    grid_dep_launch_next();

    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
      if (warp == 0) {
        const uint32_t leader = tc::in_cta(full, 0);
        int got = 0;
        bool ok = true;
        for (int t = blockIdx.x >> 1; t < tiles.total && ok; t += pairs) {
            int tm, tn;
            tiles.at(t, tm, tn);
            const int token = tm * C::kTokens + rank * 128;
            // 64 of each half's 128 features
            const int first = (kGated ? tn : 2 * tn) * kTile + (int)rank * kBox, second = kGated ? first : first + kTile;
            for (int kb = 0; kb < n; ++kb, ++got) {
                const int s = got % C::kStages, turn = got / C::kStages;
                if (turn > 0 && !(ok = tc::wait_all(empty + 8 * s, (turn - 1) & 1, a.status))) break;
                const uint32_t at = base + s * C::kStage;
                if (tc::elected()) {
                    if (rank == 0) tc::arrive_expect_tx(full + 8 * s, 2 * C::kStage);
                    tc::tma_2d_pair(at, &x_map, kb * kBlock, token, leader + 8 * s);
                    tc::tma_3d_pair(at + kTileBytes, &w_map, kb * kBlock, first, 0, leader + 8 * s);
                    tc::tma_3d_pair(at + kTileBytes + kBox * kBlock, &w_map, kb * kBlock, second, kGated ? 1 : 0,
                                    leader + 8 * s);
                }
                __syncwarp();
            }
        }
        // both CTAs' copies have landed before either ends, whatever became of the others
        if (rank == 0)
            for (int i = got > C::kStages ? got - C::kStages : 0; i < got; ++i)
                if (!tc::wait_all(full + 8 * (i % C::kStages), (i / C::kStages) & 1, a.status)) break;
      } else if (warp != 2 && rank == 0) {
        const int half = warp >> 1;
        constexpr uint32_t desc = tc::e4m3_desc(256, kTile);
        int done = 0;
        bool ok = true;
        for (int t = blockIdx.x >> 1; t < tiles.total && ok; t += pairs) {
            for (int kb = 0; kb < n; ++kb, ++done) {
                const int s = done % C::kStages, b = half + 2 * (done & 1), turn = done >> 1;
                if (turn > 0 && !(ok = tc::wait_all(sum_empty + 8 * b, (turn - 1) & 1, a.status))) break;
                if (!(ok = tc::wait_all(full + 8 * s, (done / C::kStages) & 1, a.status))) break;
                tc::fence_after();
                const uint64_t x = tc::tile_desc(base + s * C::kStage),
                               w = tc::tile_desc(base + s * C::kStage + kTileBytes + half * kBox * kBlock);
                if (tc::elected()) {
#pragma unroll
                    for (int k = 0; k < kBlock / 32; ++k)
                        tc::mma_e4m3_pair(tmem + b * kTile, x + 2 * k, w + 2 * k, desc, k > 0);
                    tc::commit_pair(sum_full + 8 * b);
                    tc::commit_pair(empty + 8 * s);
                }
                __syncwarp();
            }
        }
        // the last products have ended before tensor memory is given back
        if (done > 0)
            tc::wait_all(sum_full + 8 * (half + 2 * ((done - 1) & 1)), ((done - 1) >> 1) & 1, a.status);
      } else if (warp == 2) {
        const int64_t up = (int64_t)a.row_blocks * a.k_blocks;
        int got = 0;
        bool ok = true;
        for (int t = blockIdx.x >> 1; t < tiles.total && ok; t += pairs) {
            int tm, tn;
            tiles.at(t, tm, tn);
            const int64_t token = (int64_t)tm * C::kTokens + rank * 128 + lane;
            const float* xs = a.x_scale + token * a.xs_token;
            // lanes 0 and 1: the weights' scales of the two halves
            const int wb = kGated ? tn : min(2 * tn + lane, a.row_blocks - 1);
            const float* ws = a.w_scale + (int64_t)wb * a.k_blocks + (kGated ? lane * up : 0);
            for (int kb = 0; kb < n; kb += C::kBatch, ++got) {
                const int s = got % C::kSlots, turn = got / C::kSlots;
                const uint32_t at = slots + s * C::kSlot;
                if (turn > 0 && !(ok = tc::wait_all(slot_empty + 8 * s, (turn - 1) & 1, a.status))) break;
#pragma unroll
                for (int j = 0; j < C::kBatch; ++j) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const bool in = kb + j < n && token + 32 * i < a.tokens;
                        tc::copy4(at + (lane + 32 * i) * 16 + 4 * j,
                                  in ? xs + 32 * i * a.xs_token + (kb + j) * a.xs_block : a.x_scale, in);
                    }
                    if (lane < 2) tc::copy4(at + 2048 + lane * 16 + 4 * j, kb + j < n ? ws + kb + j : a.w_scale, kb + j < n);
                }
                tc::copy4_arrive(slot_full + 8 * s);
            }
        }
        tc::copy4_wait();
      }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
        const int half = (warp - 4) >> 2, row = (warp & 3) * 32 + lane;  // a warpgroup reads one half
        const uint32_t mine = tmem + ((uint32_t)(warp & 3) << 21) + half * kTile;
        const uint32_t empty_at = tc::in_cta(sum_empty + 8 * half, 0);
        const uint32_t staging = out_at + half * 2 * kTileBytes;
        const uint32_t top = top_at + row * 4;  // [2][128]: a group's largest magnitude of a token
        const bool issues = threadIdx.x == 128 + 128 * half;
        bool ok = true;
        int done = 0, batch = 0;
        for (int t = blockIdx.x >> 1; t < tiles.total; t += pairs) {
            int tm, tn;
            tiles.at(t, tm, tn);
            const int64_t token0 = (int64_t)tm * C::kTokens + rank * 128, token = token0 + row;
            const bool live = token < a.tokens;
            float acc[128];
#pragma unroll
            for (int c = 0; c < 128; ++c) acc[c] = 0.f;
            uint32_t even[32], odd[32];
            auto add = [&](int c, const uint32_t(&v)[32], float by) {
#pragma unroll
                for (int i = 0; i < 32; ++i) acc[32 * c + i] = fmaf(__uint_as_float(v[i]), by, acc[32 * c + i]);
            };
            for (int kb = 0; kb < n; kb += C::kBatch, ++batch) {
                const int slot = batch % C::kSlots;
                ok = ok && tc::wait_all(slot_full + 8 * slot, (batch / C::kSlots) & 1, a.status);
                const uint32_t scales = slots + slot * C::kSlot;
                const float4 x4 = ld_shared4(scales + row * 16), w4 = ld_shared4(scales + 2048 + half * 16);
                const float by[4] = {x4.x * w4.x, x4.y * w4.y, x4.z * w4.z, x4.w * w4.w};
                __syncwarp();
                if (lane == 0) tc::arrive(slot_empty + 8 * slot);
#pragma unroll
                for (int j = 0; j < C::kBatch; ++j) {
                    if (kb + j >= n) break;
                    ok = ok && tc::wait_all(sum_full + 8 * (half + 2 * (done & 1)), (done >> 1) & 1, a.status);
                    tc::fence_after();
                    const uint32_t at = mine + (done & 1) * 2 * kTile;
                    tc::ld(at, even);
                    tc::wait_ld(even);
                    tc::ld(at + 32, odd);
                    add(0, even, by[j]);
                    tc::wait_ld(odd);
                    tc::ld(at + 64, even);
                    add(1, odd, by[j]);
                    tc::wait_ld(even);
                    tc::ld(at + 96, odd);
                    add(2, even, by[j]);
                    tc::wait_ld(odd);
                    tc::fence_before();
                    if (lane == 0) tc::arrive_cluster(empty_at + 16 * (done & 1));
                    add(3, odd, by[j]);
                    ++done;
                }
            }
            // the staging's last tile has been read
            if (mapped && issues) tc::store_wait_read();
            if (kGated) {
                // One warpgroup holds the gate's 128 features of a token, the other the up part's: each gives the other half of
                // them and finishes the other half.
                const uint32_t give = out_at + kTileBytes + half * 2 * kTileBytes + row * 4;
#pragma unroll
                for (int i = 0; i < 64; ++i) st_shared1(give + i * 512, __float_as_uint(half ? acc[i] : acc[64 + i]));
                readers_sync();
                const uint32_t from = out_at + kTileBytes + (half ^ 1) * 2 * kTileBytes + row * 4;
                uint32_t m = 0;
                const int f0 = tn * kTile + half * 64;
#pragma unroll
                for (int i = 0; i < 64; ++i) {
                    const float own = half ? acc[64 + i] : acc[i], other = __uint_as_float(ld_shared<uint32_t>(from + i * 512));
                    const bool in = f0 + i < a.rows;
                    acc[i] = in ? gated(half ? other : own, half ? own : other) : 0.f;
                    m = max(m, magnitude(acc[i]));
                }
                asm volatile("st.shared.u32 [%0], %1;" ::"r"(top + half * 512), "r"(m) : "memory");
                readers_sync();  // every group's
                m = max(m, ld_shared<uint32_t>(top + (half ^ 1) * 512));
                const float s = scale_of(m);
                const Quotient by(s);
                if (by.lift != 1.f)
#pragma unroll
                    for (int i = 0; i < 64; ++i) acc[i] *= by.lift;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float* v = acc + 16 * j;
                    uint4 q;
                    q.x = by.e4m3(v[0], v[1], v[2], v[3]);
                    q.y = by.e4m3(v[4], v[5], v[6], v[7]);
                    q.z = by.e4m3(v[8], v[9], v[10], v[11]);
                    q.w = by.e4m3(v[12], v[13], v[14], v[15]);
                    st_shared(swizzled(out_at, row, half * 4 + j), q);
                }
                if (live && half == 0) a.out_scale[token * a.os_token + tn * a.os_block] = s;
                tc::fence_async();
                readers_sync();
                if (issues && half == 0) {
                    if (token0 < a.tokens) tc::tma_store_2d(&out_map, out_at, tn * kTile, (int)token0);
                    tc::store_commit();
                }
            } else if (a.dtype == ZKV_DT_F32) {
                // 32 features a tile, two tiles at a time
#pragma unroll
                for (int side = 0; side < 2; ++side) {
                    if (side && mapped && issues) tc::store_wait_read();
                    group_sync(half);
#pragma unroll
                    for (int c = 0; c < 2; ++c)
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            const float* v = acc + side * 64 + c * 32 + 4 * j;
                            st_shared(swizzled(staging + c * kTileBytes, row, j),
                                      make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]),
                                                 __float_as_uint(v[3])));
                        }
                    if (mapped) tc::fence_async();
                    group_sync(half);
                    for (int c = 0; c < 2; ++c) {
                        const int f = tn * C::kFeatures + half * kTile + side * 64 + c * 32;
                        if (!mapped || cut_short(a.rows, f, 32, 4)) copy_out<uint32_t>(a, staging + c * kTileBytes, token0, f, 32);
                        else if (issues && f < a.rows && token0 < a.tokens)
                            tc::tma_store_2d(&out_map, staging + c * kTileBytes, f, (int)token0);
                    }
                    if (mapped && issues) tc::store_commit();
                }
            } else {
                group_sync(half);
#pragma unroll
                for (int c = 0; c < 2; ++c)
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        uint32_t w[4];
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const float* v = acc + c * 64 + 8 * j + 2 * i;
                            if (a.dtype == ZKV_DT_BF16) {
                                w[i] = pack_bf162(v[0], v[1]);
                            } else {
                                const __half2 h = __floats2half2_rn(v[0], v[1]);
                                w[i] = *reinterpret_cast<const uint32_t*>(&h);
                            }
                        }
                        st_shared(swizzled(staging + c * kTileBytes, row, j), make_uint4(w[0], w[1], w[2], w[3]));
                    }
                if (mapped) tc::fence_async();
                group_sync(half);
                for (int c = 0; c < 2; ++c) {
                    const int f = tn * C::kFeatures + half * kTile + c * 64;
                    if (!mapped || cut_short(a.rows, f, 64, 2)) copy_out<uint16_t>(a, staging + c * kTileBytes, token0, f, 64);
                    else if (issues && f < a.rows && token0 < a.tokens)
                        tc::tma_store_2d(&out_map, staging + c * kTileBytes, f, (int)token0);
                }
                if (mapped && issues) tc::store_commit();
            }
        }
        if (mapped && issues) tc::store_wait();  // the staging is read until then
        tc::fence_before();
    }
    __syncthreads();
    tc::cluster_sync();  // neither CTA's memory is given up while the other may use it
    tc::fence_after();
    if (warp == 1) tc::tmem_free_pair(tmem, 512);
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

static cudaLaunchConfig_t configure(cudaLaunchAttribute (&attr)[2], unsigned x, unsigned y, int threads, int smem,
                                    unsigned cluster, cudaStream_t stream) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(x, y, 1);
    cfg.blockDim = dim3((unsigned)threads, 1, 1);
    cfg.dynamicSmemBytes = (size_t)smem;
    cfg.stream = stream;
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = cluster;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    return cfg;
}

// Clusters of s CTAs (s = 1..8) that the current device holds at once with one CTA an SM: a cluster lies within one of its
// groups of SMs, so that of three, five or seven CTAs many SMs stay empty.  Asked for one kernel that has an SM to itself
// and used for all products, so that how a product is cut depends neither on which ran first nor on whether the driver's
// count looks at what a kernel takes (580.159 counts one CTA an SM for those that share one, too; that two fit, Few asserts).
struct Places {
    int clusters[9];
};
static const Places* places() {
    using C = Few<128, 1>;
    static_assert(2 * (C::smem(C::kStages) + 1024) > 228 * 1024, "an SM to itself");
    static std::mutex mutex;
    static Places known[64] = {};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return nullptr;
    auto kernel = few_kernel<128, 1>;
    const std::lock_guard<std::mutex> lock(mutex);
    Places& p = known[dev];
    if (p.clusters[1]) return &p;
    if (!raise_smem_limit((const void*)kernel, C::smem(C::kStages))) return nullptr;
    for (int s = 8; s >= 1; --s) {
        cudaLaunchAttribute attr[2];
        cudaLaunchConfig_t cfg = configure(attr, 64 * s, 1, C::kThreads, C::smem(C::kStages), s, nullptr);
        if (cudaOccupancyMaxActiveClusters(&p.clusters[s], kernel, &cfg) != cudaSuccess) return nullptr;
    }
    return &p;
}

// How the inner dimension is cut over a cluster's CTAs: the number for which the waves of clusters take the fewest blocks
// after one another, each wave with a fixed cost of some blocks (filling the ring, joining the parts).  `halves`: two CTAs
// an SM, so that an even cluster lies on half as many SMs.  8 tokens, us by CTAs of a cluster: 4096 x 4096 1: 10.3, 2: 7.6, 4: 6.2, 8: 6.9; 6144 x 4096 11.0, 7.8, 6.9, 11.0;
// 4096 x 12288 26.7, 16.7, 13.1, 12.4; 151936 x 4096 97, 102, 124, 194.
struct Cut {
    int parts;
    int64_t cost;  // in blocks of the inner dimension
};
static Cut cut_of(int64_t tiles, int k_blocks, bool halves, const Places& p) {
    Cut best = {1, INT64_MAX};
    for (int s = 1; s <= 8 && s <= k_blocks; ++s) {
        const int64_t at_once = !halves ? p.clusters[s] : s % 2 ? 2 * p.clusters[s] : p.clusters[s / 2];
        if (at_once < 1) continue;
        const int64_t waves = (tiles + at_once - 1) / at_once, cost = waves * ((k_blocks + s - 1) / s + 4 + s);
        if (cost < best.cost) best = {s, cost};
    }
    return best;
}

constexpr int kMostWide = 65535;  // tiles of tokens that a grid's second dimension holds

template <int kTok, int kParts>
static int launch_few(const zkv_fp8_weight* w, const void* x, int64_t x_ld, const Product& a, cudaStream_t stream) {
    using C = Few<kTok, kParts>;
    CUtensorMap x_map;
    if (!encode_rows(&x_map, x, w->k, a.tokens, x_ld, 0, kTok)) return ZKV_ERR_ARG;
    const int64_t wide = (a.tokens + kTok - 1) / kTok;  // at most kMostWide, as launch() chooses
    auto kernel = few_kernel<kTok, kParts>;
    if (!raise_smem_limit((const void*)kernel, C::smem(C::kStages))) return launch_refused();
    const Places* p = places();
    if (!p) return launch_refused();
    const int parts = cut_of(a.row_blocks * wide, a.k_blocks, C::kHalves, *p).parts;
    cudaLaunchAttribute attr[2];
    const cudaLaunchConfig_t cfg = configure(attr, (unsigned)(a.row_blocks * parts), (unsigned)wide, C::kThreads,
                                             C::smem(C::kStages), (unsigned)parts, stream);
    CUtensorMap w_map;
    memcpy(&w_map, w->map, sizeof w_map);
    if (cudaLaunchKernelEx(&cfg, kernel, w_map, x_map, a) != cudaSuccess) return launch_refused();
    return launch_status();
}

// The output for stores of tiles, 128 bytes of 128 rows.
static bool encode_out(CUtensorMap* map, const Product& a, int element, int64_t columns) {
    EncodeTiled fn = encode_fn();
    if (!fn) return false;
    const cuuint64_t dims[2] = {(cuuint64_t)columns, (cuuint64_t)a.tokens}, strides[1] = {(cuuint64_t)(a.out_ld * element)};
    const cuuint32_t size[2] = {(cuuint32_t)(128 / element), 128}, es[2] = {1, 1};
    const CUtensorMapDataType type = element == 4   ? CU_TENSOR_MAP_DATA_TYPE_UINT32
                                     : element == 2 ? CU_TENSOR_MAP_DATA_TYPE_UINT16
                                                    : CU_TENSOR_MAP_DATA_TYPE_UINT8;
    return fn(map, type, 2, a.out, dims, strides, size, es, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
              CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <bool kGated>
static int launch_many(const zkv_fp8_weight* w, const void* x, int64_t x_ld, const Product& a, cudaStream_t stream) {
    using C = Many<kGated>;
    CUtensorMap maps[3];
    memcpy(&maps[0], w->map, sizeof maps[0]);
    if (!encode_rows(&maps[1], x, w->k, a.tokens, x_ld, 0, 128)) return ZKV_ERR_ARG;
    const int element = kGated ? 1 : a.dtype == ZKV_DT_F32 ? 4 : 2;
    const bool mapped = aligned16(a.out) && a.out_ld * element % 16 == 0 && a.out_ld * element < (int64_t)1 << 40;
    if (!mapped) maps[2] = maps[1];
    else if (!encode_out(&maps[2], a, element, a.rows)) return ZKV_ERR_ARG;
    const int64_t m = (a.tokens + C::kTokens - 1) / C::kTokens, n = kGated ? a.row_blocks : (a.row_blocks + 1) / 2;
    if (m * n > INT32_MAX / 2) return ZKV_ERR_CAPACITY;
    const int sms = sm_count();
    if (!sms) return launch_refused();
    auto kernel = many_kernel<kGated>;
    if (!raise_smem_limit((const void*)kernel, C::kSmem)) return launch_refused();
    const ManyTiles tiles = {(int)m, (int)n, (int)(m * n)};
    cudaLaunchAttribute attr[2];
    const cudaLaunchConfig_t cfg =
        configure(attr, (unsigned)std::min<int64_t>(2 * m * n, sms / 2 * 2), 1, C::kThreads, C::kSmem, 2, stream);
    if (cudaLaunchKernelEx(&cfg, kernel, maps[0], maps[1], maps[2], a, tiles, mapped) != cudaSuccess) return launch_refused();
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

// Up to 64 tokens features are the rows of a tile.  Above, CTAs of 128 tokens and one part's 128 features each (a cluster
// may share a tile), or pairs of CTAs of 256 tokens and 256 features: by the blocks that the waves of either take after one
// another.  A block takes the pair a little longer, and CTAs of two parts twice as long.  us of the first and of the second
// kind: 333 x 4096 x 4096 13.7 and 16.4, 768 x 4096 x 4096 31.2 and 18.1, 512 x 4096 x 12288 37.0 and 41.1, 129 x 2 x 12288
// x 4096 48.0 and 41.8, 1024 x 1024 x 4096 11.2 and 16.1.  More tokens than a grid of the first kind holds go to the pairs.
template <int kParts>
static int launch(const zkv_fp8_weight* w, const void* x, int64_t x_ld, const Product& a, cudaStream_t stream) {
    uint64_t any = 0;
    for (uint64_t word : w->map) any |= word;
    if (!any) return ZKV_ERR_ARG;  // zkv_fp8_weight_init was not called
    if (a.tokens <= 16) return launch_few<16, kParts>(w, x, x_ld, a, stream);
    if (a.tokens <= 32) return launch_few<32, kParts>(w, x, x_ld, a, stream);
    if (a.tokens <= 64) return launch_few<64, kParts>(w, x, x_ld, a, stream);
    if (a.tokens > (int64_t)kMostWide * 128) return launch_many<kParts == 2>(w, x, x_ld, a, stream);
    const Places* p = places();
    if (!p) return launch_refused();
    const int64_t few = kParts * cut_of(a.row_blocks * ((a.tokens + 127) / 128), a.k_blocks, false, *p).cost;
    const int64_t pairs = std::max(p->clusters[2], 1);
    const int64_t tiles = (a.tokens + 255) / 256 * (kParts == 2 ? a.row_blocks : (a.row_blocks + 1) / 2);
    const int64_t many = (tiles + pairs - 1) / pairs * a.k_blocks * 11 / 10 + 9;
    if (few <= many) return launch_few<128, kParts>(w, x, x_ld, a, stream);
    return launch_many<kParts == 2>(w, x, x_ld, a, stream);
}

}  // namespace fp8
}  // namespace zkv

using namespace zkv;

extern "C" int zkv_fp8_weight_init(zkv_fp8_weight* w) {
    if (const int rc = fp8::check_weight(w)) return rc;
    static_assert(sizeof(CUtensorMap) == sizeof w->map, "map");
    CUtensorMap map;
    if (!fp8::encode_rows(&map, w->w, w->k, w->rows, w->ld, w->parts, fp8::kBox)) return ZKV_ERR_ARG;
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
