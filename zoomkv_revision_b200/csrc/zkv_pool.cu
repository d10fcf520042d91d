// zkv_pool.cu -- the pooled KV cache around its attention: the plan of a step
// (block table, slot map, lengths), the write of new K/V rows into their
// slots, and the release of finished requests' blocks.
//
// Plan and release are a running sum over the requests followed by work per
// token (per block).  Both run as ONE cluster: every CTA makes the sums for
// itself (a few values per thread), the cluster meets once, and then its CTAs
// share the tokens, so the outputs may be the inputs' own buffers without a
// second launch or a counter in memory.  Release meets once more, to leave out
// ids that are not the pool's (a fifth of 32 requests 3.9 -> 5.0 us on the GPU).
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <algorithm>

#include "zkv_pool.cuh"

namespace zkv {
namespace pool {

constexpr int kMaxBatch = 8192;
constexpr int kMaxThreads = 1024;

// The last b in [0, n) with start[b] <= i (start ascending, start[0] <= i).
__device__ __forceinline__ int owner_of(const int32_t* start, int n, int i) {
    int b = 0;
    for (int step = n > 1 ? 1 << (31 - __clz(n - 1)) : 0; step > 0; step >>= 1) {
        const int at = b + step;
        if (at < n && start[at] <= i) b = at;
    }
    return b;
}

struct PlanArgs {
    const int32_t* lens;
    const int32_t* new_lens;
    int32_t* table;
    const int32_t* free_blocks;
    const int32_t* n_free;
    int64_t* slots;
    int32_t* positions;
    int32_t* cu_new;
    int32_t* lens_out;
    int32_t* n_free_out;
    int32_t* status;
    int64_t table_ld, n_blocks;
    int batch, shift, width, n_slots;
    bool vectors;  // slots and positions are 16-byte aligned
};

__global__ void __launch_bounds__(kMaxThreads) pool_plan_kernel(const __grid_constant__ PlanArgs a) {
    extern __shared__ int32_t sm[];
    __shared__ int64_t sh[32];
    __shared__ int s_used;
    int32_t* s_cu = sm;                    // [batch + 1] first token of a request
    int32_t* s_base = s_cu + a.batch + 1;  // [batch] blocks taken before it; -1: not served
    int32_t* s_len = s_base + a.batch;     // [batch]
    cg::cluster_group cluster = cg::this_cluster();
    const int rank = (int)cluster.block_rank(), ranks = (int)cluster.num_blocks();
    const int tid = threadIdx.x, nt = blockDim.x;
    const int S = 1 << a.shift;
    int code = 0;
    pdl_begin();
    int64_t n_free = *a.n_free;
    if (n_free < 0 || n_free > a.n_blocks) {
        code = ZKV_ERR_RANGE;
        n_free = n_free < 0 ? 0 : a.n_blocks;
    }
    if (tid == 0) s_used = 0;
    int64_t cu0 = 0, take0 = 0;
    for (int b0 = 0; b0 < a.batch; b0 += nt) {
        const int b = b0 + tid;
        const bool in = b < a.batch;
        const int len = in ? a.lens[b] : 0;
        const int add = in ? (a.new_lens ? a.new_lens[b] : 1) : 0;
        const int64_t n = add > 0 ? add : 0;
        int64_t total;
        const int64_t cu = cu0 + block_sum_before(n, sh, &total);
        cu0 += total;
        const int64_t have = ((int64_t)len + S - 1) >> a.shift, need = ((int64_t)len + n + S - 1) >> a.shift;
        const bool fits = in && len >= 0 && add >= 0 && need <= a.width && cu + n <= a.n_slots && len + n <= INT32_MAX;
        const int64_t take = fits ? need - have : 0;
        const int64_t base = take0 + block_sum_before(take, sh, &total);
        take0 += total;
        const bool served = fits && (take == 0 || base + take <= n_free);
        if (in) {
            s_cu[b] = (int)(cu < INT32_MAX ? cu : INT32_MAX);
            s_base[b] = served ? (int)base : -1;
            s_len[b] = len;
            // takers are served in order until one is not, so the blocks taken end with the last one served
            if (served && take > 0) atomicMax(&s_used, (int)(base + take));
            if (!served && code == 0) code = ZKV_ERR_CAPACITY;
        }
    }
    if (tid == 0) s_cu[a.batch] = (int)(cu0 < INT32_MAX ? cu0 : INT32_MAX);
    cluster.sync();  // every CTA has read lens and n_free: rank 0 may write over them
    if (rank == 0) {
        for (int b = tid; b < a.batch; b += nt) {
            const int len = s_len[b];
            a.lens_out[b] = s_base[b] >= 0 ? len + (s_cu[b + 1] - s_cu[b]) : len;
        }
        if (a.cu_new)
            for (int b = tid; b <= a.batch; b += nt) a.cu_new[b] = s_cu[b];
        if (tid == 0) *a.n_free_out = (int)n_free - s_used;
    }
    // Four tokens a turn: one search, the block ids' loads in flight together, 16-byte stores.
    const uint32_t total = (uint32_t)s_cu[a.batch], n_slots = (uint32_t)a.n_slots;
    for (uint32_t i0 = (uint32_t)(rank * nt + tid) * 4; i0 < n_slots; i0 += (uint32_t)(ranks * nt) * 4) {
        int id[4] = {-1, -1, -1, -1}, pos[4] = {-1, -1, -1, -1};
        if (i0 < total) {
            int b = owner_of(s_cu, a.batch, (int)i0);
            // a new block's id comes off the stack: the table's new entries are written, never read, here
            auto id_at = [&](int r, int base, int have, int j) {
                return j < have ? a.table[r * a.table_ld + j] : a.free_blocks[(int)n_free - 1 - base - (j - have)];
            };
            if (i0 + 3 < (uint32_t)s_cu[b + 1]) {  // one request, and so at most two blocks
                const int base = s_base[b];
                if (base >= 0) {
                    const int have = (int)(((uint32_t)s_len[b] + S - 1) >> a.shift);
                    const int p = s_len[b] + ((int)i0 - s_cu[b]), j0 = p >> a.shift, j1 = (p + 3) >> a.shift;
                    const int first = id_at(b, base, have, j0), second = id_at(b, base, have, j1);
                    // the thread of a block's first token enters it (that token is new, so the block is)
                    const int edge = -p & (S - 1);
                    if (edge < 4) a.table[b * a.table_ld + (edge ? j1 : j0)] = edge ? second : first;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        id[e] = (p + e) >> a.shift == j0 ? first : second;
                        pos[e] = p + e;
                    }
                }
            } else {
                int row[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    row[e] = -1;
                    if (i0 + e >= total) continue;
                    while ((int)i0 + e >= s_cu[b + 1]) ++b;
                    if (s_base[b] < 0) continue;
                    row[e] = b;
                    pos[e] = s_len[b] + ((int)i0 + e - s_cu[b]);
                }
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (row[e] >= 0)
                        id[e] = id_at(row[e], s_base[row[e]], (int)(((uint32_t)s_len[row[e]] + S - 1) >> a.shift),
                                      pos[e] >> a.shift);
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (row[e] >= 0 && (pos[e] & (S - 1)) == 0) a.table[row[e] * a.table_ld + (pos[e] >> a.shift)] = id[e];
            }
        }
        int64_t slot[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const bool ok = pos[e] >= 0 && (uint32_t)id[e] < (uint32_t)a.n_blocks;
            if (pos[e] >= 0 && !ok) code = ZKV_ERR_RANGE;
            slot[e] = ok ? ((int64_t)id[e] << a.shift) + (pos[e] & (S - 1)) : -1;
            pos[e] = ok ? pos[e] : -1;
        }
        if (a.vectors && i0 + 4 <= n_slots) {
            longlong2* d = reinterpret_cast<longlong2*>(a.slots + i0);
            d[0] = make_longlong2(slot[0], slot[1]);
            d[1] = make_longlong2(slot[2], slot[3]);
            if (a.positions) *reinterpret_cast<int4*>(a.positions + i0) = make_int4(pos[0], pos[1], pos[2], pos[3]);
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (i0 + e < n_slots) {
                    a.slots[i0 + e] = slot[e];
                    if (a.positions) a.positions[i0 + e] = pos[e];
                }
        }
    }
    if (code) raise_status(a.status, code);
}

struct ReleaseArgs {
    const uint8_t* done;
    const int32_t* lens;
    const int32_t* table;
    int32_t* free_blocks;
    const int32_t* n_free;
    int32_t* lens_out;
    int32_t* n_free_out;
    int32_t* status;
    int64_t table_ld, n_blocks;
    int batch, shift, width;
    bool vectors;  // free_blocks is 16-byte aligned
};

__global__ void __launch_bounds__(kMaxThreads) pool_release_kernel(const __grid_constant__ ReleaseArgs a) {
    extern __shared__ int32_t sm[];
    __shared__ int64_t sh[32];
    __shared__ int s_bad;              // rank 0's: ids outside the pool
    int32_t* s_start = sm;             // [batch] blocks pushed before a request
    int32_t* s_len = s_start + a.batch;  // [batch] its new length
    cg::cluster_group cluster = cg::this_cluster();
    const int rank = (int)cluster.block_rank(), ranks = (int)cluster.num_blocks();
    const int tid = threadIdx.x, nt = blockDim.x;
    const int S = 1 << a.shift;
    int code = 0;
    pdl_begin();
    int64_t n_free = *a.n_free;
    if (n_free < 0 || n_free > a.n_blocks) {
        code = ZKV_ERR_RANGE;
        n_free = n_free < 0 ? 0 : a.n_blocks;
    }
    if (tid == 0) s_bad = 0;
    int64_t start0 = 0;
    for (int b0 = 0; b0 < a.batch; b0 += nt) {
        const int b = b0 + tid;
        const bool in = b < a.batch;
        const int len = in ? a.lens[b] : 0;
        const bool done = in && a.done[b];
        int64_t count = done && len > 0 ? ((int64_t)len + S - 1) >> a.shift : 0;
        if (count > a.width || (done && len < 0)) {
            code = ZKV_ERR_RANGE;
            count = count > a.width ? a.width : count;
        }
        int64_t total;
        const int64_t start = start0 + block_sum_before(count, sh, &total);
        start0 += total;
        if (in) {
            s_start[b] = (int)(start < INT32_MAX ? start : INT32_MAX);
            s_len[b] = done ? 0 : len;
        }
    }
    const int64_t room = a.n_blocks - n_free;
    if (start0 > room) {
        code = code ? code : ZKV_ERR_CAPACITY;
        start0 = room;
    }
    cluster.sync();  // every CTA has read lens and n_free
    if (rank == 0)
        for (int b = tid; b < a.batch; b += nt) a.lens_out[b] = s_len[b];
    // Four places of the stack a turn, from a multiple of four on: one search, 16-byte stores.
    const int64_t end = n_free + start0;
    int bad = 0;
    for (int64_t w0 = (n_free & ~3) + ((int64_t)rank * nt + tid) * 4; w0 < end; w0 += (int64_t)ranks * nt * 4) {
        const int i0 = (int)(w0 - n_free);  // -3 .. : below 0 only in the first group
        int b = owner_of(s_start, a.batch, i0 > 0 ? i0 : 0);
        const int32_t* from[4];
        int id[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const bool in = i0 + e >= 0 && w0 + e < end;
            while (in && b + 1 < a.batch && i0 + e >= s_start[b + 1]) ++b;
            from[e] = in ? a.table + b * a.table_ld + (i0 + e - s_start[b]) : nullptr;
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) id[e] = from[e] ? *from[e] : 0;
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (from[e] && (uint32_t)id[e] >= (uint32_t)a.n_blocks) ++bad;
        if (a.vectors && from[0] && from[3]) {
            *reinterpret_cast<int4*>(a.free_blocks + w0) = make_int4(id[0], id[1], id[2], id[3]);
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (from[e]) a.free_blocks[w0 + e] = id[e];
        }
    }
    if (bad) {
        code = ZKV_ERR_RANGE;
        atomicAdd(cluster.map_shared_rank(&s_bad, 0), bad);
    }
    if (code) raise_status(a.status, code);
    cluster.sync();  // every id is on the stack and judged
    if (rank != 0) return;
    int64_t top = end;
    if (s_bad) {  // rare: the ids of the pool move up over the others, in order
        top = n_free;
        for (int64_t i0 = n_free; i0 < end; i0 += nt) {
            const int64_t i = i0 + tid;
            const int id = i < end ? __ldcg(a.free_blocks + i) : -1;
            const bool keep = (uint32_t)id < (uint32_t)a.n_blocks;
            int64_t total;
            const int64_t at = top + block_sum_before(keep, sh, &total);
            if (keep) a.free_blocks[at] = id;
            top += total;
        }
    }
    if (tid == 0) *a.n_free_out = (int)top;
}

// ---------------------------------------------------------------- write
struct WriteArgs {
    const uint8_t* src[2];
    uint8_t* dst[2];
    const float* scale[2];
    int64_t src_token[2], src_head[2];               // bytes
    int64_t dst_block[2], dst_token[2], dst_head[2];  // bytes
    const int64_t* slots;
    int32_t* status;
    int64_t pool_tokens, items;
    int heads, lg_parts, shift;
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

__device__ __forceinline__ uint32_t e4m3x4(float a, float b, float c, float d) {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
    return lo | (hi << 16);
}

// x / scale to e4m3 without a division in the common case: x times the
// reciprocal shrunk and grown by 2^-21 encloses the quotient and its fp32
// rounding (the products are off by 3 * 2^-24 at most), rounding is monotone,
// so where both ends give one code the quotient has that code; else (a
// quotient that close to the middle of two codes) it is divided.  The
// division in every element made 8191 tokens of 8 x 128 take 13.2 us
// (10.7 without, in L2).
struct Divisor {
    float scale, low, high;
    bool plain;  // the reciprocal is not a normal number: divide

    __device__ __forceinline__ explicit Divisor(float s) {
        const float r = 1.f / s;
        scale = s;
        low = r * (1.f - 4.76837158203125e-7f);
        high = r * (1.f + 4.76837158203125e-7f);
        plain = !(fabsf(s) > 1e-30f && fabsf(s) < 1e30f);
    }

    template <bool kBf16>
    __device__ __forceinline__ uint32_t e4m3(uint32_t w0, uint32_t w1) const {
        float a, b, c, d;
        to_floats<kBf16>(w0, a, b);
        to_floats<kBf16>(w1, c, d);
        const uint32_t x = e4m3x4(a * low, b * low, c * low, d * low);
        const uint32_t y = e4m3x4(a * high, b * high, c * high, d * high);
        if (x == y && !plain) return x;
        return e4m3x4(__fdiv_rn(a, scale), __fdiv_rn(b, scale), __fdiv_rn(c, scale), __fdiv_rn(d, scale));
    }
};

constexpr int kWriteThreads = 256;

// One 16-byte store per item (token, head, part of the row); K at blockIdx.y
// 0, V at 1.  kMode 0: 16-bit copy, two items a thread; 1: bf16 -> e4m3, one
// item (two loads); 2: fp16 -> e4m3.  32 source bytes a thread, all loads
// before the first store: with 128 the grid is one wave that reads, converts
// and writes in step (cold, 8191 tokens of 8 x 128 to e4m3 14.7 us, with 32
// 11.1 us, its bytes alone 7.7; 16384 tokens bf16 22.7 and 22.6, bytes 20.6).
template <int kMode>
__global__ void __launch_bounds__(kWriteThreads) pool_write_kernel(const __grid_constant__ WriteArgs a) {
    pdl_begin();
    constexpr int kWriteUnroll = kMode ? 1 : 2;
    const int y = blockIdx.y;
    constexpr int kLoads = kMode ? 2 : 1;
    const int64_t first = (int64_t)blockIdx.x * (kWriteThreads * kWriteUnroll) + threadIdx.x;
    const float* sc = a.scale[y];
    uint4 x[kWriteUnroll][kLoads];
    int64_t slot[kWriteUnroll];
    uint32_t head[kWriteUnroll];
#pragma unroll
    for (int u = 0; u < kWriteUnroll; ++u) {
        const int64_t it = first + u * kWriteThreads;
        slot[u] = -1;
        if (it >= a.items) continue;
        const uint32_t row = (uint32_t)(it >> a.lg_parts), part = (uint32_t)it & ((1u << a.lg_parts) - 1);
        const uint32_t tok = row / (uint32_t)a.heads;
        head[u] = row - tok * (uint32_t)a.heads;
        slot[u] = a.slots[tok];
        const uint4* p = reinterpret_cast<const uint4*>(a.src[y] + tok * a.src_token[y] + head[u] * a.src_head[y]) +
                         part * kLoads;
#pragma unroll
        for (int l = 0; l < kLoads; ++l) x[u][l] = p[l];
    }
    bool bad = false;
#pragma unroll
    for (int u = 0; u < kWriteUnroll; ++u) {
        const int64_t it = first + u * kWriteThreads;
        const int64_t s = slot[u];
        if (it >= a.items || s == -1) continue;
        if (s < 0 || s >= a.pool_tokens) {
            bad = true;
            continue;
        }
        const uint32_t part = (uint32_t)it & ((1u << a.lg_parts) - 1);
        uint8_t* d = a.dst[y] + (s >> a.shift) * a.dst_block[y] + (s & ((1 << a.shift) - 1)) * a.dst_token[y] +
                     head[u] * a.dst_head[y] + part * 16;
        uint4 out;
        if constexpr (kMode == 0) {
            out = x[u][0];
        } else {
            const Divisor by(sc ? __ldcg(sc + head[u]) : 1.f);
            out.x = by.e4m3<kMode == 1>(x[u][0].x, x[u][0].y);
            out.y = by.e4m3<kMode == 1>(x[u][0].z, x[u][0].w);
            out.z = by.e4m3<kMode == 1>(x[u][1].x, x[u][1].y);
            out.w = by.e4m3<kMode == 1>(x[u][1].z, x[u][1].w);
        }
        *reinterpret_cast<uint4*>(d) = out;
    }
    if (bad) raise_status(a.status, ZKV_ERR_RANGE);
}

// One cluster of CTAs for `work` tokens (or blocks) and `batch` requests.  A
// CTA alone up to 2048 of both (no cluster to gather: 256 x 1 tokens 6.0 us, in
// 8 CTAs 6.9), else 8 or, beyond 32768, the 16 that a GPC of this GPU holds.
static int launch_cluster(const void* fn, int batch, int64_t work, size_t smem, cudaStream_t st, void** args) {
    const int64_t want = std::max<int64_t>({batch, work, 1});
    const int ctas = want <= 2 * kMaxThreads ? 1 : want <= 32768 ? 8 : 16;
    const int threads = (int)std::min<int64_t>(kMaxThreads, (want + 31) / 32 * 32);
    if (ctas == 16 && cudaFuncSetAttribute(fn, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess)
        return launch_refused();
    return launch_clustered(fn, ctas, threads, ctas, smem, st, args, true);
}

}  // namespace pool
}  // namespace zkv

using namespace zkv;

extern "C" int zkv_pool_plan(const int32_t* lens, const int32_t* new_lens, int batch, int block_size,
                             int32_t* block_table, int64_t table_ld, int width, const int32_t* free_blocks,
                             const int32_t* n_free, int64_t n_blocks, int64_t* slots, int32_t* positions,
                             int64_t n_slots, int32_t* cu_new, int32_t* lens_out, int32_t* n_free_out,
                             int32_t* status, void* stream) {
    if (batch < 0 || n_slots < 0 || width < 0 || table_ld < width || n_blocks < 0) return ZKV_ERR_ARG;
    if (!pool::block_size_ok(block_size)) return ZKV_ERR_UNSUPPORTED;
    if (batch > pool::kMaxBatch || n_slots > INT32_MAX / 2 || n_blocks > INT32_MAX) return ZKV_ERR_CAPACITY;
    if ((batch > 0 && (!lens || !lens_out || (!block_table && width > 0))) || (!free_blocks && n_blocks > 0) ||
        !n_free || !n_free_out || (!slots && n_slots > 0))
        return ZKV_ERR_ARG;
    pool::PlanArgs a{lens, new_lens, block_table, free_blocks, n_free, slots, positions, cu_new, lens_out, n_free_out,
                     status, table_ld, n_blocks, batch, pool::log2_of(block_size), width, (int)n_slots,
                     pool::aligned16(slots) && pool::aligned16(positions)};
    void* args[] = {&a};
    return pool::launch_cluster((const void*)pool::pool_plan_kernel, batch, n_slots,
                                (size_t)(3 * batch + 1) * sizeof(int32_t), (cudaStream_t)stream, args);
}

extern "C" int zkv_pool_release(const uint8_t* done, const int32_t* lens, int batch, int block_size,
                                const int32_t* block_table, int64_t table_ld, int width, int32_t* free_blocks,
                                const int32_t* n_free, int64_t n_blocks, int32_t* lens_out, int32_t* n_free_out,
                                int32_t* status, void* stream) {
    if (batch < 0 || width < 0 || table_ld < width || n_blocks < 0) return ZKV_ERR_ARG;
    if (!pool::block_size_ok(block_size)) return ZKV_ERR_UNSUPPORTED;
    if (batch > pool::kMaxBatch || n_blocks > INT32_MAX) return ZKV_ERR_CAPACITY;
    if ((batch > 0 && (!done || !lens || !lens_out || (!block_table && width > 0))) ||
        (!free_blocks && n_blocks > 0) || !n_free || !n_free_out)
        return ZKV_ERR_ARG;
    pool::ReleaseArgs a{done, lens, block_table, free_blocks, n_free, lens_out, n_free_out, status, table_ld, n_blocks,
                        batch, pool::log2_of(block_size), width, pool::aligned16(free_blocks)};
    void* args[] = {&a};
    return pool::launch_cluster((const void*)pool::pool_release_kernel, batch,
                                std::min<int64_t>((int64_t)batch * width, n_blocks),
                                (size_t)(2 * batch) * sizeof(int32_t), (cudaStream_t)stream, args);
}

extern "C" int zkv_pool_write(const void* k, int64_t k_token, int64_t k_head, const void* v, int64_t v_token,
                              int64_t v_head, int dtype, const int64_t* slots, int64_t n_tokens, const zkv_pool* p,
                              int32_t* status, void* stream) {
    const int rc = pool::check_pool(p);
    if (rc != ZKV_OK) return rc;
    if (n_tokens < 0 || (dtype != ZKV_DT_BF16 && dtype != ZKV_DT_F16)) return ZKV_ERR_ARG;
    if (p->dtype != ZKV_DT_F8E4M3 && p->dtype != dtype) return ZKV_ERR_ARG;
    if (n_tokens == 0) return ZKV_OK;
    if (!k || !v || !slots) return ZKV_ERR_ARG;
    if (!pool::aligned16(k) || !pool::aligned16(v) || k_token % 8 || k_head % 8 || v_token % 8 || v_head % 8)
        return ZKV_ERR_ALIGN;
    if (n_tokens > INT32_MAX / p->kv_heads) return ZKV_ERR_CAPACITY;
    const int el = pool::element_bytes(p->dtype);
    const int lg = pool::log2_of(p->head_dim * el / 16);
    pool::WriteArgs a;
    a.src[0] = (const uint8_t*)k, a.src[1] = (const uint8_t*)v;
    a.dst[0] = (uint8_t*)p->k, a.dst[1] = (uint8_t*)p->v;
    a.scale[0] = p->k_scale, a.scale[1] = p->v_scale;
    a.src_token[0] = k_token * 2, a.src_token[1] = v_token * 2;
    a.src_head[0] = k_head * 2, a.src_head[1] = v_head * 2;
    a.dst_block[0] = p->k_block * el, a.dst_block[1] = p->v_block * el;
    a.dst_token[0] = p->k_token * el, a.dst_token[1] = p->v_token * el;
    a.dst_head[0] = p->k_head * el, a.dst_head[1] = p->v_head * el;
    a.slots = slots, a.status = status;
    a.pool_tokens = p->n_blocks * p->block_size;
    a.items = (n_tokens * p->kv_heads) << lg;
    a.heads = p->kv_heads, a.lg_parts = lg, a.shift = pool::log2_of(p->block_size);
    const int64_t per = pool::kWriteThreads * (el == 2 ? 2 : 1);
    const dim3 grid((unsigned)((a.items + per - 1) / per), 2);
    const auto kernel = el == 2                 ? pool::pool_write_kernel<0>
                        : dtype == ZKV_DT_BF16 ? pool::pool_write_kernel<1>
                                               : pool::pool_write_kernel<2>;
    return launch_pdl_kernel(kernel, grid, dim3(pool::kWriteThreads), 0, (cudaStream_t)stream, a);
}
