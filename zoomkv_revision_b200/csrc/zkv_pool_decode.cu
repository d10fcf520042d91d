// zkv_pool_decode.cu -- attention of one new token per request over a pooled
// KV cache.
//
//   o = sum_t p_t v_t / sum_t p_t,  p_t = exp(cap(scale q . k_t) - max)
//
// Every K and V byte is used for 2 G products of one grouped head (G = 4: 4
// operations a byte), so the bytes bound it.  The kernel is built to keep
// reads in flight on every SM until the last tile:
//
//  * The work is the list of all (request, kv head, tile of tokens) units, in
//    that order, cut into equal ranges, one per CTA of a one-wave grid.  Each
//    CTA finds its range from the lengths by itself (a sum over the requests),
//    so uneven requests, one long request and many short ones are spread the
//    same way and the host needs no length.  A row (request, kv head) that
//    ends in another CTA than it began in leaves partials (m, l, o), which
//    pool_join_kernel joins in CTA order.  Where the host's guess of the
//    longest request leaves little to balance (see plan_call) the rows are not cut by
//    units: a CTA takes whole rows, or a cluster of CTAs shares one row and
//    joins through distributed shared memory; one launch does, with no scan
//    and no workspace.
//  * Where there are many short rows (or windows) a warp takes a row alone and
//    loads it itself (pool_rows_kernel): nothing to join, nothing to wait for.
//  * One producer warp per CTA walks the range: block ids from the table, one
//    5-D TMA copy per block and tensor (dims | tokens | 128-byte pieces | head
//    | block; any strides, so both memory orders), a ring of stages.  An id
//    outside the pool is not copied.
//  * Four consumer warps share a tile's tokens: S^T = K Q^T (tokens x heads)
//    and O^T += V^T P^T (dims x heads) by mma.sync m16n8k16, so a group of up
//    to 8 heads fills the 8 columns of one product, 16 heads two.  More heads
//    are cut into chunks, whose CTAs walk the same range side by side, so that
//    K and V come from HBM once and from L2 again.  Up to 8 heads the bytes
//    bound the kernel with the tensor pipe active 15-19 % of the time, so
//    tcgen05 (tokens as M, heads as N, the probabilities through shared
//    memory) has nothing to win there; for many heads it was not tried.
//  * A tile is 16 KiB of K (32 for 512-byte rows): what bounds a warp is the
//    latency of its chain product - maximum - exponential - product, so rows of
//    128 bytes get 32 tokens a warp and chain instead of 16, rows of 64 get 64
//    (e4m3, 128 dims, 32 requests of 8192: 131 us with 16 tokens a chain).
//  * A warp keeps its own running max, sum and O^T in registers through the
//    row; the four are joined in the last tile's stage.
//
// Roundings: scores, statistics and accumulators are fp32.  The probability
// enters the second product as two 16-bit parts (p = hi + lo, 16 bits of
// mantissa for bf16), so that it adds little to the output's own rounding of 8
// or 11 bits; over e4m3 blocks with bf16 output one fp16 part (11 bits) does.
// Where those parts are fp16, p is 2^15 exp(x - max), at most half of what
// fp16 holds: full 11 bits down to 2^-29 of the largest and something down to
// 2^-40, where exp(x - max) itself would be gone at 2^-25 (17.3 below the
// largest score, which a first token that draws all attention reaches).
// e4m3 blocks are widened to fp16, exactly; a bf16 query is scaled by the
// power of two that puts its largest element into [2^15, 2^16) first, which
// leaves it exact in fp16 but for elements below 2^-32 of the largest.
#include <cuda.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <cstring>
#include <mutex>

#include "zkv_pool.cuh"

namespace zkv {
namespace pool {

constexpr int kConsumers = 4;                   // warps that share a tile's tokens
constexpr int kThreads = 32 * (kConsumers + 1);
constexpr int kMaxGrid = 480;                   // CTAs that a workspace is sized for
constexpr int kWholeTokens = 256;               // requests up to this length are never cut
constexpr int kMaxChunks = 320;                 // of 16 query heads per kv head
constexpr int64_t kMaxLen = INT32_MAX - 512;    // tokens of a request; 32 bits hold a tile past them
constexpr int kMaxStages = 8;                   // of a CTA's ring
constexpr int kMaxRanks = 16;                   // CTAs of a cluster that shares a row
// Up to kWholeBytes of K and V, and kRankTiles tiles a CTA or twice that where the CTAs fill their waves to 4/5, whole
// rows in one launch are ahead of ranges and a join, which 4 us more issue (8 kv heads of 128, bf16, us on the GPU, whole
// and ranges: 1 request of 4096 9.8 and 10.0, 1 of 16384 21.0 and 19.4, 16 of 1000 12.9 and 18.0, 64 of 480 25.2 and 30.7,
// 32 of 1000 24.5 and 30.9, 40 of 800 34.3 and 31.0, 16 up to 1900 19.3 and 17.7, 64 up to 1000 36.0 and 33.4).
constexpr int64_t kWholeBytes = 128 << 20;
constexpr int kRankTiles = 8;
// A warp a row (pool_rows_kernel) or the CTA's four warps a row: alone where one product's tokens are all, where a row
// is one load and every CTA has one, or where a CTA has two rows or more of up to kRowLoads loads (e4m3, whose chain is
// the longer one, kRowLoadsF8), four of which are in flight (three with 8 heads).  256 requests, 8 kv heads of 128, bf16,
// us with four warps and with one: 1 token 9.1 and 7.3, 100 26.6 and 25.6, 256 (6 loads) 45.5 and 46.9; e4m3 64 13.5 and
// 12.8, 0..256 30.4 and 27.7, all 256 29.7 and 31.6; a window of 100 31.5 and 25.9; 64 requests of 40 7.0 and 5.7, up to
// 200 12.3 and 14.5; 16 query heads, blocks of 128 (two in flight), 191 requests of 108..217 64.7 and 78.0.
constexpr int kRowLoads = 5, kRowLoadsF8 = 8;
constexpr uint64_t kWaitNs = 2000000000ull;     // limit of each wait inside a CTA

// What a unit is, written by the producer beside its stage.
struct alignas(16) Unit {
    int b, h;         // request, kv head
    int tile0;        // first token
    int lo, len;      // tokens [lo, len) of the request are attended
    int flags;        // kFirst, kLast of the row in this CTA; kEnd: the CTA's last unit
    int part;         // kAlone: the row is this CTA's alone; 0, 1: its partial slot; kShared: a cluster's
    int bad;          // boxes of the tile that are not in the pool
};
constexpr int kFirst = 1, kLast = 2, kEnd = 4;
constexpr int kAlone = -1, kShared = 2;

// Tokens of a tile, for a row of `bytes` bytes.
__host__ __device__ constexpr int tile_tokens(int bytes) { return bytes >= 256 ? 64 : 64 * 256 / bytes; }

struct DecodeArgs {
    CUtensorMap tk, tv;  // [block][head][128-byte piece][token][bytes]
    const uint8_t* q;
    const float* k_scale;
    const float* v_scale;
    const int32_t* lens;
    const int32_t* table;
    void* out;
    float* lse;
    int32_t* status;
    float* parts;   // [grid][2][heads][D] o of a row's part: slot 0 began in an earlier CTA, slot 1 goes on in later ones
    float* stats;   // [grid][2][heads][2] its m, l
    int64_t q_row, q_head;  // bytes
    int64_t table_ld, n_blocks;
    int cap;        // the longest length that the table holds
    int batch, kv_heads, G, chunks, heads;  // heads: query heads of a chunk (the last one may have fewer)
    int abreast;    // kv heads of a row: their CTAs walk one range side by side
    int head_rows;  // rows of a request: kv_heads / abreast
    int side;       // CTAs of a range: abreast * chunks; CTA x: member x % side of range x / side
    int groups;     // ranges
    int whole;      // rows are not cut by units
    int ranks;      // CTAs (a cluster) that share a row, if `whole`
    int unit, workers, ahead;   // a warp a row: tokens of a stage, warps of a CTA, stages of a warp
    int shift, lg_box, width, window;
    float scale, softcap;
};

template <int kQ, bool kF8, int D, int NT>
struct Cfg {
    static constexpr int kEl = kF8 ? 1 : 2;
    static constexpr int kRow = D * kEl;                         // bytes of a token's row
    static constexpr int kInner = kRow < 128 ? kRow : 128;       // swizzled span
    static constexpr int kPieces = kRow / kInner;
    static constexpr int kTile = tile_tokens(kRow);              // tokens of a unit
    static constexpr int kSub = kTile / (16 * kConsumers);       // 16-token products of a warp in a tile
    static constexpr int kKv = kTile * kRow;                     // K (or V) of a stage
    static constexpr int kHeadsMax = 8 * NT;
    static constexpr int kQPitch = D * 2 + 16;
    static constexpr int kQSlot = kHeadsMax * kQPitch;  // a multiple of 16
    static constexpr int kFixed = 1024;                          // alignment of the swizzled boxes
    static constexpr int kStage = 2 * kKv + kQSlot + (int)sizeof(Unit);
    static constexpr int kMl = 2 * kConsumers * kHeadsMax * 8;
    static constexpr int kOther = 1024 + 448;                    // an SM's reserve for a CTA; its static variables
    static constexpr int stages_of(int ctas) { return (233472 / ctas - kOther - kFixed - kMl) / kStage; }
    // Two n-tiles of heads read the query from shared memory for each product: its registers are worth another CTA on
    // the SM (16 heads, 32 requests of 8192, 4 kv heads: e4m3 of 128 dims 74.4 -> 61.4 us, of 256 164 -> 144, bf16 of 128
    // 98.5 -> 96.3).  512-byte rows have no room for a second CTA, one n-tile has registers to spare.
    static constexpr bool kQShared = NT == 2 && kRow <= 256;
    // CTAs of an SM: two where they keep three stages each, or three of two stages each.  64-byte rows of one n-tile take
    // three (32 requests of 8192, 8 kv heads: 67.3 us with two, 54.4 with three); 128-byte rows gain nothing by it (95.0
    // and 91.8, uneven ones 174 and 177).
    static constexpr int kPerSm = (kRow <= 64 && NT == 1) || (kQShared && D <= 128) ? 3
                                  : kQShared || stages_of(2) >= 3                    ? 2
                                                                                     : 1;
    static constexpr int kRowWarps = kPerSm == 1 ? 8 : kConsumers;  // of a CTA whose warps take rows alone
    // As many stages as fit, but two for 256-byte rows of one n-tile: their warps keep up, and more reads in flight only
    // slow the memory down (8 requests of 32768 165.2 us with three, 159.4 with two; 128-byte rows 162.8 and 173).
    static constexpr int kFit = stages_of(kPerSm);
    static constexpr int kStages = kRow == 256 && !kF8 && NT == 1 ? 2 : kFit < kMaxStages ? kFit : kMaxStages;
    static constexpr int kRing = 233472 / kPerSm - kOther - kFixed - kMl;  // bytes of a ring at most
    static constexpr int smem_of(int ring) { return ring + kFixed + kMl; }
    // The probability as hi + lo, or hi alone over e4m3 blocks with bf16 output: 11 bits under a result of 8, whose error
    // against 64 bits stays the same to three digits.  32 requests of 8192, one part and two: 8 kv heads of 128 with 4 heads
    // each 92.9 and 93.9 us, 4 of 128 with 16 60.1 and 68.2, 4 of 256 with 16 142 and 151.
    static constexpr bool kTwoParts = !(kF8 && kQ == ZKV_DT_BF16);
    static constexpr int kMTiles = D / 16;
    // n-tiles of O that fit into a stage's K and V when the warps are joined
    static constexpr int kJoinTiles = (2 * kKv) / (kConsumers * 8 * D * 4) < NT ? (2 * kKv) / (kConsumers * 8 * D * 4) : NT;
    static_assert(kJoinTiles >= 1 && NT % kJoinTiles == 0, "join buffer");
    static_assert(kStages >= 2, "a ring");
    static_assert(kHeadsMax * D * 4 <= kStages * kQSlot, "a cluster's part takes the queries' place");
};

// ------------------------------------------------------------ device helpers
__device__ __forceinline__ bool mbar_try(uint64_t* bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity)
        : "memory");
    return ok != 0;
}

// Wait for a phase, at most kWaitNs; false and ZKV_ERR_TIMEOUT on expiry.
__device__ __forceinline__ bool wait_for(uint64_t* bar, uint32_t parity, int32_t* status) {
    if (mbar_try(bar, parity)) return true;
    const uint64_t t0 = globaltimer_ns();
    while (!mbar_try(bar, parity)) {
        if (globaltimer_ns() - t0 > kWaitNs) {
            raise_status(status, ZKV_ERR_TIMEOUT);
            return false;
        }
    }
    return true;
}

__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}

// K and V rows are read once a call: they leave L2 before what the call uses again (one request of 131071 85.0 -> 83.7 us,
// 12 query heads a kv head 111.6 -> 106.9).
__device__ __forceinline__ uint64_t evict_first_policy() {
    uint64_t policy;
    asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(policy));
    return policy;
}

__device__ __forceinline__ void tma_load_5d(uint32_t dst, const CUtensorMap* map, int token, int head, int block,
                                            uint64_t* bar, uint64_t policy) {
    asm volatile(
        "cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.L2::cache_hint [%0], "
        "[%1, {%2, %3, %4, %5, %6}], [%7], %8;" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(0), "r"(token), "r"(0), "r"(head), "r"(block), "r"(smem_u32(bar)),
        "l"(policy)
        : "memory");
}

__device__ __forceinline__ void proxy_fence() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ uint32_t transposed(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ uint32_t e4m3x2_to_f16x2(uint16_t x) {
    uint32_t y;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(y) : "h"(x));
    return y;
}
__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// tanh to 2^-20 of itself: with t = exp(-2|u|), (1 - t) / (1 + t), where t's error of 2^-22 of itself leaves 2^-23; below
// 1/4, where 1 - t cancels, Taylor's polynomial, whose next term is 2^-26.  tanhf of an exact quotient in every score
// made 219 requests of 2917 e4m3 tokens, 1 kv head of 128, take 58.2 us (34.0 without a soft cap).
__device__ __forceinline__ float tanh_fast(float u) {
    const float w = fabsf(u), s = u * u, t = exp2_fast(-2.8853900817779268f * w);
    const float p = -1.f / 3 + s * (2.f / 15 + s * (-17.f / 315 + s * (62.f / 2835)));
    return w < 0.25f ? u + u * (s * p) : copysignf(__fdividef(1.f - t, 1.f + t), u);
}

// D(16x8 f32) += A(16x16, row) * B(16x8, col), both bf16 or both fp16
template <bool kBf16>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (kBf16) {
        mma_bf16_16816(d, a[0], a[1], a[2], a[3], b0, b1);
    } else {
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 "
            "{%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    }
}

template <bool kBf16>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    if constexpr (kBf16) return pack_bf162(lo, hi);
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
template <bool kBf16>
__device__ __forceinline__ float2 unpack2(uint32_t w) {
    if constexpr (kBf16) return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
    return __half22float2(*reinterpret_cast<const __half2*>(&w));
}

__device__ __forceinline__ int request_len(const DecodeArgs& a, int n) {
    return n < 0 ? 0 : (n > a.cap ? a.cap : n);
}
__device__ __forceinline__ int first_token(const DecodeArgs& a, int len) {
    return a.window > 0 && len > a.window ? len - a.window : 0;
}
// Tiles of a row; a row without tokens has one, which writes its zeros.
template <int kTile>
__device__ __forceinline__ int row_tiles(const DecodeArgs& a, int len) {
    const int t = (len + kTile - 1) / kTile - first_token(a, len) / kTile;
    return t > 0 ? t : 1;
}

// The list of units, seen by a block of kN threads: each thread holds the
// requests [b_lo, b_hi), whose units are [before, before + mine).
struct Units {
    int b_lo, b_hi;
    int len;  // of request b_lo
    int64_t before, mine, total;
};
template <int kTile, int kN>
__device__ __forceinline__ Units count_units(const DecodeArgs& a, int64_t* sh) {
    Units u;
    const int per = (a.batch + kN - 1) / kN;
    u.b_lo = min(a.batch, (int)threadIdx.x * per);
    u.b_hi = min(a.batch, u.b_lo + per);
    u.mine = 0;
    u.len = 0;
    if (u.b_lo < u.b_hi) {
        u.len = __ldcg(a.lens + u.b_lo);
        u.mine = (int64_t)row_tiles<kTile>(a, request_len(a, u.len)) * a.head_rows;
    }
    for (int b = u.b_lo + 1; b < u.b_hi; ++b)
        u.mine += (int64_t)row_tiles<kTile>(a, request_len(a, __ldcg(a.lens + b))) * a.head_rows;
    u.before = block_sum_before(u.mine, sh, &u.total);
    return u;
}
// The request of unit `u`, the unit's number in it and the request's length, by the one thread that holds it.
template <int kTile>
__device__ __forceinline__ bool locate(const DecodeArgs& a, const Units& x, int64_t u, int& b, int64_t& off, int& len) {
    if (u < x.before || u >= x.before + x.mine) return false;
    off = u - x.before;
    len = x.len;
    for (b = x.b_lo;;) {
        const int64_t n = (int64_t)row_tiles<kTile>(a, request_len(a, len)) * a.head_rows;
        if (off < n || b + 1 >= x.b_hi) return true;
        off -= n;
        len = __ldcg(a.lens + ++b);
    }
}

__device__ __forceinline__ int64_t quotient(int64_t x, int64_t y) {  // x >= 0, y > 0; in 32 bits where they allow it
    return (uint64_t)(x | y) >> 32 ? x / y : (int64_t)((uint32_t)x / (uint32_t)y);
}

// The list cut into equal ranges, the first `longer` of them one unit longer.
struct Ranges {
    int64_t count, size, longer;

    __device__ __forceinline__ Ranges(const DecodeArgs& a, int64_t total) {
        count = min((int64_t)a.groups, total);
        size = quotient(total, count);
        longer = total - size * count;
    }
    __device__ __forceinline__ int64_t begin(int64_t c) const { return c * size + min(c, longer); }
    __device__ __forceinline__ int64_t owner(int64_t u) const {
        const int64_t split = longer * (size + 1);
        return u < split ? quotient(u, size + 1) : longer + quotient(u - split, size);
    }
};

// A place in a ring and the parity that its barrier completes next.
struct Turn {
    int stage = 0;
    uint32_t phase = 0;

    __device__ __forceinline__ void next(int stages) {
        if (++stage == stages) {
            stage = 0;
            phase ^= 1;
        }
    }
    __device__ __forceinline__ void skip(int stages, int n) {  // n <= stages
        stage += n;
        if (stage >= stages) {
            stage -= stages;
            phase ^= 1;
        }
    }
};

// ------------------------------------------------------------ consumers
template <int kQ, bool kF8, int D, int NT>
struct Row {
    using C = Cfg<kQ, kF8, D, NT>;
    static constexpr bool kMmaBf16 = kQ == ZKV_DT_BF16 && !kF8;
    // Exponentials are kLift of themselves, o and a lane's l too; the warp's total and what it puts are not.  By a product:
    // 15 taken off the maximum rounds to 16 or 0 where scores pass 2^24, and 2^16 is infinite in fp16.
    static constexpr float kLift = kMmaBf16 ? 1.f : 32768.f, kDown = 1.f / kLift;
    float m[NT][2], l[NT][2];   // log2 units; heads 2t, 2t+1 of n-tile (t = lane % 4); l: this lane's tokens
    float f[NT][2];             // score factor of those heads, log2 units (under a soft cap, natural ones of it)
    float o[C::kMTiles][NT][4];
    uint32_t q_at;              // the queries' place, this lane's part
    uint32_t q[C::kQShared ? 1 : D / 16][NT][2];  // B fragments of Q^T, where they are not read from there each time

    // A bf16 query to fp16, for e4m3 rows: scaled by the power of two that puts its largest element into [2^15, 2^16)
    // (65280 at most), so that the small ones keep their bits; up: the way back.  Both factors are normal numbers.
    static __device__ __forceinline__ float down_scale(float largest, float& up) {
        int e = (int)(__float_as_uint(largest) >> 23) - 127 - 15;  // in [2^(e+15), 2^(e+16))
        e = largest > 0.f ? (e < -126 ? -126 : (e > 113 ? 113 : e)) : 0;
        up = __uint_as_float((uint32_t)(127 + e) << 23);
        return __uint_as_float((uint32_t)(127 - e) << 23);
    }

    // The same in the queries' place in shared memory: four heads at a time, eight lanes a head; `up` behind the head's row.
    static __device__ __forceinline__ void narrow_shared(uint8_t* qs, int quarter) {
        const int lane = threadIdx.x & 31;
        uint8_t* row = qs + (4 * quarter + (lane >> 3)) * C::kQPitch;
        uint4* at = reinterpret_cast<uint4*>(row) + (lane & 7);
        uint4 w[D / 64];
        float largest = 0.f;
#pragma unroll
        for (int i = 0; i < D / 64; ++i) {
            w[i] = at[8 * i];
            const uint32_t* x = reinterpret_cast<const uint32_t*>(&w[i]);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float2 y = unpack2<true>(x[k]);
                largest = fmaxf(largest, fmaxf(fabsf(y.x), fabsf(y.y)));
            }
        }
#pragma unroll
        for (int off = 4; off >= 1; off >>= 1) largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, off));
        float up;
        const float down = down_scale(largest, up);
#pragma unroll
        for (int i = 0; i < D / 64; ++i) {
            uint32_t* x = reinterpret_cast<uint32_t*>(&w[i]);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float2 y = unpack2<true>(x[k]);
                x[k] = pack2<false>(y.x * down, y.y * down);
            }
            at[8 * i] = w[i];
        }
        if ((lane & 7) == 0) *reinterpret_cast<float*>(row + 2 * D) = up;
    }

    __device__ __forceinline__ void init(const DecodeArgs& a, const uint8_t* qs, int n_heads, float k_scale) {
        const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
        const float base = a.scale * k_scale * (a.softcap > 0.f ? 1.f : 1.4426950408889634f);
        q_at = smem_u32(qs) + g * C::kQPitch + (kF8 ? 8 : 4) * t;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            m[n][0] = m[n][1] = -INFINITY;
            l[n][0] = l[n][1] = 0.f;
            f[n][0] = f[n][1] = base;
            if constexpr (C::kQShared) {
                if constexpr (kF8 && kQ == ZKV_DT_BF16)
#pragma unroll
                    for (int e = 0; e < 2; ++e)
                        f[n][e] *= *reinterpret_cast<const float*>(qs + (8 * n + 2 * t + e) * C::kQPitch + 2 * D);
                continue;
            }
            const bool in = 8 * n + g < n_heads;
            float largest = 0.f;
#pragma unroll
            for (int s = 0; s < D / 16; ++s) {
                query_at(n, s, q[s][n]);
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    if (!in) q[s][n][i] = 0u;
                    const float2 y = unpack2<true>(q[s][n][i]);
                    if (kF8 && kQ == ZKV_DT_BF16) largest = fmaxf(largest, fmaxf(fabsf(y.x), fabsf(y.y)));
                }
            }
            if constexpr (kF8 && kQ == ZKV_DT_BF16) {
                largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, 1));
                largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, 2));
                float up;
                const float down = down_scale(largest, up);
#pragma unroll
                for (int s = 0; s < D / 16; ++s)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const float2 y = unpack2<true>(q[s][n][i]);
                        q[s][n][i] = pack2<false>(y.x * down, y.y * down);
                    }
                f[n][0] *= __shfl_sync(0xffffffffu, up, 8 * t);
                f[n][1] *= __shfl_sync(0xffffffffu, up, 8 * t + 4);
            }
        }
        if (a.softcap > 0.f)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 2; ++e)  // finite, so that a score of 0 stays one
                    f[n][e] = fminf(fmaxf(f[n][e] / a.softcap, -3.4e38f), 3.4e38f);
#pragma unroll
        for (int j = 0; j < C::kMTiles; ++j)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[j][n][e] = 0.f;
    }

    // The B fragment of Q^T for 16 dims of n-tile n.  Over e4m3 rows k index 2t, 2t+1, 2t+8, 2t+9 stands for dims
    // 4t .. 4t+3, as those rows are read.
    __device__ __forceinline__ void query_at(int n, int s, uint32_t (&b)[2]) const {
        const uint32_t at = q_at + n * 8 * C::kQPitch + 32 * s;
        if constexpr (kF8) {
            asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(b[0]), "=r"(b[1]) : "r"(at) : "memory");
        } else {
            asm volatile("ld.shared.b32 %0, [%1];" : "=r"(b[0]) : "r"(at) : "memory");
            asm volatile("ld.shared.b32 %0, [%1];" : "=r"(b[1]) : "r"(at + 16) : "memory");
        }
    }

    // The warp's tokens of a tile, 16 a product: product i's K and V rows begin
    // at base + at[i] and base + half + at[i] (in a swizzled box, `piece` bytes
    // from one 128-byte piece to the next); its tokens [v0[i], v1[i]) count.
    __device__ __forceinline__ void step(const DecodeArgs& a, uint32_t base, uint32_t half, const uint32_t (&at)[C::kSub], uint32_t piece,
                                         const int (&v0)[C::kSub], const int (&v1)[C::kSub], bool partial) {
        const int lane = threadIdx.x & 31, g = lane >> 2;
        constexpr int kPerPiece = C::kInner / 16;  // 16-byte chunks of a row in a piece
        constexpr int kSub = C::kSub;
        // address of chunk c of this lane's row: the swizzle permutes the chunks of a row by the row's number
        const int tok_k = lane & 15, off_k = lane >> 4;
        const int sw_k = C::kInner == 128 ? tok_k & 7 : (tok_k >> 1) & 3;
        auto chunk = [&](uint32_t from, int tok, int sw, int c) {
            return from + (uint32_t)(c / kPerPiece) * piece + tok * C::kInner + (((c % kPerPiece) ^ sw) << 4);
        };
        // two chains of products at least, so that one does not wait for the other
        constexpr bool kSplit = kSub == 1 || !C::kQShared;
        float x[kSub][NT][4], x2[kSplit ? kSub : 1][NT][4];
#pragma unroll
        for (int i = 0; i < kSub; ++i)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    x[i][n][e] = 0.f;
                    if constexpr (kSplit) x2[i][n][e] = 0.f;
                }
#pragma unroll
        for (int s = 0; s < D / 16; s += 2) {
            uint32_t qf[2][NT][2];
#pragma unroll
            for (int k = 0; k < 2; ++k)
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    if constexpr (C::kQShared) {
                        query_at(n, s + k, qf[k][n]);
                    } else {
                        qf[k][n][0] = q[s + k][n][0];
                        qf[k][n][1] = q[s + k][n][1];
                    }
                }
#pragma unroll
            for (int i = 0; i < kSub; ++i) {
                uint32_t a0[4], a1[4];
                if constexpr (kF8) {
                    uint32_t r[4];
                    ldsm4(chunk(base + at[i], tok_k, sw_k, s + off_k), r);
                    a0[0] = e4m3x2_to_f16x2((uint16_t)r[0]), a0[1] = e4m3x2_to_f16x2((uint16_t)r[1]);
                    a0[2] = e4m3x2_to_f16x2((uint16_t)(r[0] >> 16)), a0[3] = e4m3x2_to_f16x2((uint16_t)(r[1] >> 16));
                    a1[0] = e4m3x2_to_f16x2((uint16_t)r[2]), a1[1] = e4m3x2_to_f16x2((uint16_t)r[3]);
                    a1[2] = e4m3x2_to_f16x2((uint16_t)(r[2] >> 16)), a1[3] = e4m3x2_to_f16x2((uint16_t)(r[3] >> 16));
                } else {
                    ldsm4(chunk(base + at[i], tok_k, sw_k, 2 * s + off_k), a0);
                    ldsm4(chunk(base + at[i], tok_k, sw_k, 2 * s + 2 + off_k), a1);
                }
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    mma16816<kMmaBf16>(x[i][n], a0, qf[0][n][0], qf[0][n][1]);
                    if constexpr (kSplit) mma16816<kMmaBf16>(x2[i][n], a1, qf[1][n][0], qf[1][n][1]);
                    else mma16816<kMmaBf16>(x[i][n], a1, qf[1][n][0], qf[1][n][1]);
                }
            }
        }
        if constexpr (kSplit) {
#pragma unroll
            for (int i = 0; i < kSub; ++i)
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) x[i][n][e] += x2[i][n][e];
        }
        // x[i][n][0..3]: (token g, head 2t), (g, 2t+1), (g+8, 2t), (g+8, 2t+1)
        float alpha[NT][2];
        bool moved = false;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
            for (int i = 0; i < kSub; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float y = x[i][n][e] * f[n][e & 1];
                    if (a.softcap > 0.f) y = a.softcap * 1.4426950408889634f * tanh_fast(y);
                    x[i][n][e] = y;
                }
            if (partial) {
#pragma unroll
                for (int i = 0; i < kSub; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int tok = e < 2 ? g : g + 8;
                        if (tok < v0[i] || tok >= v1[i]) x[i][n][e] = -INFINITY;
                    }
            }
#pragma unroll
            for (int i = 0; i < kSub; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) mx[e & 1] = fmaxf(mx[e & 1], x[i][n][e]);
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                mx[c] = fmaxf(mx[c], __shfl_xor_sync(0xffffffffu, mx[c], 4));
                mx[c] = fmaxf(mx[c], __shfl_xor_sync(0xffffffffu, mx[c], 8));
                mx[c] = fmaxf(mx[c], __shfl_xor_sync(0xffffffffu, mx[c], 16));
                mx[c] = fmaxf(mx[c], m[n][c]);
                const float ref = mx[c] == -INFINITY ? 0.f : mx[c];  // nothing seen yet: no inf - inf
                alpha[n][c] = exp2_fast(m[n][c] - ref);
                moved |= mx[c] != m[n][c];
                m[n][c] = mx[c];
                float sum = 0.f;
#pragma unroll
                for (int i = 0; i < kSub; ++i) {
                    x[i][n][c] = kLift * exp2_fast(x[i][n][c] - ref);
                    x[i][n][c + 2] = kLift * exp2_fast(x[i][n][c + 2] - ref);
                    sum += x[i][n][c] + x[i][n][c + 2];
                }
                l[n][c] = l[n][c] * alpha[n][c] + sum;
            }
        }
        if (__any_sync(0xffffffffu, moved)) {  // most tiles of a long row leave the maxima as they are
#pragma unroll
            for (int j = 0; j < C::kMTiles; ++j)
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[j][n][e] *= alpha[n][e & 1];
        }
#pragma unroll
        for (int i = 0; i < kSub; ++i) {
            uint32_t hi[NT][2], lo[NT][2];
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    const float p0 = x[i][n][2 * r], p1 = x[i][n][2 * r + 1];
                    const uint32_t w = pack2<kMmaBf16>(p0, p1);
                    hi[n][r] = transposed(w);
                    if constexpr (C::kTwoParts) {
                        const float2 back = unpack2<kMmaBf16>(w);
                        lo[n][r] = transposed(pack2<kMmaBf16>(p0 - back.x, p1 - back.y));
                    }
                }
            const uint32_t vs = base + half + at[i];
            // four tiles of dims at a time, their hi products before their lo ones, so that none waits for the one before
            const int tok_v = (lane & 7) + ((lane >> 4) << 3), off_v = (lane >> 3) & 1, sw_v = tok_v & 7;
#pragma unroll
            for (int j = 0; j < C::kMTiles; j += 4) {
                uint32_t v[4][4];
                if constexpr (kF8) {
#pragma unroll
                    for (int k = 0; k < 4; k += 2) {
                        uint32_t r[4];
                        ldsm4_t(chunk(vs, tok_k, sw_k, j + k + off_k), r);
#pragma unroll
                        for (int w = 0; w < 4; ++w) {
                            const uint32_t y = __byte_perm(r[w], 0, 0x3120);  // (dim 2g: tokens 2t, 2t+1), (dim 2g+1)
                            v[k + w / 2][2 * (w & 1)] = e4m3x2_to_f16x2((uint16_t)y);
                            v[k + w / 2][2 * (w & 1) + 1] = e4m3x2_to_f16x2((uint16_t)(y >> 16));
                        }
                    }
                } else {
#pragma unroll
                    for (int k = 0; k < 4; ++k) ldsm4_t(chunk(vs, tok_v, sw_v, 2 * (j + k) + off_v), v[k]);
                }
#pragma unroll
                for (int k = 0; k < 4; ++k)
#pragma unroll
                    for (int n = 0; n < NT; ++n) mma16816<kMmaBf16>(o[j + k][n], v[k], hi[n][0], hi[n][1]);
                if constexpr (C::kTwoParts) {
#pragma unroll
                    for (int k = 0; k < 4; ++k)
#pragma unroll
                        for (int n = 0; n < NT; ++n) mma16816<kMmaBf16>(o[j + k][n], v[k], lo[n][0], lo[n][1]);
                }
            }
        }
    }

    // The sum of a head's exponentials over the warp's tokens.
    __device__ __forceinline__ float total(int n, int e) const {
        float s = l[n][e];
        s += __shfl_xor_sync(0xffffffffu, s, 4);
        s += __shfl_xor_sync(0xffffffffu, s, 8);
        s += __shfl_xor_sync(0xffffffffu, s, 16);
        return s * kDown;
    }

    // O of n-tile n times a factor per head to `to` [8][D].  Dims of a head are permuted by its pair's number, so that the
    // 32 lanes meet 32 banks.
    __device__ __forceinline__ void put(float* to, int n, const float (&factor)[2]) const {
        const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
        const float fac[2] = {factor[0] * kDown, factor[1] * kDown};
        float* p = to + 2 * t * D;
#pragma unroll
        for (int j = 0; j < C::kMTiles; ++j) {
            const float* x = o[j][n];
            if constexpr (kF8) {
                const int d = (16 * j + 2 * g) ^ (t << 3);
                *reinterpret_cast<float2*>(p + d) = make_float2(x[0] * fac[0], x[2] * fac[0]);
                *reinterpret_cast<float2*>(p + D + d) = make_float2(x[1] * fac[1], x[3] * fac[1]);
            } else {
                const int d = (16 * j + g) ^ (t << 3), d8 = (16 * j + g + 8) ^ (t << 3);
                p[d] = x[0] * fac[0];
                p[D + d] = x[1] * fac[1];
                p[d8] = x[2] * fac[0];
                p[D + d8] = x[3] * fac[1];
            }
        }
    }

    // V rows of tokens outside [v0, v1) to zero: their probability is 0, but 0 times what an unwritten row may hold
    // (NaN, infinities) is not.
    __device__ __forceinline__ void clear_rows(uint8_t* vs, uint32_t piece, int v0, int v1) {
        constexpr int kPer = C::kRow / 16;
        for (int i = threadIdx.x & 31; i < 16 * kPer; i += 32) {
            const int tok = i / kPer, c = i % kPer;
            if (tok < v0 || tok >= v1)
                *reinterpret_cast<uint4*>(vs + (c / (C::kInner / 16)) * piece + tok * C::kInner +
                                          (c % (C::kInner / 16)) * 16) = make_uint4(0, 0, 0, 0);
        }
        __syncwarp();
    }

    // Part `part` of a unit: 16 tokens a product, kSub products.
    __device__ __forceinline__ void tokens(const DecodeArgs& a, const Unit& x, uint8_t* base, int half, int part) {
        // 16 tokens lie in one box (a box has 16 or more)
        uint32_t from[C::kSub];
        int v0[C::kSub], v1[C::kSub];
        bool any = false, partial = false;
#pragma unroll
        for (int k = 0; k < C::kSub; ++k) {
            const int in_tile = 16 * (C::kSub * part + k), box = in_tile >> a.lg_box;
            from[k] = (uint32_t)((box << a.lg_box) * C::kRow + (in_tile - (box << a.lg_box)) * C::kInner);
            v0[k] = max(x.lo - x.tile0 - in_tile, 0);
            v1[k] = (x.bad >> box) & 1 ? 0 : min(x.len - x.tile0 - in_tile, 16);
            any |= v0[k] < v1[k];
            partial |= v0[k] > 0 || v1[k] < 16;
        }
        if (!any) return;
        const uint32_t piece = (uint32_t)C::kInner << a.lg_box;
        if (partial) {
#pragma unroll
            for (int k = 0; k < C::kSub; ++k) clear_rows(base + half + from[k], piece, v0[k], v1[k]);
        }
        step(a, smem_u32(base), half, from, piece, v0, v1, partial);
        if (partial) proxy_fence();
    }
};

template <int kQ>
__device__ __forceinline__ void store4(void* out, int64_t i, float4 x) {
    constexpr bool kBf16 = kQ == ZKV_DT_BF16;
    *reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(out) + i) =
        make_uint2(pack2<kBf16>(x.x, x.y), pack2<kBf16>(x.z, x.w));
}

template <int kQ, bool kF8, int D, int NT>
__global__ void __launch_bounds__(kThreads, Cfg<kQ, kF8, D, NT>::kPerSm)
    pool_decode_kernel(const __grid_constant__ DecodeArgs a) {
    using C = Cfg<kQ, kF8, D, NT>;
    constexpr int stages = C::kStages, half = C::kKv;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = smem_raw + (((smem_u32(smem_raw) + 1023u) & ~1023u) - smem_u32(smem_raw));
    uint8_t* kv = smem;                                                  // [stages] K, V
    uint8_t* qs = kv + stages * 2 * half;                            // [stages] query heads, by row
    Unit* units = reinterpret_cast<Unit*>(qs + stages * C::kQSlot);    // [stages]
    float2* ml = reinterpret_cast<float2*>(units + stages);            // [2][warps][heads]
    __shared__ uint64_t full[kMaxStages], empty[kMaxStages], epi;
    __shared__ int64_t sh[32];
    __shared__ int64_t s_off;
    __shared__ int s_b, s_len;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (tid == 0) {
        for (int i = 0; i < stages; ++i) {
            mbar_init(full + i, 1);
            mbar_init(empty + i, kConsumers);
        }
        mbar_init(&epi, kConsumers);
        mbar_fence_init();
        asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&a.tk)) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&a.tv)) : "memory");
    }
    const int rank = blockIdx.x % a.ranks, block = blockIdx.x / a.ranks;
    const int member = block % a.side, chunk = member % a.chunks, abreast = member / a.chunks;
    const int64_t c = block / a.side;
    const int n_heads = min(a.heads, a.G - chunk * a.heads);
    if constexpr (C::kQShared) {  // the places of heads that the chunk has not: products of zeros
        const int per = (C::kHeadsMax - n_heads) * (D / 8);
        for (int i = tid; i < stages * per; i += kThreads)
            *reinterpret_cast<uint4*>(qs + i / per * C::kQSlot + (n_heads + i % per / (D / 8)) * C::kQPitch +
                                      i % (D / 8) * 16) = make_uint4(0, 0, 0, 0);
    }
    // the arguments' constant-cache lines, while the previous grid ends
    asm volatile("" ::"l"(a.q), "l"(a.lens), "l"(a.parts), "l"(a.q_head), "r"(a.batch), "r"(a.groups), "f"(a.softcap));
    grid_dep_wait();
    grid_dep_launch_next();  // the join kernel may become resident; it waits for this grid
    // ---- this CTA's range [u0, u1): of units, or of rows where those are not split
    int64_t u0, u1;
    if (a.whole) {
        const int64_t rows = (int64_t)a.batch * a.head_rows;
        u0 = quotient(rows * c, a.groups);
        u1 = quotient(rows * (c + 1), a.groups);
        __syncthreads();
        if (u0 == u1) return;
    } else {
        const Units x = count_units<C::kTile, kThreads>(a, sh);
        const Ranges cuts(a, x.total);
        if (c >= cuts.count) return;
        u0 = cuts.begin(c);
        u1 = cuts.begin(c + 1);
        int b, len;
        int64_t off;
        if (locate<C::kTile>(a, x, u0, b, off, len)) {
            s_b = b;
            s_len = len;
            s_off = off;
        }
        __syncthreads();
    }

    if (warp == kConsumers) {
        // ---------------------------------------------------- producer
        int b = a.whole ? (int)quotient(u0, a.head_rows) : s_b;
        int next = a.whole ? __ldcg(a.lens + b) : s_len;  // the next request's length, asked for one request ahead
        int len, lo, tile_first, tiles;
        auto begin_request = [&]() {
            if (next < 0 || next > a.cap) raise_status(a.status, ZKV_ERR_RANGE);
            len = request_len(a, next);
            lo = first_token(a, len);
            tile_first = lo / C::kTile;
            tiles = row_tiles<C::kTile>(a, len);
            if (b + 1 < a.batch) next = __ldcg(a.lens + b + 1);
        };
        // a row that begins at token 0 needs the table's first entries: asked for beside its length
        int ids = -1, ids_next = -1, ids_b = -1, ids_at = 0;
        if (a.whole && a.ranks == 1 && a.window == 0) {
            const int32_t* row = a.table + b * a.table_ld;
            ids = lane < a.width ? __ldcg(row + lane) : -1;
            ids_next = 32 + lane < a.width ? __ldcg(row + 32 + lane) : -1;
            ids_b = b;
        }
        begin_request();
        int hr, tile;  // row of the request, tile of the row
        if (a.whole) {
            hr = (int)(u0 - (int64_t)b * a.head_rows);
            tile = (int)((uint32_t)tiles * (uint32_t)rank / (uint32_t)a.ranks);
        } else {
            hr = (int)quotient(s_off, tiles);
            tile = (int)(s_off - (int64_t)hr * tiles);
        }
        bool none = false;  // more CTAs than tiles: this one has an empty unit
        if (a.ranks > 1) {
            tiles = (int)((uint32_t)tiles * (uint32_t)(rank + 1) / (uint32_t)a.ranks);
            none = tile == tiles;
            if (none) tiles = tile + 1;
        }
        int64_t row_begin = a.whole ? u0 : u0 - tile;  // unit at which the row begins (its number, where rows are whole)
        Turn at, q_at;  // of the stages; of the queries' places, a row's the next
        q_at.stage = stages - 1;
        const uint64_t policy = evict_first_policy();
        const int boxes = C::kTile >> a.lg_box, box_bytes = C::kRow << a.lg_box;
        bool ok = true, end = false;
        int done = 0;
        for (; !end; ++done) {
            const int stage = at.stage, h = hr * a.abreast + abreast;
            const bool first = done == 0 || tile == 0;
            end = a.whole ? tile == tiles - 1 && row_begin + 1 == u1 : u0 + done + 1 == u1;
            const bool last = end || tile == tiles - 1;
            int part = kAlone;
            if (!a.whole) part = row_begin < u0 ? 0 : row_begin + tiles > u1 ? 1 : kAlone;
            else if (a.ranks > 1) part = kShared;
            // ---- block ids of the tile: 32 entries of the table at a time, the next 32 on their way
            const int tile0 = (tile_first + tile) * C::kTile;
            const int entry = tile0 >> a.shift;
            if (ids_b != b || ids_at != (entry & ~31)) {
                const int32_t* row = a.table + b * a.table_ld;
                const int n_entries = (len + (1 << a.shift) - 1) >> a.shift;
                const int at = entry & ~31;
                if (ids_b == b && at == ids_at + 32) ids = ids_next;
                else ids = at + lane < n_entries ? __ldcg(row + at + lane) : -1;
                ids_next = at + 32 + lane < n_entries ? __ldcg(row + at + 32 + lane) : -1;
                ids_b = b;
                ids_at = at;
            }
            const int id = __shfl_sync(0xffffffffu, ids, (entry - ids_at + lane) & 31);  // lane j: box j
            const int tok = tile0 + (lane << a.lg_box);
            const bool wanted = lane < boxes && tok < len && tok + (1 << a.lg_box) > lo && !none;
            const bool there = wanted && id >= 0 && id < a.n_blocks;
            if (wanted && !there) raise_status(a.status, ZKV_ERR_RANGE);
            const unsigned copy = __ballot_sync(0xffffffffu, there), bad = __ballot_sync(0xffffffffu, wanted && !there);
            if (first) q_at.next(stages);
            if (done >= stages) ok = wait_for(empty + stage, at.phase ^ 1, a.status);
            if (!__all_sync(0xffffffffu, ok)) break;
            if (lane == 0) {
                Unit& x = units[stage];
                x.b = b;
                x.h = h;
                x.tile0 = tile0;
                x.lo = lo;
                x.len = none ? 0 : len;
                x.flags = (first ? kFirst : 0) | (last ? kLast : 0) | (end ? kEnd : 0);
                x.part = part;
                x.bad = (int)bad;
                mbar_arrive_expect_tx(full + stage, (uint32_t)(__popc(copy) * 2 * box_bytes + (first ? n_heads * D * 2 : 0)));
            }
            __syncwarp();
            if (there) {
                const uint32_t dst = smem_u32(kv + stage * 2 * half) + lane * box_bytes;
                // a box is a whole block, or a tile's tokens of one
                const int in_block = a.shift > a.lg_box ? tile0 & ((1 << a.shift) - 1) : 0;
                tma_load_5d(dst, &a.tk, in_block, h, id, full + stage, policy);
                tma_load_5d(dst + half, &a.tv, in_block, h, id, full + stage, policy);
            }
            if (first && lane >= 32 - C::kHeadsMax && lane - (32 - C::kHeadsMax) < n_heads) {
                const int j = lane - (32 - C::kHeadsMax);
                bulk_g2s(qs + q_at.stage * C::kQSlot + j * C::kQPitch,
                         a.q + b * a.q_row + (int64_t)(h * a.G + chunk * a.heads + j) * a.q_head, D * 2, full + stage);
            }
            // ---- next unit
            at.next(stages);
            if (++tile == tiles) {
                tile = 0;
                row_begin += a.whole ? 1 : tiles;
                if (++hr == a.head_rows) {
                    hr = 0;
                    if (++b < a.batch) begin_request();
                }
            }
        }
        // a consumer may have given up: the copies on their way land in this CTA's memory, so it does not end before them
        for (int i = max(0, done - stages); i < done; ++i)
            wait_for(full + i % stages, (uint32_t)((i / stages) & 1), a.status);
        return;
    }

    // -------------------------------------------------------- consumers
    Row<kQ, kF8, D, NT> row;
    uint32_t epi_phase = 0;
    int n_row = 0;
    const int g = lane >> 2, t = lane & 3;
    // a cluster's part of a row: this CTA's only one, so the queries and the first half of ml are free when it is done
    float* const cl_o = reinterpret_cast<float*>(qs);  // [heads][D]
    float2* const cl_ml = ml;                          // [heads]
    auto meet = [&]() -> bool {  // the four warps, at most kWaitNs
        __syncwarp();
        if (lane == 0) mbar_arrive(&epi);
        const bool got = __all_sync(0xffffffffu, wait_for(&epi, epi_phase, a.status));
        epi_phase ^= 1;
        return got;
    };
    bool alive = true;
    Turn at, q_at;
    q_at.stage = stages - 1;
    for (bool end = false; !end; at.next(stages)) {
        const int stage = at.stage;
        if (!__all_sync(0xffffffffu, wait_for(full + stage, at.phase, a.status))) {
            alive = false;
            break;
        }
        const Unit x = units[stage];
        end = (x.flags & kEnd) != 0;
        uint8_t* const base = kv + stage * 2 * half;
        if (x.flags & kFirst) {
            q_at.next(stages);
            uint8_t* const q_row = qs + q_at.stage * C::kQSlot;
            if constexpr (C::kQShared && kF8 && kQ == ZKV_DT_BF16) {
                row.narrow_shared(q_row, warp);
                __syncwarp();
                alive = meet();
                if (!alive) break;
            }
            row.init(a, q_row, n_heads, kF8 && a.k_scale ? a.k_scale[x.h] : 1.f);
            ++n_row;
        }
        row.tokens(a, x, base, half, warp);
        if (!(x.flags & kLast)) {
            __syncwarp();
            if (lane == 0) mbar_arrive(empty + stage);
            continue;
        }
        float* buf = reinterpret_cast<float*>(base);
        const float v_scale = kF8 && a.v_scale ? a.v_scale[x.h] : 1.f;
        const int64_t head0 = ((int64_t)x.b * a.kv_heads + x.h) * a.G + chunk * a.heads;
        // ---- the row's end: join the warps in the stage's K and V
        float2* mine_ml = ml + (n_row & 1) * kConsumers * C::kHeadsMax;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const float s = row.total(n, e);
                if (g == 0) mine_ml[warp * C::kHeadsMax + 8 * n + 2 * t + e] = make_float2(row.m[n][e], s);
            }
        if (!meet()) {  // statistics written, stage read by all
            alive = false;
            break;
        }
        const int64_t slot = (int64_t)blockIdx.x * 2 + x.part;
#pragma unroll
        for (int r = 0; r < NT; r += C::kJoinTiles) {
            if (r > 0 && alive) alive = meet();
#pragma unroll
            for (int n = 0; n < C::kJoinTiles; ++n) {
                float fac[2];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float mx = -INFINITY;
#pragma unroll
                    for (int w = 0; w < kConsumers; ++w)
                        mx = fmaxf(mx, mine_ml[w * C::kHeadsMax + 8 * (r + n) + 2 * t + e].x);
                    fac[e] = exp2_fast(row.m[r + n][e] - (mx == -INFINITY ? 0.f : mx));
                }
                row.put(buf + (warp * 8 * C::kJoinTiles + 8 * n) * D, r + n, fac);
            }
            if (alive) alive = meet();
            if (!alive) continue;
            for (int idx = tid; idx < 8 * C::kJoinTiles * (D / 4); idx += 32 * kConsumers) {
                const int hl = idx / (D / 4), d = 4 * (idx % (D / 4)), head = 8 * r + hl;
                if (head >= n_heads) continue;
                float mx = -INFINITY, sum = 0.f;
#pragma unroll
                for (int w = 0; w < kConsumers; ++w) mx = fmaxf(mx, mine_ml[w * C::kHeadsMax + head].x);
                const float ref = mx == -INFINITY ? 0.f : mx;
                float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                for (int w = 0; w < kConsumers; ++w) {
                    const float2 s = mine_ml[w * C::kHeadsMax + head];
                    sum += s.y * exp2_fast(s.x - ref);
                    const float4 y = *reinterpret_cast<const float4*>(buf + (w * 8 * C::kJoinTiles + hl) * D +
                                                                      (d ^ (((hl >> 1) & 3) << 3)));
                    o.x += y.x, o.y += y.y, o.z += y.z, o.w += y.w;
                }
                if (x.part == kAlone) {
                    const float inv = sum == 0.f ? 0.f : v_scale / sum;
                    store4<kQ>(a.out, (head0 + head) * D + d, make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv));
                    if (a.lse && d == 0) a.lse[head0 + head] = (mx + log2f(sum)) * 0.6931471805599453f;
                } else if (x.part == kShared) {
                    *reinterpret_cast<float4*>(cl_o + head * D + d) = o;
                    if (d == 0) cl_ml[head] = make_float2(mx, sum);
                } else {
                    *reinterpret_cast<float4*>(a.parts + (slot * C::kHeadsMax + head) * D + d) = o;
                    if (d == 0) *reinterpret_cast<float2*>(a.stats + (slot * C::kHeadsMax + head) * 2) = make_float2(mx, sum);
                }
            }
        }
        if (!alive) break;
        proxy_fence();  // the stage was written by these threads; the next copy into it is the async proxy's
        __syncwarp();
        if (lane == 0) mbar_arrive(empty + stage);
    }
    if (a.ranks == 1) return;
    // ---- the row's parts, by the cluster's ranks in order; every CTA meets here whatever became of its waits
    cg::cluster_group cluster = cg::this_cluster();
    cluster.sync();
    const int h = (int)(c % a.head_rows);
    const int64_t head0 = c * a.G + chunk * a.heads;  // (request, kv head) is the row's number: one head abreast
    for (int idx = tid * a.ranks + rank; alive && idx < n_heads * (D / 4); idx += 32 * kConsumers * a.ranks) {
        const int head = idx / (D / 4), d = 4 * (idx % (D / 4));
        float m = -INFINITY, l = 0.f;
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int r0 = 0; r0 < a.ranks; r0 += 8) {
            float2 s[8];
            float4 y[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                s[k] = make_float2(-INFINITY, 0.f);
                y[k] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (r0 + k < a.ranks) {
                    s[k] = *cluster.map_shared_rank(cl_ml + head, r0 + k);
                    y[k] = *cluster.map_shared_rank(reinterpret_cast<float4*>(cl_o + head * D + d), r0 + k);
                }
            }
            float mx = m;
#pragma unroll
            for (int k = 0; k < 8; ++k) mx = fmaxf(mx, s[k].x);
            const float ref = mx == -INFINITY ? 0.f : mx, old = exp2_fast(m - ref);
            l *= old, o.x *= old, o.y *= old, o.z *= old, o.w *= old;
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const float w = exp2_fast(s[k].x - ref);
                l += w * s[k].y;
                o.x += w * y[k].x, o.y += w * y[k].y, o.z += w * y[k].z, o.w += w * y[k].w;
            }
            m = mx;
        }
        const float v_scale = kF8 && a.v_scale ? __ldcg(a.v_scale + h) : 1.f;
        const float inv = l == 0.f ? 0.f : v_scale / l;
        store4<kQ>(a.out, (head0 + head) * D + d, make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv));
        if (a.lse && d == 0) a.lse[head0 + head] = (m + log2f(l)) * 0.6931471805599453f;
    }
    cluster.sync();  // no CTA leaves while another reads its part
}

// ------------------------------------------------------------ a warp a row
// Short rows, many of them: a warp takes whole rows alone and loads them itself,
// `unit` tokens at a time into its own stages, so no warp waits for another and
// no row is joined.  Where four warps share a row, their chain and join take
// 1.9 us a row whatever it holds.  The reads in flight are the CTA's warps', a
// load each; its stages' owner never changes, so a parity always tells its
// phases apart.  256 requests, four warps a row and one: 1 token, 8 kv heads of
// 128, bf16 17.1 -> 7.3 us, the last 8 of 17 tokens 18.3 -> 10.4, 17 tokens' last
// 8 with 16 query heads of 256 76.4 -> 30.3, 100 e4m3 tokens with 12 of 256
// 68.4 -> 41.8; 191 requests of 108..217, 16 kv heads of 256, 116 -> 98.
template <int kQ, bool kF8, int D, int NT>
__global__ void __launch_bounds__(32 * Cfg<kQ, kF8, D, NT>::kRowWarps, Cfg<kQ, kF8, D, NT>::kPerSm)
    pool_rows_kernel(const __grid_constant__ DecodeArgs a) {
    using C = Cfg<kQ, kF8, D, NT>;
    extern __shared__ uint8_t smem_raw[];
    const int stages = a.workers * a.ahead, half = a.unit * C::kRow;
    uint8_t* kv = smem_raw + (((smem_u32(smem_raw) + 1023u) & ~1023u) - smem_u32(smem_raw));  // [stages] K, V
    uint8_t* qs = kv + stages * 2 * half;                              // [stages] query heads, by row
    Unit* units = reinterpret_cast<Unit*>(qs + stages * C::kQSlot);    // [stages]
    __shared__ uint64_t full[kMaxStages];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    if (tid == 0) {
        for (int i = 0; i < stages; ++i) mbar_init(full + i, 1);
        mbar_fence_init();
        asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&a.tk)) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&a.tv)) : "memory");
    }
    const int chunk = blockIdx.x % a.side, c = blockIdx.x / a.side;
    const int n_heads = min(a.heads, a.G - chunk * a.heads);
    if constexpr (C::kQShared) {  // the places of heads that the chunk has not: products of zeros
        const int per = (C::kHeadsMax - n_heads) * (D / 8);
        for (int i = tid; i < stages * per; i += 32 * C::kRowWarps)
            *reinterpret_cast<uint4*>(qs + i / per * C::kQSlot + (n_heads + i % per / (D / 8)) * C::kQPitch +
                                      i % (D / 8) * 16) = make_uint4(0, 0, 0, 0);
    }
    grid_dep_wait();
    grid_dep_launch_next();
    __syncthreads();
    const int64_t rows = (int64_t)a.batch * a.kv_heads, stride = (int64_t)a.workers * a.groups;
    int64_t r = (int64_t)warp * a.groups + c;  // a CTA's rows are far apart, of requests of different lengths
    if (warp >= a.workers || r >= rows) return;
    kv += warp * a.ahead * 2 * half;
    qs += warp * a.ahead * C::kQSlot;
    units += warp * a.ahead;
    uint64_t* const bars = full + warp * a.ahead;

    // ---- the next unit to load: its row, first token, block ids (lane j: box j) and the length of the row after
    const int box = 1 << a.lg_box, grain = max(box, 16 * C::kSub);
    const uint64_t policy = evict_first_policy();
    int b = (int)quotient(r, a.kv_heads), h = 0, len = 0, lo = 0, tok = 0, id = -1, next = __ldcg(a.lens + b);
    bool first = true;
    auto enter = [&]() {
        b = (int)quotient(r, a.kv_heads);
        h = (int)(r - (int64_t)b * a.kv_heads);
        if (next < 0 || next > a.cap) raise_status(a.status, ZKV_ERR_RANGE);
        len = request_len(a, next);
        lo = first_token(a, len);
        tok = lo & ~(grain - 1);
        first = true;
        if (r + stride < rows) next = __ldcg(a.lens + quotient(r + stride, a.kv_heads));
    };
    auto wanted = [&]() {
        const int off = lane << a.lg_box;
        return off < a.unit && off < len - tok && off + box > lo - tok;
    };
    auto ask = [&]() { id = wanted() ? __ldcg(a.table + b * a.table_ld + (tok >> a.shift) + lane) : -1; };
    int issued = 0;
    Turn put_at, put_q;
    put_q.stage = a.ahead - 1;
    auto issue = [&]() {
        const int stage = put_at.stage;
        const bool want = wanted(), there = want && id >= 0 && id < a.n_blocks;
        if (want && !there) raise_status(a.status, ZKV_ERR_RANGE);
        const unsigned copy = __ballot_sync(0xffffffffu, there), bad = __ballot_sync(0xffffffffu, want && !there);
        const bool last = tok + a.unit >= len;
        if (first) put_q.next(a.ahead);
        if (lane == 0) {
            Unit& x = units[stage];
            x.b = b;
            x.h = h;
            x.tile0 = tok;
            x.lo = lo;
            x.len = len;
            x.flags = (first ? kFirst : 0) | (last ? kLast : 0);
            x.part = put_q.stage;
            x.bad = (int)bad;
            mbar_arrive_expect_tx(bars + stage,
                                  (uint32_t)(__popc(copy) * 2 * (C::kRow << a.lg_box) + (first ? n_heads * D * 2 : 0)));
        }
        __syncwarp();
        if (there) {
            const uint32_t dst = smem_u32(kv + stage * 2 * half) + lane * (C::kRow << a.lg_box);
            const int in_block = a.shift > a.lg_box ? tok & ((1 << a.shift) - 1) : 0;
            tma_load_5d(dst, &a.tk, in_block, h, id, bars + stage, policy);
            tma_load_5d(dst + half, &a.tv, in_block, h, id, bars + stage, policy);
        }
        if (first && lane >= 32 - C::kHeadsMax && lane - (32 - C::kHeadsMax) < n_heads) {
            const int j = lane - (32 - C::kHeadsMax);
            bulk_g2s(qs + put_q.stage * C::kQSlot + j * C::kQPitch,
                     a.q + b * a.q_row + (int64_t)(h * a.G + chunk * a.heads + j) * a.q_head, D * 2, bars + stage);
        }
        put_at.next(a.ahead);
        ++issued;
        if (last) r += stride;
        if (last && r < rows) enter();
        else {
            tok += a.unit;
            first = false;
        }
        if (r < rows) ask();
    };
    enter();
    ask();
    for (int i = 0; i < a.ahead && r < rows; ++i) issue();

    Row<kQ, kF8, D, NT> row;
    Turn at;
    int done = 0;
    for (; done < issued; ++done, at.next(a.ahead)) {
        const int stage = at.stage;
        if (!__all_sync(0xffffffffu, wait_for(bars + stage, at.phase, a.status))) break;
        const Unit x = units[stage];
        uint8_t* const base = kv + stage * 2 * half;
        if (x.flags & kFirst) {
            uint8_t* const q_row = qs + x.part * C::kQSlot;
            if constexpr (C::kQShared && kF8 && kQ == ZKV_DT_BF16) {
                for (int p = 0; p < kConsumers; ++p) row.narrow_shared(q_row, p);
                __syncwarp();
            }
            row.init(a, q_row, n_heads, kF8 && a.k_scale ? a.k_scale[x.h] : 1.f);
        }
#pragma unroll 1
        for (int p = 0; p * 16 * C::kSub < a.unit; ++p) row.tokens(a, x, base, half, p);
        if (x.flags & kLast) {  // through the stage to whole lines of the output
            float* buf = reinterpret_cast<float*>(base);
            const float v_scale = kF8 && a.v_scale ? a.v_scale[x.h] : 1.f;
            const int64_t head0 = ((int64_t)x.b * a.kv_heads + x.h) * a.G + chunk * a.heads;
            __syncwarp();
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                float inv[2];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const float sum = row.total(n, e);
                    const int head = 8 * n + 2 * t + e;
                    inv[e] = sum == 0.f ? 0.f : v_scale / sum;
                    if (a.lse && g == 0 && head < n_heads)
                        a.lse[head0 + head] = (row.m[n][e] + log2f(sum)) * 0.6931471805599453f;
                }
                row.put(buf, n, inv);
                __syncwarp();
                for (int idx = lane; idx < 8 * (D / 4); idx += 32) {
                    const int hl = idx / (D / 4), d = 4 * (idx % (D / 4));
                    if (8 * n + hl >= n_heads) continue;
                    const float4 y = *reinterpret_cast<const float4*>(buf + hl * D + (d ^ (((hl >> 1) & 3) << 3)));
                    store4<kQ>(a.out, (head0 + 8 * n + hl) * D + d, y);
                }
                __syncwarp();
            }
        }
        proxy_fence();  // the stage was read and written by these threads; the next copy into it is the async proxy's
        __syncwarp();
        if (r < rows) issue();
    }
    for (; done < issued; ++done, at.next(a.ahead))  // a wait gave up: the copies on their way land in this CTA's memory
        wait_for(bars + at.stage, at.phase, a.status);
}

// ------------------------------------------------------------ joining split rows
constexpr int kJoinThreads = 128;  // few enough to wait beside two decode CTAs

// The parts of a split row, in CTA order: slot 1 of its first CTA, slot 0 of
// the others.  One block per (candidate row, chunk; query head of the chunk):
// the candidates are the rows if there are no more of them than CTAs, else the
// rows in which a CTA's range ends.  Which parts there are follows from the
// lengths, so it is known before the decode grid is waited for; then a warp
// takes every fourth part, eight loads in flight, with the dims over its lanes.
template <int kQ, int D, int kTile>
__global__ void __launch_bounds__(kJoinThreads) pool_join_kernel(const __grid_constant__ DecodeArgs a, int heads_max,
                                                                 int by_row) {
    constexpr int kWarps = kJoinThreads / 32, E = D / 32, kBatch = 8;
    __shared__ int64_t sh[32];
    __shared__ float s_o[kWarps][D];
    __shared__ float2 s_ml[kWarps];
    __shared__ int64_t s_row[2];
    __shared__ int s_bh[2];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int member = blockIdx.x % a.side, chunk = member % a.chunks, cand = blockIdx.x / a.side, head = blockIdx.y;
    // Every path waits for the decode grid before it ends: the next kernel on
    // the stream waits for this one alone.
    if (head >= min(a.heads, a.G - chunk * a.heads)) {
        grid_dep_wait();
        return;
    }
    const Units x = count_units<kTile, kJoinThreads>(a, sh);
    const Ranges cuts(a, x.total);
    if (by_row) {
        const int b = cand / a.head_rows;
        if (b >= x.b_lo && b < x.b_hi) {
            int64_t begin = x.before;
            for (int i = x.b_lo; i < b; ++i)
                begin += (int64_t)row_tiles<kTile>(a, request_len(a, __ldcg(a.lens + i))) * a.head_rows;
            const int tiles = row_tiles<kTile>(a, request_len(a, __ldcg(a.lens + b)));
            s_bh[0] = b;
            s_bh[1] = cand - b * a.head_rows;
            s_row[0] = begin + (int64_t)s_bh[1] * tiles;
            s_row[1] = s_row[0] + tiles;
        }
    } else {
        if (cand >= cuts.count) {
            grid_dep_wait();
            return;
        }
        const int64_t u = cuts.begin(cand + 1) - 1;
        int b, len;
        int64_t off;
        if (locate<kTile>(a, x, u, b, off, len)) {
            const int tiles = row_tiles<kTile>(a, request_len(a, len));
            s_bh[0] = b;
            s_bh[1] = (int)quotient(off, tiles);
            s_row[0] = u - (off - (int64_t)s_bh[1] * tiles);
            s_row[1] = s_row[0] + tiles;
        }
    }
    __syncthreads();
    const int64_t c0 = cuts.owner(s_row[0]);
    const int n = (int)(cuts.owner(s_row[1] - 1) - c0) + 1;
    const int b = s_bh[0], h = s_bh[1] * a.abreast + member / a.chunks;
    grid_dep_wait();
    grid_dep_launch_next();
    if (n == 1 || (!by_row && c0 != cand)) return;
    float m = -INFINITY, l = 0.f, o[E];
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = 0.f;
    for (int i0 = warp; i0 < n; i0 += kWarps * kBatch) {
        float2 y[kBatch][E / 2], s[kBatch];
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {
            const int i = i0 + k * kWarps;
            s[k] = make_float2(-INFINITY, 0.f);
            if (i < n) {
                const int64_t slot = (((c0 + i) * a.side + member) * 2 + (i == 0 ? 1 : 0)) * heads_max + head;
                s[k] = __ldcg(reinterpret_cast<const float2*>(a.stats) + slot);
#pragma unroll
                for (int e = 0; e < E / 2; ++e)
                    y[k][e] = __ldcg(reinterpret_cast<const float2*>(a.parts + slot * D) + 32 * e + lane);
            }
        }
        float mx = m;
#pragma unroll
        for (int k = 0; k < kBatch; ++k) mx = fmaxf(mx, s[k].x);
        const float ref = mx == -INFINITY ? 0.f : mx;
        const float old = exp2_fast(m - ref);
        l *= old;
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] *= old;
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {
            if (i0 + k * kWarps >= n) continue;
            const float w = exp2_fast(s[k].x - ref);
            l += w * s[k].y;
#pragma unroll
            for (int e = 0; e < E / 2; ++e) {
                o[2 * e] += w * y[k][e].x;
                o[2 * e + 1] += w * y[k][e].y;
            }
        }
        m = mx;
    }
    if (lane == 0) s_ml[warp] = make_float2(m, l);
#pragma unroll
    for (int e = 0; e < E / 2; ++e)
        *reinterpret_cast<float2*>(&s_o[warp][64 * e + 2 * lane]) = make_float2(o[2 * e], o[2 * e + 1]);
    __syncthreads();
    float mx = -INFINITY, sum = 0.f, f[kWarps];
#pragma unroll
    for (int w = 0; w < kWarps; ++w) mx = fmaxf(mx, s_ml[w].x);
    const float ref = mx == -INFINITY ? 0.f : mx;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
        f[w] = exp2_fast(s_ml[w].x - ref);
        sum += f[w] * s_ml[w].y;
    }
    const int64_t at = ((int64_t)b * a.kv_heads + h) * a.G + chunk * a.heads + head;
    const float inv = sum == 0.f ? 0.f : (a.v_scale ? __ldcg(a.v_scale + h) : 1.f) / sum;
    if (tid < D / 4) {
        float4 r = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            const float4 y = *reinterpret_cast<const float4*>(&s_o[w][4 * tid]);
            r.x += f[w] * y.x, r.y += f[w] * y.y, r.z += f[w] * y.z, r.w += f[w] * y.w;
        }
        store4<kQ>(a.out, at * D + 4 * tid, make_float4(r.x * inv, r.y * inv, r.z * inv, r.w * inv));
    }
    if (tid == 0 && a.lse) a.lse[at] = (mx + log2f(sum)) * 0.6931471805599453f;
}

// ------------------------------------------------------------ host side
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

// A box holds one head's tokens of a block, at most a tile's and 256.
static int box_tokens(const zkv_pool* p) {
    return std::min(p->block_size, tile_tokens(p->head_dim * element_bytes(p->dtype)));
}

// [block][head][piece][token][bytes of a piece]
static bool encode_pool(uint64_t* to, const zkv_pool* p, void* base, int64_t block, int64_t token, int64_t head) {
    EncodeTiled fn = encode_fn();
    if (!fn) return false;
    const int el = element_bytes(p->dtype), row = p->head_dim * el, inner = std::min(row, 128);
    const cuuint64_t dims[5] = {(cuuint64_t)(inner / el), (cuuint64_t)p->block_size, (cuuint64_t)(row / inner),
                                (cuuint64_t)p->kv_heads, (cuuint64_t)p->n_blocks};
    const cuuint64_t strides[4] = {(cuuint64_t)(token * el), (cuuint64_t)inner, (cuuint64_t)(head * el),
                                   (cuuint64_t)(block * el)};
    const cuuint32_t box[5] = {(cuuint32_t)(inner / el), (cuuint32_t)box_tokens(p),
                               (cuuint32_t)(row / inner), 1, 1};
    const cuuint32_t es[5] = {1, 1, 1, 1, 1};
    const CUtensorMapDataType type = p->dtype == ZKV_DT_BF16  ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                     : p->dtype == ZKV_DT_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                              : CU_TENSOR_MAP_DATA_TYPE_UINT8;
    // L2 fills no more than the bytes a box wants in a row: a 256-byte fill for a token-major pool's 128-byte rows reads
    // the next head's row too, long before its CTA comes to it
    const int64_t run = token * el == row ? 256 : row;
    const CUtensorMapL2promotion fill = run >= 256   ? CU_TENSOR_MAP_L2_PROMOTION_L2_256B
                                        : run >= 128 ? CU_TENSOR_MAP_L2_PROMOTION_L2_128B
                                                     : CU_TENSOR_MAP_L2_PROMOTION_L2_64B;
    CUtensorMap map;
    if (fn(&map, type, 5, base, dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
           inner == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, fill,
           CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
        return false;
    static_assert(sizeof(map) == 128, "tensor map");
    std::memcpy(to, &map, sizeof(map));
    return true;
}

static int sm_count() {
    static int cached[64] = {};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
    if (!cached[dev]) {
        int n = 0;
        if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0) n = 148;
        cached[dev] = n;
    }
    return cached[dev];
}

// Query heads of a row: the G heads of a kv head in equal chunks of at most 16.
struct Heads {
    int chunks, heads, tiles;  // tiles: n-tiles of 8 heads
};
static Heads split_heads(int G) {
    Heads h;
    h.chunks = (G + 15) / 16;
    h.heads = (G + h.chunks - 1) / h.chunks;
    h.chunks = (G + h.heads - 1) / h.heads;  // no chunk without a head
    h.tiles = h.heads <= 8 ? 1 : 2;
    return h;
}

// Ranges that a call can use, `side` CTAs each: its units at most, and what the largest grid has room for.
static int64_t most_groups(int batch, int head_rows, int side, int64_t max_len, int tile) {
    const int64_t tiles = std::max<int64_t>(1, (max_len + tile - 1) / tile);
    const int64_t rows = (int64_t)batch * head_rows, most = kMaxGrid / side;
    return rows >= most ? most : std::min<int64_t>(most, rows * tiles);
}

// Rows of partials in the workspace: two parts of a chunk's heads per CTA of the largest grid.
static size_t part_rows(int batch, int kv_heads, const Heads& h, int64_t max_len) {
    return (size_t)most_groups(batch, kv_heads, h.chunks, max_len, 64) * h.chunks * 2 * 8 * h.tiles;
}

// How a call's rows are cut, from what the host knows: a guess of the longest request.  Every way is right for every
// length; a guess far too short leaves long rows to one CTA, or a cluster, each.
struct Cut {
    bool whole;    // not by units
    int ranks;     // CTAs of a cluster that share a row, if `whole`
    int abreast;   // kv heads walked side by side, if not
};
static Cut plan_call(int batch, int kv_heads, int chunks, int row_bytes, int window, int64_t guess) {
    Cut c{false, 1, 8};
    const int tile = tile_tokens(row_bytes);
    const int64_t longest = window > 0 ? std::min<int64_t>(guess, window) : guess;
    const int64_t rows = (int64_t)batch * kv_heads * chunks;
    const int64_t tiles = (longest + tile - 1) / tile + (window > 0 ? 1 : 0);
    const int64_t bytes = 2 * (int64_t)batch * kv_heads * longest * row_bytes;
    const int64_t wave = 2 * sm_count();  // (one CTA an SM, as 256 dims have it, takes two turns)
    while (c.ranks < kMaxRanks && rows * c.ranks * 2 <= wave && c.ranks * 2 <= tiles) c.ranks *= 2;
    const int64_t ctas = rows * c.ranks, slots = (ctas + wave - 1) / wave * wave;
    const int most = 5 * ctas >= 4 * slots ? 2 * kRankTiles : kRankTiles;
    c.whole = longest <= kWholeTokens || (bytes <= kWholeBytes && tiles <= c.ranks * most);
    if (!c.whole) c.ranks = 1;
    while (kv_heads % c.abreast || c.abreast * chunks > kMaxGrid) --c.abreast;
    return c;
}

// A decode kernel's launch, its limits raised on its first one on a device.
template <int kQ, bool kF8, int D, int NT, bool kRows>
static int launch_kernel(const DecodeArgs& a, int grid, int smem, cudaStream_t st) {
    using C = Cfg<kQ, kF8, D, NT>;
    const auto kernel = kRows ? pool_rows_kernel<kQ, kF8, D, NT> : pool_decode_kernel<kQ, kF8, D, NT>;
    static int raised[64] = {};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return launch_refused();
    if (!raised[dev]) {
        if (cudaFuncSetAttribute((const void*)kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::smem_of(C::kRing)) !=
                cudaSuccess ||
            cudaFuncSetAttribute((const void*)kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess)
            return launch_refused();
        raised[dev] = 1;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)grid);
    cfg.blockDim = dim3(kRows ? 32 * C::kRowWarps : kThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)a.ranks;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = a.ranks > 1 ? 2 : 1;
    if (cudaLaunchKernelEx(&cfg, kernel, a) != cudaSuccess) return launch_refused();
    return launch_status();
}

template <int kQ, bool kF8, int D, int NT>
static int launch_decode(DecodeArgs& a, int guess, cudaStream_t st) {
    using C = Cfg<kQ, kF8, D, NT>;
    const Cut cut = plan_call(a.batch, a.kv_heads, a.chunks, C::kRow, a.window, guess);
    a.whole = cut.whole, a.ranks = cut.ranks, a.abreast = cut.whole ? 1 : cut.abreast;
    a.head_rows = a.kv_heads / a.abreast, a.side = a.abreast * a.chunks;
    if (!a.whole && !a.parts) return ZKV_ERR_ARG;
    const int64_t rows = (int64_t)a.batch * a.head_rows;
    const int64_t wave = std::max(1, C::kPerSm * sm_count() / a.side);
    if (a.ranks > 1) a.groups = (int)rows;
    else a.groups = (int)std::min(wave, most_groups(a.batch, a.head_rows, a.side, a.whole ? 0 : guess, C::kTile));
    const int grid = a.groups * a.side * a.ranks;
    if (a.whole && a.ranks == 1) {
        // A warp a row: in equal loads of whole boxes and products, of which four fit into the ring (or two or three, if a
        // box is too large for that: it is a tile's at most, so two always fit).
        const int longest = a.window > 0 ? std::min(guess, a.window) : guess;
        const int grain = std::max(1 << a.lg_box, 16 * C::kSub), other = C::kQSlot + (int)sizeof(Unit);
        const int most = std::min(C::kTile, std::max(grain, (C::kRing / 4 - other) / (2 * C::kRow) / grain * grain));
        const int loads = std::max(1, (longest + most - 1) / most);
        const int unit = std::max(1, ((longest + loads - 1) / loads + grain - 1) / grain) * grain;
        const int stage = 2 * unit * C::kRow + other, fit = std::min(kMaxStages, C::kRing / stage);
        if (longest <= 16 * C::kSub ||
            (loads == 1 ? rows >= wave
                        : rows >= 2 * wave && loads <= (kF8 ? kRowLoadsF8 : kRowLoads) && fit >= (NT == 1 ? 3 : 4))) {
            a.unit = unit;
            a.workers = std::min(C::kRowWarps, fit);
            a.ahead = fit / a.workers;
            return launch_kernel<kQ, kF8, D, NT, true>(a, grid, C::smem_of(a.workers * a.ahead * stage), st);
        }
    }
    int rc = launch_kernel<kQ, kF8, D, NT, false>(a, grid, C::smem_of(C::kStages * C::kStage), st);
    if (rc == ZKV_OK && !a.whole && a.groups > 1) {
        const int by_row = rows <= a.groups;
        const int cands = by_row ? (int)rows : a.groups;
        rc = launch_pdl_kernel(pool_join_kernel<kQ, D, C::kTile>, dim3(cands * a.side, a.heads), dim3(kJoinThreads), 0,
                               st, a, C::kHeadsMax, by_row);
    }
    return rc;
}

template <int kQ, bool kF8>
static int launch_shape(DecodeArgs& a, int guess, int D, int tiles, cudaStream_t st) {
    if (tiles == 1) {
        if (D == 64) return launch_decode<kQ, kF8, 64, 1>(a, guess, st);
        if (D == 128) return launch_decode<kQ, kF8, 128, 1>(a, guess, st);
        return launch_decode<kQ, kF8, 256, 1>(a, guess, st);
    }
    if (D == 64) return launch_decode<kQ, kF8, 64, 2>(a, guess, st);
    if (D == 128) return launch_decode<kQ, kF8, 128, 2>(a, guess, st);
    return launch_decode<kQ, kF8, 256, 2>(a, guess, st);
}

static size_t up256(size_t x) { return (x + 255) & ~(size_t)255; }

}  // namespace pool
}  // namespace zkv

using namespace zkv;

extern "C" int zkv_pool_init(zkv_pool* p) {
    const int rc = pool::check_pool(p);
    if (rc != ZKV_OK) return rc;
    if (!pool::encode_pool(p->maps, p, p->k, p->k_block, p->k_token, p->k_head) ||
        !pool::encode_pool(p->maps + 16, p, p->v, p->v_block, p->v_token, p->v_head))
        return launch_refused();
    return ZKV_OK;
}

static bool needs_parts(const zkv_pool* p, int batch, const pool::Heads& h, int window, int64_t guess) {
    return !pool::plan_call(batch, p->kv_heads, h.chunks, p->head_dim * pool::element_bytes(p->dtype), window, guess).whole;
}

extern "C" size_t zkv_pool_decode_ws_bytes(const zkv_pool* p, int batch, int q_heads, int window, int64_t max_len) {
    if (pool::check_pool(p) != ZKV_OK || batch < 0 || q_heads < 1 || q_heads % p->kv_heads || window < 0 || max_len < 0)
        return 0;
    const pool::Heads h = pool::split_heads(q_heads / p->kv_heads);
    const int64_t guess = max_len > 0 ? max_len : pool::kMaxLen;  // the table is not known here: the most that any needs
    if (h.chunks > pool::kMaxChunks || !needs_parts(p, batch, h, window, guess)) return 0;
    const size_t rows = pool::part_rows(batch, p->kv_heads, h, guess);
    return pool::up256(rows * 8) + pool::up256(rows * p->head_dim * 4);
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
    if (!q || !lens || !out || (!block_table && width > 0)) return ZKV_ERR_ARG;
    if (!pool::aligned16(q) || q_row % 8 || q_head % 8 || !pool::aligned16(out)) return ZKV_ERR_ALIGN;
    if ((reinterpret_cast<uintptr_t>(workspace) & 255) != 0) return ZKV_ERR_ALIGN;
    const int64_t room = (int64_t)width * p->block_size;
    const int64_t cap = std::min<int64_t>(room, pool::kMaxLen);
    const int64_t guess = max_len > 0 ? std::min(max_len, cap) : cap;
    const pool::Heads hs = pool::split_heads(q_heads / p->kv_heads);
    if (hs.chunks > pool::kMaxChunks) return ZKV_ERR_CAPACITY;
    const bool parts = needs_parts(p, batch, hs, window, guess);  // not with guess 0, a table of no columns
    if (parts && !workspace) return ZKV_ERR_ARG;
    if (parts && ws_bytes < zkv_pool_decode_ws_bytes(p, batch, q_heads, window, guess)) return ZKV_ERR_CAPACITY;
    uint64_t any = 0;
    for (uint64_t w : p->maps) any |= w;
    if (!any) return ZKV_ERR_ARG;  // zkv_pool_init was not called
    pool::DecodeArgs a;
    std::memcpy(&a.tk, p->maps, sizeof(a.tk));
    std::memcpy(&a.tv, p->maps + 16, sizeof(a.tv));
    a.q = (const uint8_t*)q;
    a.k_scale = p->k_scale, a.v_scale = p->v_scale;
    a.lens = lens, a.table = block_table, a.out = out, a.lse = lse, a.status = status;
    a.stats = parts ? (float*)workspace : nullptr;
    a.parts = parts ? a.stats + pool::up256(pool::part_rows(batch, p->kv_heads, hs, guess) * 8) / 4 : nullptr;
    a.q_row = q_row * 2, a.q_head = q_head * 2;
    a.table_ld = table_ld, a.n_blocks = p->n_blocks, a.cap = (int)cap;
    a.batch = batch, a.kv_heads = p->kv_heads, a.G = q_heads / p->kv_heads, a.chunks = hs.chunks, a.heads = hs.heads;
    a.shift = pool::log2_of(p->block_size), a.lg_box = pool::log2_of(pool::box_tokens(p)), a.width = width, a.window = window;
    a.scale = scale, a.softcap = softcap;
    cudaStream_t st = (cudaStream_t)stream;
    if (p->dtype == ZKV_DT_BF16) return pool::launch_shape<ZKV_DT_BF16, false>(a, (int)guess, p->head_dim, hs.tiles, st);
    if (p->dtype == ZKV_DT_F16) return pool::launch_shape<ZKV_DT_F16, false>(a, (int)guess, p->head_dim, hs.tiles, st);
    if (dtype == ZKV_DT_BF16) return pool::launch_shape<ZKV_DT_BF16, true>(a, (int)guess, p->head_dim, hs.tiles, st);
    return pool::launch_shape<ZKV_DT_F16, true>(a, (int)guess, p->head_dim, hs.tiles, st);
}
