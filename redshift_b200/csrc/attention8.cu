// Decode / verify attention over the 8-bit K/V cache (1..10 new tokens): the
// layer of attention.cu's decode kernel with the positions [0, packed) read as
// int8 codes with a scale for every 64 tokens and head (quant8.cu), and the
// positions from `packed` on as fp16 rows of a ring, to which the new tokens'
// rows are appended.
//
//   s_j = (q . k_j) ks_j / 16,  out = sum_j p_j vs_j v_j / sum_j p_j * sigmoid(gate)
//
// with p = softmax(s), integer codes k_j, v_j and the scales of their blocks.  A
// tile of 64 positions is one block, so its two scales are one factor of its
// scores and one of its probabilities.
//
// The floor is the cache's bytes, 2 KB a position: 8 tokens at 139,256 take 73 us
// (3.9 TB/s, 375 TFLOP/s of products, 44 us at the copy rate), 5 at 32,767 27 us, 1
// at 777 12 us; the fp16 cache's kernel takes 101 us for the longest.  What bounds
// it is what a tile moves through shared memory (fp16 images written 64 KB and
// read 64 KB by the MMAs, codes 32 KB: half as much again, and 3 % slower, when the
// codes were staged there too) and, in calls without a pause, the power limit: 990 W
// and 1.45 GHz, 88 us.  About 10 us of a call are its two ends: 4.4 us to the first
// scores, 5.5 us from the last product through the splits' combination.
// What keeps the tensor cores fed at twice the fp16 cache's tile rate:
//  * eight converter warps (four for K, four for V) write the codes as exact fp16
//    numbers into the MMA's swizzled operand images.  They ask for the next tile's
//    codes, straight into registers, as soon as this tile's are written; bulk
//    prefetches into L2 run AHEAD tiles before that;
//  * the eight warps that prepared the queries are the softmax, two for each
//    quarter of TMEM's lanes, which take the tiles in turn: a tile's latency from
//    its scores to its probabilities is longer than its share of the time, and
//    only the running maximum passes from one tile to the next.  They read their
//    scores as 16-lane fragments, which puts the hi and lo halves of a score into
//    the same thread, and write the probabilities back to TMEM over them, where
//    the PV MMA reads its A operand;
//  * a warp of its own issues the MMAs, as one (mma_f16_ts_by), which keeps the
//    issue fast beside warps that use every slot.
// The rest is the fp16 kernel's: queries in TMEM as fp16 hi + lo rows, a lazily
// moved maximum, probabilities as fp16 hi + lo rows, one CTA per (split, K/V
// head), the splits combined in the tail.
//
// Probabilities times the value scale: the running maximum is kept over s + log2
// vs (log2 units), the MMA gets P = 2^(s + log2 vs - max + 6), and the sum adds
// P / vs, so that neither large nor small scales leave fp16's range, and an error
// of the logarithm touches numerator and denominator alike.  The largest P of a
// row is 2^6 to 2^14; hi + lo resolve 2^-25 absolute, 2^-31 of the largest.
#include "attention_core.cuh"
#include "common.cuh"
#include "hotpath.h"

#include <algorithm>
#include <stdexcept>
#include <string>

namespace qv {
namespace {

constexpr int IMAGES = 2;        // fp16 tile images (K and V each)
constexpr int AHEAD = 4;         // code tiles on their way into L2 (K and V each)
constexpr int WARP_ROWS = 16;    // a converter warp's rows of a tile
constexpr int SOFT_WARPS = 8, CONV_WARPS = 4, MMA_WARP = SOFT_WARPS + 2 * CONV_WARPS;
constexpr int THREADS8 = 32 * (MMA_WARP + 1);
constexpr int CODES_TILE = BN * HD;                               // codes of one (block, head)
constexpr int MAX_TILES8 = 160;  // tiles of a CTA (59 at the longest context on 148 SMs)
constexpr float P_BIAS = 6.f;    // log2 units above the running maximum
struct A8Layout {
    static constexpr int SM_KV = 0;                               // images: (K, V) of two tiles
    static constexpr int SM_KV_STAGE = 2 * TILE_BYTES;
    static constexpr int SM_QSTAGE = EPILOGUE_BYTES;              // the queries on their way to TMEM, then the tail's scratch
    static constexpr int SM_BAR = SM_QSTAGE + 2 * DECODE_ROWS * 256;
    static constexpr int SM_ROPE = SM_BAR + 384;                  // (cos, sin) [T][32]; then maxima and scales
    static constexpr int SMEM_BYTES = SM_ROPE + MAX_DECODE_T * 32 * 8;
    static_assert((2 * DECODE_ROWS + 2 * MAX_TILES8) * 4 <= MAX_DECODE_T * 32 * 8);
};
static_assert(A8Layout::SMEM_BYTES <= 227 * 1024, "attention kernel exceeds the shared memory of a CTA");
static_assert(IMAGES * A8Layout::SM_KV_STAGE <= A8Layout::SM_QSTAGE, "the images overlap the staged queries");
static_assert(BN == CACHE8_BLOCK, "a tile is a block of the cache");

// A tile's codes are read once by this SM: not kept in L1.
__device__ __forceinline__ uint4 ld_once(const uint4 *a) {
    uint4 v;
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(a) : "memory");
    return v;
}
// `bytes` (a multiple of 16) on their way into L2.
__device__ __forceinline__ void prefetch_l2_bulk(const void *a, uint32_t bytes) {
    asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" :: "l"(a), "r"(bytes) : "memory");
}
struct Cache8View {
    const int8_t *kc, *vc;       // codes [block][4][64][256]
    const float *ks, *vs;        // scales [block][4]
    int blocks;                  // packed blocks: tiles [0, blocks)
    int ring;                    // rows of the fp16 ring
};

// Eight codes as fp16 numbers: 1024 + u is the fp16 number 0x6400 | u of a biased
// byte u = code + 128, and its difference to 1152, the code, is exact.  (Keys as the
// subnormal numbers u 2^-24, their bias taken off the scores again, need no
// subtraction here, 69.7 instead of 72.3 us for 8 tokens at 139,256, but the
// scores are then small differences of sums four times their size and more, and the
// outputs' error grew by 1.6.)
__device__ __forceinline__ uint32_t fp16_pair(uint32_t biased, uint32_t select) {
    const uint32_t w = __byte_perm(biased, 0x64646464u, select);
    return half2_bits(__hsub2(*reinterpret_cast<const __half2 *>(&w), __half2half2(__ushort_as_half(0x6480))));
}
__device__ __forceinline__ uint4 fp16_codes(uint32_t a, uint32_t b) {
    a ^= 0x80808080u;
    b ^= 0x80808080u;
    return make_uint4(fp16_pair(a, 0x4140), fp16_pair(a, 0x4342), fp16_pair(b, 0x4140), fp16_pair(b, 0x4342));
}

// Append (converter warps, positions pos, pos + 8, ... below `end`): RMSNorm +
// rotary of the new keys, fp16 keys and values into the ring.  What lands in the
// cache is read by every later token, so the keys are formed in 64 bits, and the
// correctly rounded fp32 value goes to fp16 (formed in 32 bits, a value near a border
// of two fp16 numbers now and then went to the further one); the warps are idle
// meanwhile.  Returns the tokens, as bits, whose fp16 values are not all finite.
__device__ __forceinline__ uint32_t append_row8(const FaParams &p, int ring, int kv_head, int pos, int end) {
    const int lane = threadIdx.x & 31;
    uint32_t bad = 0;
#pragma unroll 1
    for (; pos < end; pos += 2 * CONV_WARPS) {
        const int t = pos - p.position;
        const size_t src = ((size_t)t * NKV + kv_head) * HD + 4 * lane, dst = ((size_t)(pos % ring) * NKV + kv_head) * HD + 4 * lane;
        float k[8], w[8], v[8];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            *reinterpret_cast<float4 *>(k + 4 * h) = *reinterpret_cast<const float4 *>(p.key + src + 128 * h);
            *reinterpret_cast<float4 *>(w + 4 * h) = *reinterpret_cast<const float4 *>(p.kn + 4 * lane + 128 * h);
            *reinterpret_cast<float4 *>(v + 4 * h) = *reinterpret_cast<const float4 *>(p.value + src + 128 * h);
        }
        double ss = 0., x[8], cosine, sine;
        sincospi((double)pos * kRopeInvFreq[lane] * 0.3183098861837907, &sine, &cosine);      // angle of dims lane, lane + 32
#pragma unroll
        for (int e = 0; e < 8; ++e) ss = fma((double)k[e], (double)k[e], ss);
#pragma unroll
        for (int o = 16; o; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        const double inv = rsqrt(ss / HD + (double)p.eps);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = (double)k[e] * inv * (double)w[e];
#pragma unroll
        for (int e = 0; e < 4; ++e) {                          // dims 4 lane + e: lanes 0..7 pair with 8..15
            const double partner = __shfl_xor_sync(0xffffffffu, x[e], 8);
            const double c = __shfl_sync(0xffffffffu, cosine, 4 * (lane & 7) + e), s = __shfl_sync(0xffffffffu, sine, 4 * (lane & 7) + e);
            if (lane < 16) x[e] = fma(partner, lane < 8 ? -s : s, x[e] * c);
        }
        bool finite = true;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            __half2 kh[2], vh[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                kh[e] = __floats2half2_rn((float)x[4 * h + 2 * e], (float)x[4 * h + 2 * e + 1]);
                vh[e] = __floats2half2_rn(v[4 * h + 2 * e], v[4 * h + 2 * e + 1]);
                const float2 f = __half22float2(__habs2(vh[e]));
                finite = finite && f.x <= 65504.f && f.y <= 65504.f;
            }
            *reinterpret_cast<uint2 *>(p.kc + dst + 128 * h) = make_uint2(half2_bits(kh[0]), half2_bits(kh[1]));
            *reinterpret_cast<uint2 *>(p.vc + dst + 128 * h) = make_uint2(half2_bits(vh[0]), half2_bits(vh[1]));
        }
        if (!__all_sync(0xffffffffu, finite)) bad |= 1u << t;
    }
    return bad;
}

__global__ void __launch_bounds__(THREADS8, 1) attention8_kernel(const FaParams p, const Cache8View c) {
    using L = A8Layout;
    extern __shared__ __align__(1024) uint8_t smem[];
    if (smem_addr(smem) & 1023) {           // 128B-swizzle atoms need a 1024-byte aligned base
        if (threadIdx.x == 0) raise_status(STATUS_BAD_ARGUMENT);
        return;
    }
    uint64_t *k_full = reinterpret_cast<uint64_t *>(smem + L::SM_BAR), *v_full = k_full + 2, *k_empty = k_full + 4,
             *v_empty = k_full + 6, *s_full = k_full + 8, *p_full = k_full + 10, *p_free = k_full + 12, *mma_done = k_full + 14,
             *q_ready = k_full + 15, *app_done = k_full + 16, *cbar = k_full + 17, *q_loaded = k_full + 18, *maximum_of = k_full + 19;  // 27 in all
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(smem + L::SM_BAR + 320);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(smem + L::SM_BAR + 324);
    uint32_t *bad_values = reinterpret_cast<uint32_t *>(smem + L::SM_BAR + 328);
    float2 *rope = reinterpret_cast<float2 *>(smem + L::SM_ROPE);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int kv_head = blockIdx.y;
    const int total = (p.kv_rows + BN - 1) / BN;
    const int tile0 = blockIdx.x * p.split_tiles;
    const int ntiles = min(p.split_tiles, total - tile0);
    // The block's new rows that fall into this CTA's tiles (absolute positions).
    const int app_lo = max(p.position, tile0 * BN), app_hi = min(p.position + p.T, (tile0 + ntiles) * BN);
    const bool appends = app_hi > app_lo;

    for (int i = threadIdx.x; i < p.T * GROUP * 8; i += blockDim.x) {    // 8 lines of 128 B per query row
        const int rr = i >> 3;
        prefetch_l2(p.q_gate + ((size_t)(rr / GROUP) * NQ + kv_head * GROUP + rr % GROUP) * 2 * HD + (i & 7) * 32);
    }
    if (threadIdx.x == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(k_full + i, CONV_WARPS); mbar_init(v_full + i, CONV_WARPS);
            mbar_init(k_empty + i, 1); mbar_init(v_empty + i, 1);
            mbar_init(s_full + i, 1); mbar_init(p_full + i, SOFT_WARPS / 2); mbar_init(p_free + i, 1);
        }
        mbar_init(mma_done, 1);
        mbar_init(q_loaded, 1);
        mbar_init(q_ready, 8);
        mbar_init(cbar, 1);
        mbar_init(app_done, 2 * CONV_WARPS * 32);
        for (int i = 0; i < 8; ++i) mbar_init(maximum_of + i, 1);
        *abort_flag = 0;
        *bad_values = 0;
        fence_barrier_init();
    }
    if (warp == 1) { tmem_alloc(tmem_slot, 512); tmem_relinquish(); }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    // A converter warp's quarter of the tiles.  The first ones are asked for into L2 while
    // the kernel before still runs; what it may yet write to them arrives there too
    // (behind a norm8, 5 tokens at 32,767: 31.5 -> 30.0 us for both).
    const int code_tiles = max(0, min(ntiles, c.blocks - tile0));       // tiles of codes, the first of this CTA's
    const bool converts = warp >= SOFT_WARPS && warp < MMA_WARP;
    const size_t step = (size_t)NKV * CODES_TILE;
    const int8_t *codes = ((warp - SOFT_WARPS) >> 2 ? c.vc : c.kc) + ((size_t)tile0 * NKV + kv_head) * CODES_TILE + WARP_ROWS * (warp & 3) * HD;
    auto prefetch = [&](int j) {
        if (lane == 0 && j < code_tiles) prefetch_l2_bulk(codes + j * step, WARP_ROWS * HD);
    };
    if (converts)
        for (int i = 0; i < AHEAD; ++i) prefetch(i);
    grid_dependency_wait();
    if (threadIdx.x == 0) launch_dependents();

    if (converts) {
        // ------------------------------------------------ converters (warps 8-11: K, 12-15: V)
        // A lane takes 16 codes (16 dims of a row) at a time: 16 bytes of the
        // block, two 16-byte chunks of a 64-dim box of the image.  Eight
        // lanes are four neighbouring pieces of an even row and four, in the
        // box's neighbour, of the odd row after it: their loads cover the two
        // halves of 128 bytes and their stores, swizzled by the row, even and
        // odd chunks.
        const int part = (warp - SOFT_WARPS) >> 2, w = warp & 3, q = lane & 3, odd = lane >> 2 & 1;
        const int box = (lane >> 3) ^ odd, piece = 4 * box + q, row0 = WARP_ROWS * w + odd;
        const uint32_t image = box * (BN * 128) + row0 * 128;
        uint4 x[8];
        auto load = [&](int j) {
            const int8_t *src = codes + j * step + odd * HD + piece * 16;
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = ld_once(reinterpret_cast<const uint4 *>(src + i * 2 * HD));
        };
        auto convert = [&](uint8_t *dst) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                uint8_t *d = dst + image + i * 256;
                const int swizzle = (2 * i + odd) & 7;
                *reinterpret_cast<uint4 *>(d + (((2 * q) ^ swizzle) << 4)) =
                    fp16_codes(x[i].x, x[i].y);
                *reinterpret_cast<uint4 *>(d + (((2 * q + 1) ^ swizzle) << 4)) =
                    fp16_codes(x[i].z, x[i].w);
            }
        };
        // A tile of fp16 rows; rows past the last position and value rows in `skip` (new tokens, bits) are zero.
        auto copy_rows = [&](uint8_t *dst, const __half *rows, int j, uint32_t skip) {
            const int pos0 = (tile0 + j) * BN + row0;
#pragma unroll 4
            for (int i = 0; i < 8; ++i) {
                const int pos = pos0 + 2 * i;
                uint4 a = make_uint4(0u, 0u, 0u, 0u), b = a;
                if (pos < p.kv_rows && !(pos >= p.position && (skip >> (pos - p.position) & 1u))) {
                    const uint4 *src = reinterpret_cast<const uint4 *>(rows + ((size_t)(pos % c.ring) * NKV + kv_head) * HD + piece * 16);
                    a = src[0]; b = src[1];
                }
                uint8_t *d = dst + image + i * 256;
                const int swizzle = (2 * i + odd) & 7;
                *reinterpret_cast<uint4 *>(d + (((2 * q) ^ swizzle) << 4)) = a;
                *reinterpret_cast<uint4 *>(d + (((2 * q + 1) ^ swizzle) << 4)) = b;
            }
        };
        auto publish = [&](uint64_t *bar) {
            fence_async_shared();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar);
        };
        if (appends) {                                        // while the first tiles are on their way
            const uint32_t bad = append_row8(p, c.ring, kv_head, app_lo + (warp - SOFT_WARPS), app_hi);
            if (lane == 0 && bad) atomicOr(bad_values, bad);
            __threadfence_block();
            mbar_arrive(app_done);
        }
        uint64_t *full = part ? v_full : k_full, *empty = part ? v_empty : k_empty;
        const __half *rows = part ? p.vc : p.kc;
        // The first tile is asked for once the query rows have arrived, which would
        // wait behind it.
        if (!warp_wait(q_loaded, 0, abort_flag)) return;
        if (code_tiles > 0) load(0);
        for (int j = 0; j < ntiles; ++j) {
            const int s = j & 1;
            uint8_t *dst = smem + L::SM_KV + s * L::SM_KV_STAGE + part * TILE_BYTES;
            const bool fresh = appends && (tile0 + j + 1) * BN > p.position;      // the tile holds new rows
            prefetch(j + AHEAD);
            if (fresh && !warp_wait(app_done, 0, abort_flag)) break;
            if (j >= 2 && !warp_wait(empty + s, (uint32_t)((j >> 1) - 1) & 1, abort_flag)) break;
            if (j >= code_tiles) copy_rows(dst, rows, j, part && fresh ? *reinterpret_cast<volatile uint32_t *>(bad_values) : 0u);
            else convert(dst);
            if (j + 1 < code_tiles) load(j + 1);
            publish(full + s);
        }
        return;                          // the later barriers count the first eight warps
    }

    if (warp == MMA_WARP) {
        // ------------------------------------------------ MMA issuer (the whole warp, one elected lane)
        const uint32_t lead = elect_lane(), tm = __shfl_sync(0xffffffffu, tmem, 0);
        const uint32_t idesc_qk = idesc_f16(128, BN, false, false), idesc_pv = idesc_f16(128, HD, false, true);
        auto issue_pv = [&](int i) -> bool {
            const int b = i & 1, s = i & 1;
            if (!warp_wait(p_full + b, (i >> 1) & 1, abort_flag)) return false;
            if (!warp_wait(v_full + s, (i >> 1) & 1, abort_flag)) return false;
            tc_fence_after();
            const uint64_t vd = sw128_desc(smem_addr(smem + L::SM_KV + s * L::SM_KV_STAGE + TILE_BYTES), BN * 128, 1024);
#pragma unroll
            for (int k = 0; k < BN / 16; ++k)     // P (hi / lo rows) from TMEM
                mma_f16_ts_by(lead, tm + TM_O, tm + TM_S + b * BN + k * 8, vd + k * 128, idesc_pv, (i > 0 || k > 0) ? 1u : 0u);
            mma_commit_by(lead, p_free + b);
            mma_commit_by(lead, v_empty + s);
            return true;
        };
        bool ok = warp_wait(q_ready, 0, abort_flag);
        tc_fence_after();
        for (int j = 0; j < ntiles && ok; ++j) {
            const int b = j & 1, s = j & 1;
            if (!warp_wait(k_full + s, (j >> 1) & 1, abort_flag)) { ok = false; break; }
            // S / P buffer b is free: PV(j-2), issued before, has read its P first.
            tc_fence_after();
            const uint64_t kd = sw128_desc(smem_addr(smem + L::SM_KV + s * L::SM_KV_STAGE), 16, 1024);
#pragma unroll
            for (int k = 0; k < HD / 16; ++k)
                mma_f16_ts_by(lead, tm + TM_S + b * BN, tm + TM_Q + k * 8, kd + (k >> 2) * (BN * 128 / 16) + (k & 3) * 2,
                              idesc_qk, k > 0 ? 1u : 0u);
            mma_commit_by(lead, s_full + b);
            mma_commit_by(lead, k_empty + s);
            if (j >= 1) ok = issue_pv(j - 1);
        }
        if (ok && ntiles > 0) issue_pv(ntiles - 1);
        // All MMAs must finish before TMEM is released.
        mma_commit_by(lead, mma_done);
        const long long t0 = clock64();
        while (!mbar_try_wait(mma_done, 0) && clock64() - t0 < WAIT_LIMIT_CYCLES) {}
        return;
    }

    // The scales of this CTA's tiles, one tile a thread: read one by one inside
    // the loop, each tile waited for a miss in memory.
    float k_scale = 1.f, v_scale = 1.f;
    if ((int)threadIdx.x < code_tiles) {
        k_scale = c.ks[(size_t)(tile0 + threadIdx.x) * NKV + kv_head];
        v_scale = c.vs[(size_t)(tile0 + threadIdx.x) * NKV + kv_head];
    }
    prepare_queries(p, kv_head, rope, smem + L::SM_QSTAGE, tmem, q_ready, [&] { mbar_arrive(q_loaded); });
    {
        // ------------------------------------------------ softmax
        // Lanes 32g + i and 32g + 16 + i of TMEM hold the hi and lo halves of query
        // row 16g + i.  Warps g and g + 4 have the rows of g, the first in the even
        // tiles, the second in the odd ones; thread l of them the rows 16g + l / 4 +
        // 8 u (u = 0, 1) and, of these, the columns 8 n + 2 (l % 4) + e in x[2 n + u].
        const int wq = warp & 3, turn = warp >> 2;
        const uint32_t t_hi = tmem + ((uint32_t)(wq * 32) << 16), t_lo = t_hi + (16u << 16);
        const int r0 = wq * 16 + (lane >> 2), rows = p.T * GROUP;
        int last[2];                                               // last visible position
        float m_use[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
        for (int u = 0; u < 2; ++u) last[u] = r0 + 8 * u < rows ? p.position + (r0 + 8 * u) / GROUP : -1;
        // Once the queries are rotated, the rotary table's place takes the running
        // maxima and the scales.
        float *maxima = reinterpret_cast<float *>(rope);           // [tile parity][64 rows]
        float *scales = maxima + 2 * DECODE_ROWS;
        named_barrier(4, 32 * SOFT_WARPS);
        if (threadIdx.x < MAX_TILES8) *reinterpret_cast<float2 *>(scales + 2 * threadIdx.x) = make_float2(k_scale, v_scale);
        named_barrier(6, 32 * SOFT_WARPS);
        for (int j = turn; j < ntiles; j += 2) {
            const int b = turn;
            const bool codes = j < code_tiles;
            const float2 scale = *reinterpret_cast<const float2 *>(scales + 2 * j);
            const float to_log2 = SCORE_LOG2 * scale.x;            // a score in log2 units (rows have the scales 1)
            // a scale of (almost) zero: its codes count nothing, its keys still do; NaN stays
            const float vs = scale.y < 0x1p-100f ? 0x1p-100f : scale.y;
            const float v_log2 = log2_approx(vs), v_inv = rcp_approx(vs);
            // The running maximum of the tile before, from this row's other warp; its
            // tile is half a round ahead, so that this costs nothing before the scores.
            float before[2] = {-INFINITY, -INFINITY};
            if (j > 0) {
                if (!warp_wait(maximum_of + 2 * wq + (b ^ 1), ((j - 1) >> 1) & 1, abort_flag)) break;
#pragma unroll
                for (int u = 0; u < 2; ++u) before[u] = maxima[(b ^ 1) * DECODE_ROWS + r0 + 8 * u];
            }
            if (!warp_wait(s_full + b, (j >> 1) & 1, abort_flag)) break;
            tc_fence_after();
            float2 x[16];
#pragma unroll
            for (int part = 0; part < 2; ++part) {
                float hi[16], lo[16];
                tmem_ld_16x256b_x4(t_hi + TM_S + b * BN + part * 32, hi);
                tmem_ld_16x256b_x4(t_lo + TM_S + b * BN + part * 32, lo);
                tmem_wait_ld();
#pragma unroll
                for (int q = 0; q < 8; ++q)
                    x[8 * part + q] = fadd2(make_float2(hi[2 * q], hi[2 * q + 1]), make_float2(lo[2 * q], lo[2 * q + 1]));
            }
            if (!codes) {                                          // only fp16 tiles hold positions past a query
                const int key0 = (tile0 + j) * BN + 2 * (lane & 3);
                uint32_t bad = 0;
                if (appends && (tile0 + j + 1) * BN > p.position) {
                    if (!warp_wait(app_done, 0, abort_flag)) break;
                    bad = *reinterpret_cast<volatile uint32_t *>(bad_values);
                }
                // A new value row that is not finite was left out of the V tile (0 *
                // NaN would reach the queries that do not see it): the queries that
                // see it become NaN here.
                auto masked = [&](float v, int key, int u) {
                    const int age = key - p.position;
                    if (bad && age >= 0 && age < 32 && (bad >> age & 1u)) v = __int_as_float(0x7FC00000);
                    return key <= last[u] ? v : -INFINITY;
                };
#pragma unroll
                for (int q = 0; q < 16; ++q) {
                    x[q].x = masked(x[q].x, key0 + 8 * (q >> 1), q & 1);
                    x[q].y = masked(x[q].y, key0 + 8 * (q >> 1) + 1, q & 1);
                }
            }
            // The largest of this thread's columns, in log2 units.  The running maximum
            // moves only when a tile's is far above it, so that most tiles need no
            // more than this and a vote.
            float m[2];
            bool above = false;
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                float m0 = fmaxf(x[u].x, x[u].y), m1 = fmaxf(x[2 + u].x, x[2 + u].y);
#pragma unroll
                for (int n = 2; n < 8; n += 2) {
                    m0 = fmaxf(m0, fmaxf(x[2 * n + u].x, x[2 * n + u].y));
                    m1 = fmaxf(m1, fmaxf(x[2 * n + 2 + u].x, x[2 * n + 2 + u].y));
                }
                m[u] = fmaf(fmaxf(m0, m1), to_log2, v_log2);       // -inf stays -inf
                above = above || m[u] > before[u] + RESCALE_THRESHOLD;
            }
            const bool need = __any_sync(0xffffffffu, above);
            if (need) {                                            // the rows' maxima: their other three threads
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    m[u] = fmaxf(m[u], __shfl_xor_sync(0xffffffffu, m[u], 1));
                    m[u] = fmaxf(m[u], __shfl_xor_sync(0xffffffffu, m[u], 2));
                    m[u] = m[u] > before[u] + RESCALE_THRESHOLD ? m[u] : before[u];
                }
            } else {
#pragma unroll
                for (int u = 0; u < 2; ++u) m[u] = before[u];
            }
            if (j > 0 && need) {
                // O holds the tiles before j: wait for PV(j-1), then rescale its rows.
                if (!warp_wait(p_free + (b ^ 1), ((j - 1) >> 1) & 1, abort_flag)) break;
                tc_fence_after();
                float factor[2];
#pragma unroll
                for (int u = 0; u < 2; ++u) factor[u] = m[u] == before[u] ? 1.f : exp2_approx(before[u] - m[u]);
#pragma unroll 1
                for (int q = 0; q < 2 * HD / 32; ++q) {
                    const uint32_t at = (q & 1 ? t_lo : t_hi) + TM_O + (q >> 1) * 32;
                    float o[16];
                    uint32_t scaled[16];
                    tmem_ld_16x256b_x4(at, o);
                    tmem_wait_ld();
#pragma unroll
                    for (int e = 0; e < 16; ++e) scaled[e] = __float_as_uint(o[e] * factor[e >> 1 & 1]);
                    tmem_st_16x256b_x4(at, scaled);
                }
                tmem_wait_st();
                tc_fence_before();
            }
            if ((lane & 3) == 0) {
#pragma unroll
                for (int u = 0; u < 2; ++u) maxima[b * DECODE_ROWS + r0 + 8 * u] = m[u];
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(maximum_of + 2 * wq + b);
            const float2 scale2 = make_float2(to_log2, to_log2), minus = make_float2(-1.f, -1.f);
            float2 shift[2], sum[2];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                if (m[u] != m_use[u]) {                            // moved since this warp's last tile
                    l[u] *= exp2_approx(m_use[u] - m[u]);
                    m_use[u] = m[u];
                }
                const float f = v_log2 + P_BIAS - (m_use[u] == -INFINITY ? 0.f : m_use[u]);
                shift[u] = make_float2(f, f);
                sum[u] = make_float2(0.f, 0.f);
            }
            __syncwarp();                                          // all lanes store to TMEM together
#pragma unroll
            for (int part = 0; part < 2; ++part) {
                uint32_t hi[8], lo[8];
#pragma unroll
                for (int q = 0; q < 8; ++q) {
                    const float2 arg = ffma2(x[8 * part + q], scale2, shift[q & 1]);
                    const float2 e = make_float2(exp2_approx(arg.x), exp2_approx(arg.y));
                    sum[q & 1] = fadd2(sum[q & 1], e);
                    const __half2 h = __floats2half2_rn(e.x, e.y);
                    hi[q] = half2_bits(h);
                    const float2 rest = ffma2(__half22float2(h), minus, e);
                    lo[q] = half2_bits(__floats2half2_rn(rest.x, rest.y));
                }
                tmem_st_16x128b_x4(t_hi + TM_S + b * BN + part * 16, hi);
                tmem_st_16x128b_x4(t_lo + TM_S + b * BN + part * 16, lo);
            }
#pragma unroll
            for (int u = 0; u < 2; ++u) l[u] = fmaf(sum[u].x + sum[u].y, v_inv, l[u]);
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(p_full + b);
        }
        // The rows' maximum and sum, for the split combine: the last tile's warp has
        // the final maximum, the other brings its sum to it.
        float *finals = maxima + 2 * DECODE_ROWS;                  // (max, sum) [64], over the scales
        const bool ends = turn == ((ntiles - 1) & 1);
        named_barrier(4, 32 * SOFT_WARPS);
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            l[u] += __shfl_xor_sync(0xffffffffu, l[u], 1);
            l[u] += __shfl_xor_sync(0xffffffffu, l[u], 2);
            if (!ends && (lane & 3) == 0)
                *reinterpret_cast<float2 *>(finals + 2 * (r0 + 8 * u)) = make_float2(m_use[u], l[u]);
        }
        named_barrier(8 + wq, 64);
#pragma unroll
        for (int u = 0; u < 2; ++u)
            if (ends && (lane & 3) == 0 && r0 + 8 * u < rows) {
                const float2 o = *reinterpret_cast<const float2 *>(finals + 2 * (r0 + 8 * u));
                const float w = o.x == m_use[u] ? 1.f : exp2_approx(o.x - m_use[u]);
                const size_t slot = ((size_t)kv_head * DECODE_ROWS + r0 + 8 * u) * MAXS + blockIdx.x;
                p.part_ml[slot * 2] = m_use[u];
                p.part_ml[slot * 2 + 1] = fmaf(o.y, w, l[u]);
            }
    }
    // The final PV's commit on p_free marks O complete and every image consumed.
    __syncwarp();
    named_barrier(5, 256);
    const bool o_ready = ntiles > 0 && warp_wait(p_free + ((ntiles - 1) & 1), ((ntiles - 1) >> 1) & 1, abort_flag);
    if (o_ready) {
        tc_fence_after();
        store_partials(p, kv_head, tmem, smem + L::SM_KV);
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 1) tmem_dealloc(tmem, 512);     // the warp that allocated it
    decode_tail(p, kv_head, smem + L::SM_QSTAGE, reinterpret_cast<float *>(smem + L::SM_KV), cbar, abort_flag);
}

PerDeviceOnce g_configured8;

}  // namespace

size_t attention8_workspace_bytes(int kv_rows) { return decode_parts_bytes(decode_split(kv_rows)); }

void attention8_run(float *out, const int8_t *kc, const float *ks, const int8_t *vc, const float *vs, int packed,
                    __half *k_tail, __half *v_tail, int ring, const float *q_gate, const float *key, const float *value,
                    const float *qn, const float *kn, int T, int position, float eps, void *ws, size_t ws_bytes,
                    cudaStream_t st) {
    g_configured8.run([] {
        if (cudaFuncSetAttribute(attention8_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, A8Layout::SMEM_BYTES) !=
            cudaSuccess)
            throw std::runtime_error("cannot reserve shared memory for the 8-bit attention kernel");
    });
    const int rows = position + T;
    const Split sp = decode_split(rows);
    if (ws_bytes < decode_parts_bytes(sp)) throw std::invalid_argument("attention workspace too small");
    if (sp.tiles > MAX_TILES8) throw std::runtime_error("too few SMs for the 8-bit attention kernel");
    const DecodeParts parts = decode_parts(ws, sp);
    FaParams p{};
    p.q_gate = q_gate; p.out = out; p.T = T; p.position = position; p.kv_rows = rows;
    p.split_tiles = sp.tiles; p.splits = sp.splits;
    p.part_o = parts.o; p.part_ml = parts.ml; p.sync = parts.sync;
    p.tail = TAIL_GATED; p.world = 1;
    p.key = key; p.value = value; p.qn = qn; p.kn = kn; p.kc = k_tail; p.vc = v_tail;
    p.append_row0 = position; p.eps = eps;
    const Cache8View c{kc, vc, ks, vs, packed / CACHE8_BLOCK, ring};
    const cudaError_t e = launch_chained(attention8_kernel, dim3(sp.splits, NKV), dim3(THREADS8), A8Layout::SMEM_BYTES, st, p, c);
    if (e != cudaSuccess) throw std::runtime_error(std::string("8-bit attention: ") + cudaGetErrorString(e));
}

}  // namespace qv
