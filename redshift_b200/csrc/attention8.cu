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
// Bound by the cache's bytes, 2 KB a position.  What keeps the tensor cores fed
// at twice the fp16 cache's tile rate:
//  * a block of one head is 16 KB in a row: one bulk copy each, into a ring of
//    six (96 KB in flight per SM);
//  * four converter warps write the codes as exact fp16 integers into the MMA's
//    swizzled operand images, without bank conflicts on either side;
//  * the softmax reads its scores as 16-lane fragments, which puts the hi and lo
//    halves of a score into the same thread, and writes the probabilities back to
//    TMEM over them, where the PV MMA reads its A operand;
//  * the MMA warp issues as one (mma_f16_ts_by), which keeps it fast beside warps
//    that use every issue slot.
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
constexpr int RAW_SLOTS = 6;     // tiles of codes in flight
constexpr int CODES_TILE = BN * HD;                               // codes of one (block, head)
constexpr float P_BIAS = 6.f;    // log2 units above the running maximum
struct A8Layout {
    static constexpr int SM_KV = 0;                               // images: (K, V) of two tiles
    static constexpr int SM_KV_STAGE = 2 * TILE_BYTES;
    static constexpr int SM_RAW = SM_KV + IMAGES * SM_KV_STAGE;   // ring of code tiles, K and V in turn
    static constexpr int SM_QSTAGE = SM_RAW + 4 * CODES_TILE;     // slots 4 and 5 until the queries are in TMEM
    static constexpr int SM_BAR = SM_RAW + RAW_SLOTS * CODES_TILE;
    static constexpr int SM_ROPE = SM_BAR + 256;                  // (cos, sin) [T][32]
    static constexpr int SMEM_BYTES = SM_ROPE + MAX_DECODE_T * 32 * 8;
};
static_assert(A8Layout::SMEM_BYTES <= 227 * 1024, "attention kernel exceeds the shared memory of a CTA");
static_assert(EPILOGUE_BYTES <= A8Layout::SM_BAR, "O staging exceeds the images and the ring");
static_assert(BN == CACHE8_BLOCK, "a tile is a block of the cache");

struct Cache8View {
    const int8_t *kc, *vc;       // codes [block][4][64][256]
    const float *ks, *vs;        // scales [block][4]
    int blocks;                  // packed blocks: tiles [0, blocks)
    int ring;                    // rows of the fp16 ring
};

// Two fp16 integers of the codes' biased bytes (code + 128): 1024 + byte is the
// fp16 number 0x6400 | byte, and the difference to 1152 is exact.
__device__ __forceinline__ uint32_t fp16_codes(uint32_t biased, uint32_t select) {
    const uint32_t w = __byte_perm(biased, 0x64646464u, select);
    return half2_bits(__hsub2(*reinterpret_cast<const __half2 *>(&w), __half2half2(__ushort_as_half(0x6480))));
}
__global__ void __launch_bounds__(384, 1) attention8_kernel(const FaParams p, const Cache8View c) {
    using L = A8Layout;
    constexpr int SOFT_WARPS = 4, CONV_WARPS = 4;
    extern __shared__ __align__(1024) uint8_t smem[];
    if (smem_addr(smem) & 1023) {           // 128B-swizzle atoms need a 1024-byte aligned base
        if (threadIdx.x == 0) raise_status(STATUS_BAD_ARGUMENT);
        return;
    }
    uint64_t *raw_full = reinterpret_cast<uint64_t *>(smem + L::SM_BAR), *raw_empty = raw_full + RAW_SLOTS;
    uint64_t *k_full = raw_empty + RAW_SLOTS, *v_full = k_full + 2, *k_empty = k_full + 4, *v_empty = k_full + 6,
             *s_full = k_full + 8, *p_full = k_full + 10, *p_free = k_full + 12, *mma_done = k_full + 14,
             *q_ready = k_full + 15, *app_done = k_full + 16, *cbar = k_full + 17;      // 30 barriers
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(smem + L::SM_BAR + 240);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(smem + L::SM_BAR + 244);
    uint32_t *bad_values = reinterpret_cast<uint32_t *>(smem + L::SM_BAR + 248);
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
        for (int i = 0; i < RAW_SLOTS; ++i) { mbar_init(raw_full + i, 1); mbar_init(raw_empty + i, CONV_WARPS); }
        for (int i = 0; i < 2; ++i) {
            mbar_init(k_full + i, CONV_WARPS); mbar_init(v_full + i, CONV_WARPS);
            mbar_init(k_empty + i, 1); mbar_init(v_empty + i, 1);
            mbar_init(s_full + i, 1); mbar_init(p_full + i, SOFT_WARPS); mbar_init(p_free + i, 1);
        }
        mbar_init(mma_done, 1);
        mbar_init(q_ready, 8);
        mbar_init(cbar, 1);
        mbar_init(app_done, 64);
        *abort_flag = 0;
        *bad_values = 0;
        fence_barrier_init();
    }
    if (warp == 1) { tmem_alloc(tmem_slot, 512); tmem_relinquish(); }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    grid_dependency_wait();
    if (threadIdx.x == 0) launch_dependents();

    // Tiles of codes among this CTA's (the first ones), as halves: tile j's K is 2 j, its V 2 j + 1.
    const int code_tiles = max(0, min(ntiles, c.blocks - tile0));
    auto issue_half = [&](int h) {
        const int8_t *src = (h & 1 ? c.vc : c.kc) + ((size_t)(tile0 + (h >> 1)) * NKV + kv_head) * CODES_TILE;
        uint64_t *bar = raw_full + h % RAW_SLOTS;
        mbar_expect_tx(bar, CODES_TILE);
        bulk_load(smem + L::SM_RAW + h % RAW_SLOTS * CODES_TILE, src, CODES_TILE, bar);
    };

    if (warp >= 8) {
        // ------------------------------------------------ converters
        // A lane takes 16 codes (16 dims of a row) at a time: 16 bytes of the
        // code tile, two 16-byte chunks of a 64-dim box of the image.  Eight
        // lanes are four neighbouring pieces of an even row in box w and four of
        // the odd row after it in box w ^ 1: their loads cover the two halves of
        // 128 bytes and their stores, swizzled by the row, even and odd chunks.
        const int w = warp - 8, q = lane & 3, row0 = lane >> 2, box = w ^ (row0 & 1), piece = 4 * box + q;
        const uint32_t from = row0 * HD + piece * 16;
        const uint32_t image = box * (BN * 128) + row0 * 128;
        const uint32_t at0 = image + (((2 * q) ^ row0) << 4), at1 = image + (((2 * q + 1) ^ row0) << 4);
        auto convert = [&](uint8_t *dst, int h) {
            uint4 x[8];
            const uint8_t *src = smem + L::SM_RAW + h % RAW_SLOTS * CODES_TILE + from;
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = *reinterpret_cast<const uint4 *>(src + i * 8 * HD);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const uint32_t w0 = x[i].x ^ 0x80808080u, w1 = x[i].y ^ 0x80808080u;
                const uint32_t w2 = x[i].z ^ 0x80808080u, w3 = x[i].w ^ 0x80808080u;
                *reinterpret_cast<uint4 *>(dst + at0 + i * 1024) =
                    make_uint4(fp16_codes(w0, 0x4140), fp16_codes(w0, 0x4342), fp16_codes(w1, 0x4140), fp16_codes(w1, 0x4342));
                *reinterpret_cast<uint4 *>(dst + at1 + i * 1024) =
                    make_uint4(fp16_codes(w2, 0x4140), fp16_codes(w2, 0x4342), fp16_codes(w3, 0x4140), fp16_codes(w3, 0x4342));
            }
        };
        // A tile of fp16 rows; rows past the last position and value rows in `skip` (new tokens, bits) are zero.
        auto copy_rows = [&](uint8_t *dst, const __half *rows, int j, uint32_t skip) {
            const int pos0 = (tile0 + j) * BN + row0;
#pragma unroll 4
            for (int i = 0; i < 8; ++i) {
                const int pos = pos0 + 8 * i;
                uint4 a = make_uint4(0u, 0u, 0u, 0u), b = a;
                if (pos < p.kv_rows && !(pos >= p.position && (skip >> (pos - p.position) & 1u))) {
                    const uint4 *src = reinterpret_cast<const uint4 *>(rows + ((size_t)(pos % c.ring) * NKV + kv_head) * HD + piece * 16);
                    a = src[0]; b = src[1];
                }
                *reinterpret_cast<uint4 *>(dst + at0 + i * 1024) = a;
                *reinterpret_cast<uint4 *>(dst + at1 + i * 1024) = b;
            }
        };
        auto publish = [&](uint64_t *bar) {
            fence_async_shared();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar);
        };
        for (int j = 0; j < ntiles; ++j) {
            const int s = j & 1;
            const uint32_t before = (uint32_t)((j >> 1) - 1) & 1;
            uint8_t *kd = smem + L::SM_KV + s * L::SM_KV_STAGE;
            const bool fresh = appends && (tile0 + j + 1) * BN > p.position;      // the tile holds new rows
            bool ok = true;
            for (int part = 0; part < 2 && ok; ++part) {                           // K, then V
                const int h = 2 * j + part;
                uint8_t *dst = kd + part * TILE_BYTES;
                if (j >= 2) ok = warp_wait((part ? v_empty : k_empty) + s, before, abort_flag);
                if (j < code_tiles) {
                    ok = ok && warp_wait(raw_full + h % RAW_SLOTS, (uint32_t)(h / RAW_SLOTS) & 1, abort_flag);
                    if (!ok) break;
                    convert(dst, h);
                } else {
                    ok = ok && (!fresh || warp_wait(app_done, 0, abort_flag));
                    if (!ok) break;
                    copy_rows(dst, part ? p.vc : p.kc, j, part && fresh ? *reinterpret_cast<volatile uint32_t *>(bad_values) : 0u);
                }
                publish((part ? v_full : k_full) + s);
                if (j < code_tiles && lane == 0) mbar_arrive(raw_empty + h % RAW_SLOTS);
            }
            if (!ok) break;
        }
        return;                          // the later barriers count the other eight warps
    }

    // The first tiles' codes are asked for once the query rows have arrived (issued
    // before them they would queue in front), slots 4 and 5 once they stage no queries.
    const int early = min(2 * code_tiles, 4);
    prepare_queries(p, kv_head, rope, smem + L::SM_QSTAGE, tmem, q_ready, [&] { for (int h = 0; h < early; ++h) issue_half(h); });
    if ((warp == 2 || warp == 3) && appends) {
        const int ring = c.ring;
        const uint32_t bad = append_rows<true>(p, kv_head, warp - 2, app_lo, app_hi, rope, [ring](int pos) { return pos % ring; });
        if (lane == 0 && bad) atomicOr(bad_values, bad);
        __threadfence_block();
        mbar_arrive(app_done);
    }

    if (warp == 0) {
        // ------------------------------------------------ producer
        if (lane == 0) {
            int issued = early;
            if (2 * code_tiles > early && mbar_wait(q_ready, 0, abort_flag)) {
                fence_async_shared();            // the staged queries were written and read by plain accesses
                for (int h = early; h < 2 * code_tiles; ++h) {
                    if (h >= RAW_SLOTS && !mbar_wait(raw_empty + h % RAW_SLOTS, (uint32_t)(h / RAW_SLOTS - 1) & 1, abort_flag)) break;
                    issue_half(h);
                    issued = h + 1;
                }
            }
            // Every issued copy must land before the CTA may exit.
            const long long t0 = clock64();
            for (int h = max(0, issued - RAW_SLOTS); h < issued; ++h)
                while (!mbar_try_wait(raw_full + h % RAW_SLOTS, (uint32_t)(h / RAW_SLOTS) & 1) && clock64() - t0 < WAIT_LIMIT_CYCLES) {}
        }
    } else if (warp == 1) {
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
    } else if (warp >= 4) {
        // ------------------------------------------------ softmax
        // Lanes 32w + i and 32w + 16 + i of TMEM hold the hi and lo halves of query
        // row 16w + i.  Thread l of warp w has the rows 16w + l / 4 + 8 u (u = 0,
        // 1), in each 16 of a tile's 64 columns: 8 n + 2 (l % 4) + e in x[2 n + u].
        const int wq = warp & 3;
        const uint32_t t_hi = tmem + ((uint32_t)(wq * 32) << 16), t_lo = t_hi + (16u << 16);
        const int r0 = wq * 16 + (lane >> 2), rows = p.T * GROUP;
        int last[2];                                               // last visible position
        float m_use[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
        for (int u = 0; u < 2; ++u) last[u] = r0 + 8 * u < rows ? p.position + (r0 + 8 * u) / GROUP : -1;
        auto scales_of = [&](int j, float &ks, float &vs) {
            const bool codes = j < code_tiles;
            ks = codes ? c.ks[(size_t)(tile0 + j) * NKV + kv_head] : 1.f;
            vs = codes ? c.vs[(size_t)(tile0 + j) * NKV + kv_head] : 1.f;
        };
        float ks, vs;
        scales_of(0, ks, vs);
        for (int j = 0; j < ntiles; ++j) {
            const int b = j & 1;
            const float to_log2 = SCORE_LOG2 * ks;
            // a scale of (almost) zero: its codes count nothing, its keys still do; NaN stays
            const float v_scale = vs < 0x1p-100f ? 0x1p-100f : vs;
            const float v_log2 = log2f(v_scale), v_inv = 1.f / v_scale;
            scales_of(j + 1, ks, vs);
            if (!warp_wait(s_full + b, (j >> 1) & 1, abort_flag)) break;
            tc_fence_after();
            float2 x[16];
            {
                float hi[32], lo[32];
                tmem_ld_16x256b_x8(t_hi + TM_S + b * BN, hi);
                tmem_ld_16x256b_x8(t_lo + TM_S + b * BN, lo);
                tmem_wait_ld();
#pragma unroll
                for (int q = 0; q < 16; ++q)
                    x[q] = fadd2(make_float2(hi[2 * q], hi[2 * q + 1]), make_float2(lo[2 * q], lo[2 * q + 1]));
            }
            if (j >= code_tiles) {                                 // only fp16 tiles hold positions past a query
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
            float factor[2];
            bool need = false;
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                float m0 = fmaxf(x[u].x, x[u].y), m1 = fmaxf(x[2 + u].x, x[2 + u].y);
#pragma unroll
                for (int n = 2; n < 8; n += 2) {
                    m0 = fmaxf(m0, fmaxf(x[2 * n + u].x, x[2 * n + u].y));
                    m1 = fmaxf(m1, fmaxf(x[2 * n + 2 + u].x, x[2 * n + 2 + u].y));
                }
                float m = fmaxf(m0, m1);
                m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
                m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
                m = fmaf(m, to_log2, v_log2);                      // log2 units (-inf stays -inf)
                factor[u] = 1.f;
                if (m > m_use[u] + RESCALE_THRESHOLD) {
                    factor[u] = exp2_approx(m_use[u] - m);
                    m_use[u] = m;
                    l[u] *= factor[u];
                    need = true;
                }
            }
            if (j > 0 && __any_sync(0xffffffffu, need)) {
                // O already holds tiles < j: wait for PV(j-1), then rescale its rows.
                if (!warp_wait(p_free + ((j - 1) & 1), ((j - 1) >> 1) & 1, abort_flag)) break;
                tc_fence_after();
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
            }
            uint32_t hi[16], lo[16];
            const float2 scale2 = make_float2(to_log2, to_log2), minus = make_float2(-1.f, -1.f);
            float2 shift[2], sum[2];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const float f = v_log2 + P_BIAS - (m_use[u] == -INFINITY ? 0.f : m_use[u]);
                shift[u] = make_float2(f, f);
                sum[u] = make_float2(0.f, 0.f);
            }
#pragma unroll
            for (int q = 0; q < 16; ++q) {
                const float2 arg = ffma2(x[q], scale2, shift[q & 1]);
                const float2 e = make_float2(exp2_approx(arg.x), exp2_approx(arg.y));
                sum[q & 1] = fadd2(sum[q & 1], e);
                const __half2 h = __floats2half2_rn(e.x, e.y);
                hi[q] = half2_bits(h);
                const float2 rest = ffma2(__half22float2(h), minus, e);
                lo[q] = half2_bits(__floats2half2_rn(rest.x, rest.y));
            }
#pragma unroll
            for (int u = 0; u < 2; ++u) l[u] = fmaf(sum[u].x + sum[u].y, v_inv, l[u]);
            tmem_st_16x128b_x8(t_hi + TM_S + b * BN, hi);
            tmem_st_16x128b_x8(t_lo + TM_S + b * BN, lo);
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(p_full + b);
        }
        // The rows' running max and sum, for the split combine.
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            l[u] += __shfl_xor_sync(0xffffffffu, l[u], 1);
            l[u] += __shfl_xor_sync(0xffffffffu, l[u], 2);
            if ((lane & 3) == 0 && r0 + 8 * u < rows) {
                const size_t slot = ((size_t)kv_head * DECODE_ROWS + r0 + 8 * u) * MAXS + blockIdx.x;
                p.part_ml[slot * 2] = m_use[u];
                p.part_ml[slot * 2 + 1] = l[u];
            }
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
    if (warp == 1) tmem_dealloc(tmem, 512);
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
    const DecodeParts parts = decode_parts(ws, sp);
    FaParams p{};
    p.q_gate = q_gate; p.out = out; p.T = T; p.position = position; p.kv_rows = rows;
    p.split_tiles = sp.tiles; p.splits = sp.splits;
    p.part_o = parts.o; p.part_ml = parts.ml; p.sync = parts.sync;
    p.tail = TAIL_GATED; p.world = 1;
    p.key = key; p.value = value; p.qn = qn; p.kn = kn; p.kc = k_tail; p.vc = v_tail;
    p.append_row0 = position; p.eps = eps;
    const Cache8View c{kc, vc, ks, vs, packed / CACHE8_BLOCK, ring};
    const cudaError_t e = launch_chained(attention8_kernel, dim3(sp.splits, NKV), dim3(384), A8Layout::SMEM_BYTES, st, p, c);
    if (e != cudaSuccess) throw std::runtime_error(std::string("8-bit attention: ") + cudaGetErrorString(e));
}

}  // namespace qv
