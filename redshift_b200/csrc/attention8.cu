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
//  * four converter warps read the codes straight from memory into registers (a
//    tile ahead) and write them as exact fp16 integers in the MMA's swizzled
//    operand image, so that a tile crosses shared memory only as its operands;
//  * the rest is the fp16 kernel's: queries in TMEM as fp16 hi + lo rows,
//    softmax warps with a lazily moved maximum, probabilities as fp16 hi + lo
//    rows, one CTA per (split, K/V head), the splits combined in the tail.
//
// Probabilities times the value scale: with vs = m 2^e the running maximum is
// kept over s + e (log2 units), the MMA gets m 2^(s + e - max) <= 2^9, and the
// sum adds 2^(s + e - max) 2^-e, so neither large nor small scales leave
// fp16's range.  The lo row is stored times 2^12 (its accumulator is its own
// TMEM lane), which keeps small probabilities at 2^-36 absolute.
#include "attention_core.cuh"
#include "common.cuh"
#include "hotpath.h"

#include <algorithm>
#include <stdexcept>
#include <string>

namespace qv {
namespace {

constexpr int STAGES8 = 3;       // fp16 tile images
constexpr int LO_SHIFT = 12;     // P_lo rows are stored times 2^LO_SHIFT
constexpr int CODES_TILE = BN * HD;                               // codes of one (block, head)
struct A8Layout {
    static constexpr int SM_KV = 0;                               // ring of (K, V) images
    static constexpr int SM_KV_STAGE = 2 * TILE_BYTES;
    static constexpr int SM_P = SM_KV + STAGES8 * SM_KV_STAGE;    // 2 x [128 A-rows][64 pos] fp16
    static constexpr int SM_BAR = SM_P + 2 * 128 * 128;
    static constexpr int SM_ROPE = SM_BAR + 256;                  // (cos, sin) [T][32]
    static constexpr int SMEM_BYTES = SM_ROPE + MAX_DECODE_T * 32 * 8;
};
static_assert(A8Layout::SMEM_BYTES <= 227 * 1024, "attention kernel exceeds the shared memory of a CTA");
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
__device__ __forceinline__ uint4 load_codes(const int8_t *p) {
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}

// A value scale as mant * 2^exp; a scale that is zero or not finite keeps the exponent of the tile before.
// unscale = 2^-exp.
__device__ __forceinline__ void split_scale(float vs, float &mant, float &exp, float &unscale) {
    const int e = (int)(__float_as_uint(vs) >> 23 & 255u) - 127;
    if (vs != 0.f && e <= 100) {
        exp = (float)max(e, -100);
        unscale = __int_as_float((127 - max(e, -100)) << 23);
    }
    mant = vs * unscale;
}

__global__ void __launch_bounds__(384, 1) attention8_kernel(const FaParams p, const Cache8View c) {
    using L = A8Layout;
    constexpr int SOFT_WARPS = 4, CONV_WARPS = 4;
    extern __shared__ __align__(1024) uint8_t smem[];
    if (smem_addr(smem) & 1023) {           // 128B-swizzle atoms need a 1024-byte aligned base
        if (threadIdx.x == 0) raise_status(STATUS_BAD_ARGUMENT);
        return;
    }
    uint64_t *bars = reinterpret_cast<uint64_t *>(smem + L::SM_BAR);
    uint64_t *k_full = bars, *v_full = bars + 3, *k_empty = bars + 6, *v_empty = bars + 9,
             *s_full = bars + 12, *s_free = bars + 14, *p_full = bars + 16, *p_free = bars + 18,
             *mma_done = bars + 20, *q_ready = bars + 21, *app_done = bars + 22, *cbar = bars + 23;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(smem + L::SM_BAR + 224);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(smem + L::SM_BAR + 228);
    uint32_t *bad_values = reinterpret_cast<uint32_t *>(smem + L::SM_BAR + 232);
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
        for (int i = 0; i < STAGES8; ++i) {
            mbar_init(k_full + i, CONV_WARPS); mbar_init(v_full + i, CONV_WARPS);
            mbar_init(k_empty + i, 1); mbar_init(v_empty + i, 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(s_full + i, 1); mbar_init(s_free + i, SOFT_WARPS);
            mbar_init(p_full + i, SOFT_WARPS); mbar_init(p_free + i, 1);
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
    const int wq = (warp - 4) & 3;
    const uint32_t t_lane = tmem + ((uint32_t)(wq * 32) << 16);
    const int half = lane >> 4;
    const int r = wq * 16 + (lane & 15);                                // logical query row
    int t = 0, h = 0;
    const bool valid = warp >= 4 && warp < 8 && row_token_head(p, r, t, h);

    grid_dependency_wait();
    if (threadIdx.x == 0) launch_dependents();

    if (warp >= 8) {
        // ------------------------------------------------ converters
        // Thread = 16 dims of the rows tid / 16 + 8 i of a tile: two 16-byte
        // chunks of one 64-dim box of the operand image.  Odd boxes store their
        // second chunk first, so the eight lanes of a store phase cover all banks.
        const int tid = threadIdx.x - 256, row0 = tid >> 4, piece = tid & 15;
        const uint32_t image = (piece >> 2) * (BN * 128) + row0 * 128;
        const int unit = 2 * (piece & 3), swap = piece >> 2 & 1;
        const uint32_t at0 = image + (((unit + swap) ^ (row0 & 7)) << 4);
        const uint32_t at1 = image + (((unit + 1 - swap) ^ (row0 & 7)) << 4);
        const size_t mine = (size_t)kv_head * CODES_TILE + tid * 16;
        const int packed = min(ntiles, c.blocks - tile0);               // this CTA's tiles of codes (may be negative)
        uint4 kr[8], vr[8];
        auto load = [&](const int8_t *codes, int j, uint4 (&x)[8]) {
            const int8_t *src = codes + (size_t)(tile0 + j) * (NKV * CODES_TILE) + mine;
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = load_codes(src + i * 2048);
        };
        auto convert = [&](uint8_t *dst, const uint4 (&x)[8]) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const uint32_t w0 = x[i].x ^ 0x80808080u, w1 = x[i].y ^ 0x80808080u;
                const uint32_t w2 = x[i].z ^ 0x80808080u, w3 = x[i].w ^ 0x80808080u;
                const uint4 a = make_uint4(fp16_codes(w0, 0x4140), fp16_codes(w0, 0x4342), fp16_codes(w1, 0x4140), fp16_codes(w1, 0x4342));
                const uint4 b = make_uint4(fp16_codes(w2, 0x4140), fp16_codes(w2, 0x4342), fp16_codes(w3, 0x4140), fp16_codes(w3, 0x4342));
                *reinterpret_cast<uint4 *>(dst + at0 + i * 1024) = swap ? b : a;
                *reinterpret_cast<uint4 *>(dst + at1 + i * 1024) = swap ? a : b;
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
                *reinterpret_cast<uint4 *>(dst + at0 + i * 1024) = swap ? b : a;
                *reinterpret_cast<uint4 *>(dst + at1 + i * 1024) = swap ? a : b;
            }
        };
        auto publish = [&](uint64_t *bar) {
            fence_async_shared();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar);
        };
        if (packed > 0) { load(c.kc, 0, kr); load(c.vc, 0, vr); }
        for (int j = 0; j < ntiles; ++j) {
            const int s = j % STAGES8;
            const uint32_t before = (uint32_t)(j / STAGES8 - 1) & 1;
            uint8_t *kd = smem + L::SM_KV + s * L::SM_KV_STAGE, *vd = kd + TILE_BYTES;
            const bool fresh = appends && (tile0 + j + 1) * BN > p.position;      // the tile holds new rows
            if (j >= packed && fresh && !warp_wait(app_done, 0, abort_flag)) break;
            if (j >= STAGES8 && !warp_wait(k_empty + s, before, abort_flag)) break;
            if (j < packed) convert(kd, kr);
            else copy_rows(kd, p.kc, j, 0u);
            publish(k_full + s);
            if (j + 1 < packed) load(c.kc, j + 1, kr);
            if (j >= STAGES8 && !warp_wait(v_empty + s, before, abort_flag)) break;
            if (j < packed) convert(vd, vr);
            else copy_rows(vd, p.vc, j, fresh ? *reinterpret_cast<volatile uint32_t *>(bad_values) : 0u);
            publish(v_full + s);
            if (j + 1 < packed) load(c.vc, j + 1, vr);
        }
        return;                          // the later barriers count the other eight warps
    }

    prepare_queries(p, kv_head, rope, smem + L::SM_P, tmem, q_ready, [] {});
    if ((warp == 2 || warp == 3) && appends) {
        const int ring = c.ring;
        const uint32_t bad = append_rows<true>(p, kv_head, warp - 2, app_lo, app_hi, rope, [ring](int pos) { return pos % ring; });
        if (lane == 0 && bad) atomicOr(bad_values, bad);
        __threadfence_block();
        mbar_arrive(app_done);
    }

    if (warp == 1) {
        // ------------------------------------------------ MMA issuer
        if (lane == 0) {
            const uint32_t idesc_qk = idesc_f16(128, BN, false, false);
            const uint32_t idesc_pv = idesc_f16(128, HD, false, true);
            auto issue_pv = [&](int i) -> bool {
                const int b = i & 1, s = i % STAGES8;
                if (!mbar_wait(p_full + b, (i >> 1) & 1, abort_flag)) return false;
                if (!mbar_wait(v_full + s, (i / STAGES8) & 1, abort_flag)) return false;
                tc_fence_after();
                const uint32_t pa = smem_addr(smem + L::SM_P + b * 128 * 128);
                const uint32_t vb = smem_addr(smem + L::SM_KV + s * L::SM_KV_STAGE + TILE_BYTES);
#pragma unroll
                for (int k = 0; k < BN / 16; ++k)     // P (hi / lo rows) from shared memory
                    mma_f16_ss(tmem + TM_O, sw128_desc(pa + k * 32, 16, 1024),
                               sw128_desc(vb + k * 16 * 128, BN * 128, 1024), idesc_pv, (i > 0 || k > 0) ? 1u : 0u);
                mma_commit(p_free + b);
                mma_commit(v_empty + s);
                return true;
            };
            bool ok = mbar_wait(q_ready, 0, abort_flag);
            tc_fence_after();
            for (int j = 0; j < ntiles && ok; ++j) {
                const int b = j & 1, s = j % STAGES8;
                if (!mbar_wait(k_full + s, (j / STAGES8) & 1, abort_flag)) { ok = false; break; }
                // S buffer b is reusable once the softmax has read tile j-2.
                if (j >= 2 && !mbar_wait(s_free + b, ((j >> 1) - 1) & 1, abort_flag)) { ok = false; break; }
                tc_fence_after();
                const uint32_t kb = smem_addr(smem + L::SM_KV + s * L::SM_KV_STAGE);
#pragma unroll
                for (int k = 0; k < HD / 16; ++k)
                    mma_f16_ts(tmem + TM_S + b * BN, tmem + TM_Q + k * 8,
                               sw128_desc(kb + (k >> 2) * (BN * 128) + (k & 3) * 32, 16, 1024), idesc_qk, k > 0 ? 1u : 0u);
                mma_commit(s_full + b);
                mma_commit(k_empty + s);
                if (j >= 1) ok = issue_pv(j - 1);
            }
            if (ok && ntiles > 0) issue_pv(ntiles - 1);
            // All MMAs of this thread must finish before TMEM is released.
            mma_commit(mma_done);
            const long long t0 = clock64();
            while (!mbar_try_wait(mma_done, 0) && clock64() - t0 < WAIT_LIMIT_CYCLES) {}
        }
    } else if (warp >= 4) {
        // ------------------------------------------------ softmax
        // As in the fp16 kernel: lanes i and i+16 of warp w hold the hi and lo
        // score halves of query row 16w+i and take 32 columns of the row each.
        constexpr int NC = 32;
        const int pos_limit = valid ? p.position + t : -1;         // last visible position
        const int arow_hi = wq * 32 + (lane & 15), arow_lo = arow_hi + 16;
        float m_use = -INFINITY, l = 0.f, v_exp = 0.f, v_unscale = 1.f;
        auto scales_of = [&](int j, float &ks, float &vs) {
            const bool codes = j < ntiles && tile0 + j < c.blocks;
            ks = codes ? c.ks[(size_t)(tile0 + j) * NKV + kv_head] : 1.f;
            vs = codes ? c.vs[(size_t)(tile0 + j) * NKV + kv_head] : 1.f;
        };
        float ks, vs;
        scales_of(0, ks, vs);
        for (int j = 0; j < ntiles; ++j) {
            const int b = j & 1;
            const bool codes = tile0 + j < c.blocks;
            const float to_log2 = SCORE_LOG2 * ks;
            float v_mant;
            split_scale(vs, v_mant, v_exp, v_unscale);
            scales_of(j + 1, ks, vs);
            if (!warp_wait(s_full + b, (j >> 1) & 1, abort_flag)) break;
            tc_fence_after();
            float x[64];
#pragma unroll
            for (int q = 0; q < 4; ++q)
                tmem_ld16(t_lane + TM_S + b * BN + q * 16, *reinterpret_cast<float(*)[16]>(x + q * 16));
            tmem_wait_ld();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(s_free + b);
#pragma unroll
            for (int q = 0; q < 32; ++q) {
                const float recv = __shfl_xor_sync(0xffffffffu, half ? x[q] : x[32 + q], 16);
                x[q] = (half ? x[32 + q] : x[q]) + recv;
            }
            if (!codes) {                                          // only fp16 tiles hold positions past a query
                const int key0 = (tile0 + j) * BN + half * 32;
                const int lim = pos_limit - key0;                  // columns <= lim are visible
#pragma unroll
                for (int q = 0; q < NC; ++q) x[q] = q <= lim ? x[q] : -INFINITY;
                if (appends && (tile0 + j + 1) * BN > p.position) {
                    if (!warp_wait(app_done, 0, abort_flag)) break;
                    // A new value row that is not finite was left out of the V
                    // tile (0 * NaN would reach the queries that do not see it):
                    // the queries that see it become NaN here.
                    const uint32_t bad = *reinterpret_cast<volatile uint32_t *>(bad_values);
                    if (bad) {
#pragma unroll
                        for (int q = 0; q < NC; ++q) {
                            const int age = key0 + q - p.position;
                            if (age >= 0 && age < 32 && (bad >> age & 1u) && q <= lim) x[q] = __int_as_float(0x7FC00000);
                        }
                    }
                }
            }
            float mp[8];
#pragma unroll
            for (int q = 0; q < 8; ++q) mp[q] = -INFINITY;
#pragma unroll
            for (int q = 0; q < NC; ++q) mp[q & 7] = fmaxf(mp[q & 7], x[q]);
            float m_tile = fmaxf(fmaxf(fmaxf(mp[0], mp[1]), fmaxf(mp[2], mp[3])),
                                 fmaxf(fmaxf(mp[4], mp[5]), fmaxf(mp[6], mp[7])));
            m_tile = fmaxf(m_tile, __shfl_xor_sync(0xffffffffu, m_tile, 16));
            m_tile = m_tile * to_log2 + v_exp;                     // log2 units (-inf stays -inf)
            float factor = 1.f;
            const bool need = m_tile > m_use + RESCALE_THRESHOLD;
            if (need) { factor = exp2_approx(m_use - m_tile); m_use = m_tile; l *= factor; }
            if (j > 0 && __any_sync(0xffffffffu, need)) {
                // O already holds tiles < j: wait for PV(j-1), then rescale its rows.
                if (!warp_wait(p_free + ((j - 1) & 1), ((j - 1) >> 1) & 1, abort_flag)) break;
                tc_fence_after();
#pragma unroll 1
                for (int q = 0; q < HD / 16; ++q) {
                    float o[16];
                    tmem_ld16(t_lane + TM_O + q * 16, o);
                    tmem_wait_ld();
#pragma unroll
                    for (int e = 0; e < 16; ++e) o[e] *= factor;
                    tmem_st16(t_lane + TM_O + q * 16, o);
                }
                tmem_wait_st();
            }
            const float shift = v_exp - (m_use == -INFINITY ? 0.f : m_use);
            uint32_t hi[NC / 2], lo[NC / 2];
            float sp[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int q = 0; q < NC; q += 2) {
                const float e0 = exp2_approx(fmaf(x[q], to_log2, shift)), e1 = exp2_approx(fmaf(x[q + 1], to_log2, shift));
                const float p0 = e0 * v_mant, p1 = e1 * v_mant;
                const __half2 hp = __floats2half2_rn(p0, p1);
                hi[q / 2] = half2_bits(hp);
                const float2 back = __half22float2(hp);
                constexpr float up = (float)(1 << LO_SHIFT);
                lo[q / 2] = half2_bits(__floats2half2_rn((p0 - back.x) * up, (p1 - back.y) * up));
                sp[(q >> 1) & 3] += e0 + e1;
            }
            l = fmaf((sp[0] + sp[1]) + (sp[2] + sp[3]), v_unscale, l);
            if (j >= 2 && !warp_wait(p_free + b, ((j - 2) >> 1) & 1, abort_flag)) break;
            uint8_t *pbuf = smem + L::SM_P + b * 128 * 128;
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const int unit = half * 4 + w;
                *reinterpret_cast<uint4 *>(pbuf + arow_hi * 128 + ((unit ^ (arow_hi & 7)) << 4)) =
                    make_uint4(hi[4 * w], hi[4 * w + 1], hi[4 * w + 2], hi[4 * w + 3]);
                *reinterpret_cast<uint4 *>(pbuf + arow_lo * 128 + ((unit ^ (arow_lo & 7)) << 4)) =
                    make_uint4(lo[4 * w], lo[4 * w + 1], lo[4 * w + 2], lo[4 * w + 3]);
            }
            fence_async_shared();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(p_full + b);
        }
        // The row's running max and sum, for the split combine.
        l += __shfl_xor_sync(0xffffffffu, l, 16);
        if (valid && half == 0) {
            const size_t slot = ((size_t)kv_head * DECODE_ROWS + r) * MAXS + blockIdx.x;
            p.part_ml[slot * 2] = m_use;
            p.part_ml[slot * 2 + 1] = l;
        }
    }
    // The final PV's commit on p_free marks O complete and every image consumed.
    __syncwarp();                                      // warp 1: lane 0 is back from its role
    named_barrier(5, 256);
    const bool o_ready = ntiles > 0 && warp_wait(p_free + ((ntiles - 1) & 1), ((ntiles - 1) >> 1) & 1, abort_flag);
    if (o_ready) {
        tc_fence_after();
        static_assert(EPILOGUE_BYTES <= STAGES8 * L::SM_KV_STAGE, "O staging exceeds the image ring");
        store_partials<LO_SHIFT>(p, kv_head, tmem, smem + L::SM_KV);
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 1) tmem_dealloc(tmem, 512);
    decode_tail(p, kv_head, smem + L::SM_P, reinterpret_cast<float *>(smem + L::SM_KV), cbar, abort_flag);
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
