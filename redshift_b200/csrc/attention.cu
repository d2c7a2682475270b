// Full-attention hot path for sm_100a: the decode/verify kernel (split-KV, all
// 6 GQA heads x T tokens of one KV head share every K/V tile, the prepare step
// of RMSNorm + partial RoPE + fp16 KV append folded in, the split combine or
// the peer exchange in its tail), the prepare kernel of the prefill regime
// (whose attention is prefill.cu's precise instantiation), and the shard
// merge kernel.
//
// Semantics follow the reference's attn_prepare / attention / attention_tiled
// (src/kernels.cu:415-503) and the CPU oracle tests/cpu_reference.py:55-89:
// scores q.k/16 over cache rows [0, position+t], softmax, P.V, times
// sigmoid(gate).
//
// Precision: 64 logical query rows per CTA.  Q is split into fp16 hi and
//    lo = fp16(q - hi) and the QK MMA's A operand (held in TMEM) interleaves them: A row 32w+i = Q_hi and
//    32w+16+i = Q_lo of query row 16w+i, so one M=128 MMA leaves both score
//    halves of a row in lanes i and i+16 of warp w, which add them while they
//    split the row's columns.  Every probability p is split the same way; the
//    PV MMA's A rows 32w+i / 32w+16+i are P_hi / P_lo of row 16w+i, so O_hi and
//    O_lo land in the same warp and are summed in the epilogue.  Scores and
//    probabilities keep ~22 mantissa bits (the reference computes them in fp32).
#include "attention_core.cuh"
#include "common.cuh"
#include "hotpath.h"

#include <algorithm>
#include <cuda.h>
#include <cudaTypedefs.h>
#include <stdexcept>
#include <string>

namespace qv {

constexpr int STAGES3 = 3;       // K/V tile ring depth
struct FaLayout {
    static constexpr int SM_KV = 0;                           // ring of (K tile, V tile)
    static constexpr int SM_KV_STAGE = 2 * TILE_BYTES;
    static constexpr int SM_P = SM_KV + STAGES3 * SM_KV_STAGE; // 2 x [128 A-rows][64 pos] fp16
    static constexpr int SM_BAR = SM_P + 2 * 128 * 128;       // mbarriers, TMEM address, abort flag
    static constexpr int SM_ROPE = SM_BAR + 256;              // decode: (cos, sin) [T][32]
    static constexpr int SMEM_BYTES = SM_ROPE + MAX_DECODE_T * 32 * 8;
};
static_assert(FaLayout::SMEM_BYTES <= 227 * 1024, "attention kernel exceeds the shared memory of a CTA");

__global__ void __launch_bounds__(256, 1)
fa_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
          const FaParams p) {
    using L = FaLayout;
    constexpr int SOFT_WARPS = 4;                              // softmax warps
    extern __shared__ __align__(1024) uint8_t smem[];
    if (smem_addr(smem) & 1023) {           // 128B-swizzle atoms need a 1024-byte aligned base
        if (threadIdx.x == 0) raise_status(STATUS_BAD_ARGUMENT);
        return;
    }
    if (threadIdx.x == 0) QV_STAMP(0);
    uint64_t *bars = reinterpret_cast<uint64_t *>(smem + L::SM_BAR);
    uint64_t *k_full = bars, *v_full = bars + 3, *k_empty = bars + 6, *v_empty = bars + 9,
             *s_full = bars + 12, *s_free = bars + 14, *p_full = bars + 16, *p_free = bars + 18,
             *mma_done = bars + 20, *q_ready = bars + 21, *app_done = bars + 22, *cbar = bars + 23;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(smem + L::SM_BAR + 224);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(smem + L::SM_BAR + 228);
    float2 *rope = reinterpret_cast<float2 *>(smem + L::SM_ROPE);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int kv_head = blockIdx.y;

    // KV tile range of this CTA's split (tile = 64 cache rows, local numbering).
    const int total = (p.kv_rows + BN - 1) / BN;
    const int tile0 = blockIdx.x * p.split_tiles;
    const int ntiles = min(p.split_tiles, total - tile0);
    // The block's new cache rows that fall into this CTA's tiles.
    int app_lo = 0, app_hi = 0;
    if (p.append_row0 >= 0) {
        app_lo = max(p.append_row0, tile0 * BN);
        app_hi = min(p.append_row0 + p.T, (tile0 + ntiles) * BN);
    }
    const bool appends = app_hi > app_lo;
    const int app_tile = appends ? app_lo / BN - tile0 : ntiles;    // first tile holding a new row

    // Before anything else: L2 prefetch hints for this CTA's query rows (the
    // q half of q_gate), so that their HBM latency overlaps the previous
    // kernel's tail.  (Prefetching K/V tiles as well measured slower: the
    // extra traffic delays the query loads and thrashes L2.)
    for (int i = threadIdx.x; i < p.T * GROUP * 8; i += blockDim.x) {    // 8 lines of 128 B per row
        const int rr = i >> 3;
        prefetch_l2(p.q_gate + ((size_t)(rr / GROUP) * NQ + kv_head * GROUP + rr % GROUP) * 2 * HD + (i & 7) * 32);
    }

    if (threadIdx.x == 0) {
        for (int i = 0; i < STAGES3; ++i) {
            mbar_init(k_full + i, 1); mbar_init(v_full + i, 1);
            mbar_init(k_empty + i, 1); mbar_init(v_empty + i, 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(s_full + i, 1); mbar_init(s_free + i, SOFT_WARPS);
            mbar_init(p_full + i, SOFT_WARPS); mbar_init(p_free + i, 1);
        }
        mbar_init(mma_done, 1);
        mbar_init(q_ready, 8);                     // every warp, once its query rows are in TMEM
        mbar_init(cbar, 1);
        mbar_init(app_done, 64);
        *abort_flag = 0;
        fence_barrier_init();
    }
    if (warp == 0 && lane == 0) { prefetch_tmap(&tmK); prefetch_tmap(&tmV); }
    if (warp == 1) { tmem_alloc(tmem_slot, 512); tmem_relinquish(); }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;

    // Softmax warps 4-7: thread = TMEM lane = A row of the QK MMA; lanes i and
    // i+16 of warp w carry the hi and lo halves of query row 16w+i (one M=128
    // MMA yields both).
    const int wq = (warp - 4) & 3;
    const uint32_t t_lane = tmem + ((uint32_t)(wq * 32) << 16);
    const int half = lane >> 4;
    const int r = wq * 16 + (lane & 15);                                // logical query row
    int t = 0, h = 0;
    const bool valid = warp >= 4 && row_token_head(p, r, t, h);

    // Everything below may read what the previous kernel of the stream wrote.
    grid_dependency_wait();
    if (threadIdx.x == 0) { launch_dependents(); QV_STAMP(1); }

    // The query rows and norm weights are loaded first (from L2, ahead of the
    // bulk K/V data, which would otherwise queue in front of them on the way
    // into the SM); once every warp's rows have arrived, tiles 0..2 (all
    // three stages) go out, unless they hold new rows, which must be written
    // first, and the preparation overlaps their loads.
    const int early = min(ntiles, min(app_tile, STAGES3));
    auto issue_early = [&](int j0, int j1) {
        for (int j = j0; j < j1; ++j) {
            uint8_t *kd = smem + L::SM_KV + j * L::SM_KV_STAGE, *vd = kd + TILE_BYTES;
            const int y = (tile0 + j) * BN;
            mbar_expect_tx(k_full + j, TILE_BYTES);
            for (int c = 0; c < 4; ++c) tma_load_2d(kd + c * BN * 128, &tmK, k_full + j, kv_head * HD + c * 64, y);
            mbar_expect_tx(v_full + j, TILE_BYTES);
            for (int c = 0; c < 4; ++c) tma_load_2d(vd + c * BN * 128, &tmV, v_full + j, kv_head * HD + c * 64, y);
        }
        QV_STAMP(2);
    };
    prepare_queries(p, kv_head, rope, smem + L::SM_P, tmem, q_ready, [&] { issue_early(0, early); });
    if ((warp == 2 || warp == 3) && appends) {
        // The new rows become visible to the TMA loads of this CTA.
        append_rows(p, kv_head, warp - 2, app_lo, app_hi, rope);
        fence_async_global();
        mbar_arrive(app_done);
    }

    if (warp == 0) {
        // ------------------------------------------------ TMA producer
        // K tiles are released after QK, V tiles after PV, so the next K load
        // overlaps the softmax and PV of the current tile.
        if (lane == 0) {
            int k_issued = early, v_issued = early;        // tiles issued before the query preparation
            for (int j = early; j < ntiles; ++j) {
                const int s = j % STAGES3;
                const uint32_t use = (uint32_t)(j / STAGES3);
                const int y = (tile0 + j) * BN;
                uint8_t *kd = smem + L::SM_KV + s * L::SM_KV_STAGE, *vd = kd + TILE_BYTES;
                if (j == app_tile && !mbar_wait(app_done, 0, abort_flag)) break;   // new rows written
                if (j >= STAGES3 && !mbar_wait(k_empty + s, (use - 1) & 1, abort_flag)) break;
                mbar_expect_tx(k_full + s, TILE_BYTES);
                for (int c = 0; c < 4; ++c) tma_load_2d(kd + c * BN * 128, &tmK, k_full + s, kv_head * HD + c * 64, y);
                k_issued = j + 1;
                if (j >= STAGES3 && !mbar_wait(v_empty + s, (use - 1) & 1, abort_flag)) break;
                mbar_expect_tx(v_full + s, TILE_BYTES);
                for (int c = 0; c < 4; ++c) tma_load_2d(vd + c * BN * 128, &tmV, v_full + s, kv_head * HD + c * 64, y);
                v_issued = j + 1;
            }
            QV_STAMP(9);
            // Drain: every issued load must land before the CTA may exit.
            const long long t0 = clock64();
            for (int j = max(0, k_issued - STAGES3); j < k_issued; ++j)
                while (!mbar_try_wait(k_full + j % STAGES3, (j / STAGES3) & 1) && clock64() - t0 < WAIT_LIMIT_CYCLES) {}
            for (int j = max(0, v_issued - STAGES3); j < v_issued; ++j)
                while (!mbar_try_wait(v_full + j % STAGES3, (j / STAGES3) & 1) && clock64() - t0 < WAIT_LIMIT_CYCLES) {}
        }
    } else if (warp == 1) {
        // ------------------------------------------------ MMA issuer
        if (lane == 0) {
            const uint32_t idesc_qk = idesc_f16(128, BN, false, false);
            const uint32_t idesc_pv = idesc_f16(128, HD, false, true);
            auto issue_pv = [&](int i) -> bool {
                const int b = i & 1, s = i % STAGES3;
                if (!mbar_wait(p_full + b, (i >> 1) & 1, abort_flag)) return false;
                if (!mbar_wait(v_full + s, (i / STAGES3) & 1, abort_flag)) return false;
                tc_fence_after();
                const uint32_t pa = smem_addr(smem + L::SM_P + b * 128 * 128);
                const uint32_t vb = smem_addr(smem + L::SM_KV + s * L::SM_KV_STAGE + TILE_BYTES);
#pragma unroll
                for (int k = 0; k < BN / 16; ++k)     // P (hi / lo rows) from shared memory
                    mma_f16_ss(tmem + TM_O, sw128_desc(pa + k * 32, 16, 1024),
                               sw128_desc(vb + k * 16 * 128, BN * 128, 1024), idesc_pv,
                               (i > 0 || k > 0) ? 1u : 0u);
                mma_commit(p_free + b);
                mma_commit(v_empty + s);
                return true;
            };
            bool ok = mbar_wait(q_ready, 0, abort_flag);
            tc_fence_after();
            for (int j = 0; j < ntiles && ok; ++j) {
                const int b = j & 1, s = j % STAGES3;
                if (!mbar_wait(k_full + s, (j / STAGES3) & 1, abort_flag)) { ok = false; break; }
                // S buffer b is reusable once the softmax has read tile j-2.
                if (j >= 2 && !mbar_wait(s_free + b, ((j >> 1) - 1) & 1, abort_flag)) { ok = false; break; }
                tc_fence_after();
                const uint32_t kb = smem_addr(smem + L::SM_KV + s * L::SM_KV_STAGE);
#pragma unroll
                for (int k = 0; k < HD / 16; ++k)
                    mma_f16_ts(tmem + TM_S + b * BN, tmem + TM_Q + k * 8,
                               sw128_desc(kb + (k >> 2) * (BN * 128) + (k & 3) * 32, 16, 1024),
                               idesc_qk, k > 0 ? 1u : 0u);
                mma_commit(s_full + b);
                mma_commit(k_empty + s);
                if (j >= 1) ok = issue_pv(j - 1);
            }
            if (ok && ntiles > 0) issue_pv(ntiles - 1);
            QV_STAMP(10);
            // All MMAs of this thread must finish before TMEM is released.
            mma_commit(mma_done);
            const long long t0 = clock64();
            while (!mbar_try_wait(mma_done, 0) && clock64() - t0 < WAIT_LIMIT_CYCLES) {}
        }
    } else if (warp >= 4) {
        // ------------------------------------------------ softmax + epilogue
        // Each thread handles 32 columns of its row per tile: lane i keeps
        // columns [0,32) and lane i+16 columns [32,64) of row 16w+i, each summing
        // the hi and lo score halves, and each writes the hi and lo
        // probabilities of its columns.
        constexpr int NC = 32;                                     // columns per thread
        const int cpart = half;                                    // which 32 columns
        const int pos_limit = valid ? p.position + t - p.kv_begin : -1;   // last visible local row
        const int arow_hi = wq * 32 + (lane & 15);                 // A rows of P (hi, lo)
        const int arow_lo = arow_hi + 16;
        float m_use = -INFINITY, l = 0.f;
        for (int j = 0; j < ntiles; ++j) {
            const int b = j & 1;
            if (!warp_wait(s_full + b, (j >> 1) & 1, abort_flag)) break;
            if (j == 0 && threadIdx.x == 128) QV_STAMP(4);
            tc_fence_after();
            float x[64];
#pragma unroll
            for (int c = 0; c < 4; ++c)
                tmem_ld16(t_lane + TM_S + b * BN + c * 16, *reinterpret_cast<float(*)[16]>(x + c * 16));
            tmem_wait_ld();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(s_free + b);
#pragma unroll
            for (int c = 0; c < 32; ++c) {
                const float recv = __shfl_xor_sync(0xffffffffu, half ? x[c] : x[32 + c], 16);
                x[c] = (half ? x[32 + c] : x[c]) + recv;
            }
            const int key0 = (tile0 + j) * BN + cpart * 32;
            const int lim = min(pos_limit, p.kv_rows - 1) - key0;     // columns <= lim are visible
            // Row max and (below) row sum over 8 / 4 independent partials, so
            // neither is one long dependent chain.
            float mp[8];
#pragma unroll
            for (int q = 0; q < 8; ++q) mp[q] = -INFINITY;
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                x[c] = c <= lim ? x[c] : -INFINITY;
                mp[c & 7] = fmaxf(mp[c & 7], x[c]);
            }
            float m_tile = fmaxf(fmaxf(fmaxf(mp[0], mp[1]), fmaxf(mp[2], mp[3])),
                                 fmaxf(fmaxf(mp[4], mp[5]), fmaxf(mp[6], mp[7])));
            m_tile = fmaxf(m_tile, __shfl_xor_sync(0xffffffffu, m_tile, 16));
            m_tile *= SCORE_LOG2;                                  // log2 units (-inf stays -inf)
            float factor = 1.f;
            const bool need = m_tile > m_use + RESCALE_THRESHOLD;
            if (need) { factor = exp2_approx(m_use - m_tile); m_use = m_tile; l *= factor; }
            if (j > 0 && __any_sync(0xffffffffu, need)) {
                // O already holds tiles < j: wait for PV(j-1), then rescale rows in
                // TMEM.
                if (!warp_wait(p_free + ((j - 1) & 1), ((j - 1) >> 1) & 1, abort_flag)) break;
                tc_fence_after();
#pragma unroll 1
                for (int c = 0; c < HD / 16; ++c) {
                    float o[16];
                    tmem_ld16(t_lane + TM_O + c * 16, o);
                    tmem_wait_ld();
#pragma unroll
                    for (int e = 0; e < 16; ++e) o[e] *= factor;
                    tmem_st16(t_lane + TM_O + c * 16, o);
                }
                tmem_wait_st();
            }
            const float mref = m_use == -INFINITY ? 0.f : m_use;
            uint32_t hi[NC / 2], lo[NC / 2];
            float sp[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int c = 0; c < NC; c += 2) {
                const float p0 = exp2_approx(fmaf(x[c], SCORE_LOG2, -mref));
                const float p1 = exp2_approx(fmaf(x[c + 1], SCORE_LOG2, -mref));
                const __half2 hp = __floats2half2_rn(p0, p1);
                hi[c / 2] = *reinterpret_cast<const uint32_t *>(&hp);
                const float2 back = __half22float2(hp);
                const __half2 lp = __floats2half2_rn(p0 - back.x, p1 - back.y);
                lo[c / 2] = *reinterpret_cast<const uint32_t *>(&lp);
                sp[(c >> 1) & 3] += p0 + p1;
            }
            l += (sp[0] + sp[1]) + (sp[2] + sp[3]);
            if (j >= 2 && !warp_wait(p_free + b, ((j - 2) >> 1) & 1, abort_flag)) break;
            uint8_t *pbuf = smem + L::SM_P + b * 128 * 128;
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const int unit = cpart * 4 + w;
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
        if (threadIdx.x == 128) QV_STAMP(5);
        // The row's running max and sum, for the split combine.
        l += __shfl_xor_sync(0xffffffffu, l, 16);
        if (valid && half == 0) {
            const size_t slot = ((size_t)kv_head * DECODE_ROWS + r) * MAXS + blockIdx.x;
            p.part_ml[slot * 2] = m_use;
            p.part_ml[slot * 2 + 1] = l;
        }
    }
    // ------------------------------------------------ epilogue (all 8 warps)
    // The final PV's commit on p_free marks O complete (and every K/V tile
    // consumed, so the ring is idle).  Warps w and w+4 share TMEM lane
    // quarter w%4 (O_hi of row 16(w%4)+i in lane i, O_lo in lane 16+i) and
    // take O columns [0,128) (warps 4-7) and [128,256) (warps 0-3): each lane
    // puts its lane's columns into a padded staging row, then the warp
    // stores each of its rows, the sum of its hi and lo staging rows, as
    // 512-byte pieces of this split's unnormalised partial.
    __syncwarp();                                      // warps 0 and 1: lane 0 is back from its role
    named_barrier(5, 256);
    const bool o_ready = ntiles > 0 &&
                         warp_wait(p_free + ((ntiles - 1) & 1), ((ntiles - 1) >> 1) & 1, abort_flag);
    if (o_ready) {
        tc_fence_after();
        static_assert(EPILOGUE_BYTES <= STAGES3 * L::SM_KV_STAGE, "O staging exceeds the K/V ring");
        store_partials(p, kv_head, tmem, smem + L::SM_KV);
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 1) tmem_dealloc(tmem, 512);
    if (threadIdx.x == 0) QV_STAMP(11);
    // The split combine of this CTA's share of the KV head's rows (the K/V
    // ring and the P buffers are idle now; the P region is scratch).
    decode_tail(p, kv_head, smem + L::SM_P, reinterpret_cast<float *>(smem + L::SM_KV), cbar, abort_flag);
}

// ---------------------------------------------------------------- prepare
// One block per token, 8 warps; warp w prepares rows w, w+8, w+16 (and w+24)
// of the token's 28: the 24 query heads, then the 4 key heads.  RMSNorm with
// weight, rotary embedding on dims [0,64) as pairs (i, i+32) with angle
// (position+t) * 1e7^(-i/32) evaluated in double precision (the token's 32
// angles once per block), queries written as fp16 hi / lo operand rows,
// keys / values rounded to fp16 into the cache.  Lane l of a row holds dims
// [4l,4l+4) and [128+4l,128+4l+4), as in the decode kernel's prepare step.
// Used by the prefill regime; decode batches fold this step into fa_kernel.
__global__ void __launch_bounds__(256)
attn_prepare_kernel(const float *q_gate, const float *key, const float *value, const float *qn,
                    const float *kn, __half *qw, __half *qw_lo, __half *kc, __half *vc, int position,
                    int append_row0, float eps) {
    constexpr int ROWS = NQ + NKV, RPW = (ROWS + 7) / 8;          // rows per token, per warp
    const int t = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    __shared__ float2 cs[32];
    grid_dependency_wait();
    launch_dependents();
    float4 a[RPW], b[RPW];
#pragma unroll
    for (int j = 0; j < RPW; ++j) {
        const int h = warp + 8 * j;
        if (h < ROWS) {
            const float *src = h < NQ ? q_gate + ((size_t)t * NQ + h) * 2 * HD : key + ((size_t)t * NKV + h - NQ) * HD;
            a[j] = *reinterpret_cast<const float4 *>(src + 4 * lane);
            b[j] = *reinterpret_cast<const float4 *>(src + 128 + 4 * lane);
        }
    }
    if (threadIdx.x < 32) cs[threadIdx.x] = rope_angle(position + t, threadIdx.x);
    __syncthreads();
#pragma unroll
    for (int j = 0; j < RPW; ++j) {
        const int h = warp + 8 * j;
        if (h >= ROWS) continue;
        const bool isq = h < NQ;
        const float *nw = isq ? qn : kn;
        const float4 n0 = *reinterpret_cast<const float4 *>(nw + 4 * lane);
        const float4 n1 = *reinterpret_cast<const float4 *>(nw + 128 + 4 * lane);
        const float4 u = a[j], v = b[j];
        const float ss = warp_sum(u.x * u.x + u.y * u.y + u.z * u.z + u.w * u.w + v.x * v.x + v.y * v.y +
                                  v.z * v.z + v.w * v.w);
        const float inv = rsqrtf(ss / HD + eps);
        float x0[4] = {u.x * inv * n0.x, u.y * inv * n0.y, u.z * inv * n0.z, u.w * inv * n0.w};
        const float x1[4] = {v.x * inv * n1.x, v.y * inv * n1.y, v.z * inv * n1.z, v.w * inv * n1.w};
        rope_row(x0, cs, lane, true);
        if (isq) {
            __half *hi = qw + ((size_t)t * NQ + h) * HD, *lo = qw_lo + ((size_t)t * NQ + h) * HD;
#pragma unroll
            for (int part = 0; part < 2; ++part) {
                const float *x = part ? x1 : x0;
                const __half2 h0 = __floats2half2_rn(x[0], x[1]), h1 = __floats2half2_rn(x[2], x[3]);
                const float2 f0 = __half22float2(h0), f1 = __half22float2(h1);
                *reinterpret_cast<uint2 *>(hi + part * 128 + 4 * lane) = make_uint2(half2_bits(h0), half2_bits(h1));
                *reinterpret_cast<uint2 *>(lo + part * 128 + 4 * lane) =
                    make_uint2(half2_bits(__floats2half2_rn(x[0] - f0.x, x[1] - f0.y)),
                               half2_bits(__floats2half2_rn(x[2] - f1.x, x[3] - f1.y)));
            }
        } else if (append_row0 >= 0) {
            const int kh = h - NQ;
            const size_t o = ((size_t)(append_row0 + t) * NKV + kh) * HD;
            const float *vs = value + ((size_t)t * NKV + kh) * HD;
            const float4 va = *reinterpret_cast<const float4 *>(vs + 4 * lane);
            const float4 vb = *reinterpret_cast<const float4 *>(vs + 128 + 4 * lane);
            *reinterpret_cast<uint2 *>(kc + o + 4 * lane) =
                make_uint2(half2_bits(__floats2half2_rn(x0[0], x0[1])), half2_bits(__floats2half2_rn(x0[2], x0[3])));
            *reinterpret_cast<uint2 *>(kc + o + 128 + 4 * lane) =
                make_uint2(half2_bits(__floats2half2_rn(x1[0], x1[1])), half2_bits(__floats2half2_rn(x1[2], x1[3])));
            *reinterpret_cast<uint2 *>(vc + o + 4 * lane) =
                make_uint2(half2_bits(__floats2half2_rn(va.x, va.y)), half2_bits(__floats2half2_rn(va.z, va.w)));
            *reinterpret_cast<uint2 *>(vc + o + 128 + 4 * lane) =
                make_uint2(half2_bits(__floats2half2_rn(vb.x, vb.y)), half2_bits(__floats2half2_rn(vb.z, vb.w)));
        }
    }
}

// Merge per-GPU shard partials (normalised O, natural-log LSE) into the gated
// output: O = sum_g exp(lse_g - LSE) O_g, times sigmoid(gate).
__global__ void __launch_bounds__(256)
attn_merge_kernel(float *out, const float *parts, const float *lses, int shards, int T,
                  const float *q_gate) {
    const int t = blockIdx.x / NQ, h = blockIdx.x % NQ, d = threadIdx.x;
    const size_t row = (size_t)t * NQ + h, stride_o = (size_t)T * NQ * HD, stride_l = (size_t)T * NQ;
    grid_dependency_wait();
    launch_dependents();
    float M = -INFINITY;
    for (int g = 0; g < shards; ++g) M = fmaxf(M, lses[g * stride_l + row]);
    float num = 0.f, den = 0.f;
    if (M != -INFINITY)
        for (int g = 0; g < shards; ++g) {
            const float L = lses[g * stride_l + row];
            if (L == -INFINITY) continue;
            const float w = expf(L - M);
            den += w;
            num += w * parts[g * stride_o + row * HD + d];
        }
    out[row * HD + d] = (den > 0.f ? num / den : 0.f) * sigmoidf_(q_gate[row * 2 * HD + HD + d]);
}

// ======================================================================= host
namespace {
PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
    static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
    if (!fn) {
        cudaDriverEntryPointQueryResult q;
        void *ptr = nullptr;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) != cudaSuccess ||
            q != cudaDriverEntryPointSuccess || !ptr)
            throw std::runtime_error("cuTensorMapEncodeTiled is unavailable");
        fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(ptr);
    }
    return fn;
}

// 2-D map over a [rows][4*256] fp16 cache: box = 64 dims x 64 rows, 128B swizzle.
CUtensorMap cache_map(const void *base, int rows) {
    CUtensorMap m;
    cuuint64_t dims[2] = {(cuuint64_t)NKV * HD, (cuuint64_t)rows};
    cuuint64_t strides[1] = {(cuuint64_t)NKV * HD * sizeof(__half)};
    cuuint32_t box[2] = {64, (cuuint32_t)BN};
    cuuint32_t estr[2] = {1, 1};
    const CUresult r = encode_fn()(&m, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, const_cast<void *>(base), dims,
                                   strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                                   CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                                   CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) throw std::runtime_error("cuTensorMapEncodeTiled failed: " + std::to_string((int)r));
    return m;
}

// The shared-memory limit of a kernel is a per-device attribute: set it on
// every device the process launches on.
PerDeviceOnce g_configured;
void configure() {
    g_configured.run([] {
        if (cudaFuncSetAttribute(fa_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, FaLayout::SMEM_BYTES) !=
            cudaSuccess)
            throw std::runtime_error("cannot reserve shared memory for the attention kernel");
    });
}

void launch_fa(const CUtensorMap &mk, const CUtensorMap &mv, const FaParams &p, dim3 grid, cudaStream_t st) {
    const cudaError_t e = launch_chained(fa_kernel, grid, dim3(256), FaLayout::SMEM_BYTES, st,
                                         mk, mv, p);
    if (e != cudaSuccess) throw std::runtime_error(std::string("attention kernel launch: ") + cudaGetErrorString(e));
}


// Split-KV decode / verify, one launch: the CTAs normalise and rotate the
// queries, append the new keys / values (when `append`), attend over their
// split, and at the tail combine the splits and write the rows as `tail`
// says (out = gated output, or shard partial with lse, or the peer exchange).
void launch_decode(float *out, float *lse, __half *kc, __half *vc, const float *q_gate, const float *key,
                   const float *value, const float *qn, const float *kn, int T, int position, int kv_begin,
                   int kv_rows, bool append, float eps, void *ws, size_t ws_bytes, DecodeTail tail,
                   const uint64_t *peers, int world, int rank, int seq, cudaStream_t st) {
    configure();
    const Split sp = decode_split(kv_rows);
    if (ws_bytes < decode_parts_bytes(sp)) throw std::invalid_argument("attention workspace too small");
    const DecodeParts parts = decode_parts(ws, sp);
    const CUtensorMap mk = cache_map(kc, kv_rows), mv = cache_map(vc, kv_rows);
    FaParams p{};
    p.q_gate = q_gate; p.out = out; p.lse = lse; p.T = T; p.position = position; p.kv_begin = kv_begin;
    p.kv_rows = kv_rows; p.split_tiles = sp.tiles; p.splits = sp.splits;
    p.part_o = parts.o; p.part_ml = parts.ml; p.sync = parts.sync;
    p.tail = tail; p.peers = peers; p.world = world; p.rank = rank; p.seq = seq;
    p.key = key; p.value = value; p.qn = qn; p.kn = kn; p.kc = kc; p.vc = vc;
    p.append_row0 = append ? position - kv_begin : -1; p.eps = eps;
    launch_fa(mk, mv, p, dim3(sp.splits, NKV), st);
}
}  // namespace

size_t attention_workspace_bytes(int T, int kv_rows) {
    if (decode_regime(T)) return decode_parts_bytes(decode_split(kv_rows));
    return 2 * align256((size_t)T * NQ * HD * sizeof(__half));     // prefill: Q hi and lo, direct output
}

int attention_max_shard_batch() { return MAX_DECODE_T; }

// One attention layer over a device cache holding absolute positions
// [kv_begin, kv_begin + kv_rows).  New rows are appended at local row
// position - kv_begin when append is true.  Writes either the final gated
// output (shard_lse == nullptr) or a normalised partial + LSE (shard mode).
// Decode / verify batches (T <= 10) use the split-KV regime (one launch, the
// split combine in its tail); longer blocks use the prefill regime: a prepare
// launch, then prefill.cu's precise kernel (128 queries per CTA, 128-key tiles).
void attention_run(float *out, float *shard_lse, __half *kc, __half *vc, const float *q_gate,
                   const float *key, const float *value, const float *qn, const float *kn, int T,
                   int position, int kv_begin, int kv_rows, bool append, float eps, void *ws,
                   size_t ws_bytes, cudaStream_t st) {
    if (ws_bytes < attention_workspace_bytes(T, kv_rows)) throw std::invalid_argument("attention workspace too small");
    if (decode_regime(T)) {
        launch_decode(out, shard_lse, kc, vc, q_gate, key, value, qn, kn, T, position, kv_begin, kv_rows, append, eps,
                      ws, ws_bytes, shard_lse ? TAIL_SHARD : TAIL_GATED, nullptr, 1, 0, 0, st);
        return;
    }
    if (shard_lse) throw std::invalid_argument("shard partials are limited to decode batches");
    configure();
    uint8_t *w = static_cast<uint8_t *>(ws);
    const size_t q_bytes = align256((size_t)T * NQ * HD * sizeof(__half));
    __half *qw = reinterpret_cast<__half *>(w), *qw_lo = reinterpret_cast<__half *>(w + q_bytes);
    const cudaError_t e = launch_chained(attn_prepare_kernel, dim3(T), dim3(256), 0, st, q_gate, key, value,
                                         qn, kn, qw, qw_lo, kc, vc, position, append ? position - kv_begin : -1, eps);
    if (e != cudaSuccess) throw std::runtime_error(std::string("attention prepare: ") + cudaGetErrorString(e));
    prefill_precise(out, qw, qw_lo, q_gate, kc, vc, T, position - kv_begin, kv_rows, st);
}

size_t attention_exchange_bytes(int world) { return ex_bytes(world); }
int attention_exchange_max_world() { return EX_MAX_WORLD; }

// Shard attention + all-to-all exchange + merge, one launch (the exchange is
// the decode kernel's tail, see exchange_rows).
void attention_shard_exchange(float *out, __half *kc, __half *vc, const float *q_gate, const float *key,
                              const float *value, const float *qn, const float *kn, int T, int position,
                              int kv_begin, int kv_rows, bool append, float eps, const uint64_t *peers,
                              int world, int rank, int seq, void *ws, size_t ws_bytes, cudaStream_t st) {
    if (!decode_regime(T)) throw std::invalid_argument("the exchange supports decode batches only");
    if (world < 1 || world > EX_MAX_WORLD || rank < 0 || rank >= world || seq < 0)
        throw std::invalid_argument("invalid exchange group");
    if (ws_bytes < attention_workspace_bytes(T, kv_rows)) throw std::invalid_argument("attention workspace too small");
    launch_decode(out, nullptr, kc, vc, q_gate, key, value, qn, kn, T, position, kv_begin, kv_rows, append, eps, ws,
                  ws_bytes, TAIL_EXCHANGE, peers, world, rank, seq, st);
}

void attention_merge(float *out, const float *parts, const float *lses, int shards, int T,
                     const float *q_gate, cudaStream_t st) {
    const cudaError_t e = launch_chained(attn_merge_kernel, dim3(T * NQ), dim3(256), 0, st, out, parts, lses, shards,
                                         T, q_gate);
    if (e != cudaSuccess) throw std::runtime_error(std::string("attention merge: ") + cudaGetErrorString(e));
}

}  // namespace qv
