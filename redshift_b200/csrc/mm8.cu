// Matrix product of e4m3 codes with block scales (sm_100a tcgen05, kind::f8f6f4):
//   out[t][r] = sum over blocks b of 128 columns of
//               weight_scale[r / 128][b] * scale[b][t] * sum_{k in b} W[r][k] X[t][k]
// for weights W [rows][width], activations X [tokens][width] and fp32 scales.
//
// Every block's sum of 128 products leaves the tensor core as fp32 and is
// multiplied by the product of its two scales and added in fp32 registers, so a long
// width costs no precision (the products of one block are exact in the accumulator's
// alignment for codes of like size).  The scales may be any fp32 values: outputs
// with a product of scales that leaves fp32's normal range are computed anew
// (again_in_range).
//
// Two kernels:
//  * few_kernel<NT> (tokens as the MMA's N, 16..128 of them): 128 weight rows
//    per CTA.  Up to 16 tokens bound by reading the weights once from HBM (8 tokens x
//    5,120 x 17,408: 17.7 us, 5.0 TB/s; 1 x 6,144 x 5,120, 31 MB, 9.9 us), at 128 by the
//    way of the sums out of TMEM (128 x 5,120 x 10,240: 24.0 us); the width is split
//    over a cluster of up to six CTAs whose partial sums meet in distributed
//    shared memory in a fixed order, so that also few rows fill the SMs and no
//    workspace or atomics are needed.
//  * many_kernel (128 tokens as the MMA's M, 256 weight rows as its N): persistent
//    CTAs.  With tokens in the TMEM lanes the two scales of a thread's columns are
//    one factor per block.  Bound by the way of a block's sums out of TMEM, see
//    there (4,001 x 5,120 x 17,408: 368-410 us, up to 1.9 PFLOP/s; in calls without a
//    pause the power limit holds the SMs at 1.3-1.5 GHz, 425-455 us; 1,000 x 5,120 x
//    10,240 71 us).
#include "common.cuh"
#include "hotpath.h"

#include <algorithm>
#include <stdexcept>
#include <string>

namespace qv {
namespace {

constexpr int KB = 128;                        // columns of a block = one 128-byte swizzled row of codes
constexpr int ROWS = 128;                      // weight rows that share a scale
constexpr int MAX_SPLITS = 6;                  // CTAs of a few_kernel cluster

// D[tmem] (+)= A[smem] * B[smem]^T for e4m3 codes, fp32 accumulate, K = 32;
// issued by a whole warp, one elected lane (see mma_f16_ts_by).
__device__ __forceinline__ void mma_e4m3_ss_by(uint32_t elected, uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc,
                                               uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p, q;\n\t"
                 "setp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
                 "@q tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
                 :: "r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate), "r"(elected) : "memory");
}
// Instruction descriptor: e4m3 operands (format 0 of kind::f8f6f4), both K-major, fp32 accumulator.
__host__ __device__ constexpr uint32_t idesc_e4m3(int M, int N) {
    return (1u << 4) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}
// Asynchronous copy of one float into shared memory, zero when !live.
__device__ __forceinline__ void copy_float(float *dst, const float *src, bool live) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;"
                 :: "r"(smem_addr(dst)), "l"(src), "r"(live ? 4 : 0) : "memory");
}
// Arrive on `bar` (counted in its initial count) once this thread's copies have landed.
__device__ __forceinline__ void arrive_copies(uint64_t *bar) {
    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" :: "r"(smem_addr(bar)) : "memory");
}
// The box of `map` at (x, y) on its way into L2.
__device__ __forceinline__ void prefetch_l2_2d(const CUtensorMap *map, int x, int y) {
    asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global.tile [%0, {%1, %2}];" :: "l"(map), "r"(x), "r"(y) : "memory");
}
__device__ __forceinline__ bool warp_wait8(uint64_t *bar, uint32_t parity, volatile int *abort_flag) {
    return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag));
}
// The values of four e4m3 codes.
__device__ __forceinline__ void e4m3_values(uint32_t codes, float (&v)[4]) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        uint32_t h;
        asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((unsigned short)(codes >> (16 * i))));
        const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&h));
        v[2 * i] = f.x;
        v[2 * i + 1] = f.y;
    }
}
__device__ __forceinline__ float ld_cluster_f32(uint32_t addr) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
    return v;
}
// The shared address of this CTA's `addr` in CTA `rank` of the cluster.
__device__ __forceinline__ uint32_t cluster_rank(uint32_t addr, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
__device__ __forceinline__ float4 ld_cluster_f32x4(uint32_t addr) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
    return v;
}
// Every lane of the cluster's CTAs.  The aligned form wants a warp's lanes together, and
// the code before it branches on the lane.
__device__ __forceinline__ void cluster_sync() {
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

struct Mm8Params {
    float *out;
    const float *weight_scales, *scales;
    const uint8_t *weights, *codes;
    int tokens, rows, width, blocks;           // blocks = ceil(width / 128)
    int splits;                                // cluster size (few_kernel)
    int m_tiles, tiles;                        // many_kernel: token tiles, all tiles
};

// ---------------------------------------------------------------- scales whose product leaves fp32
// A product a b that is infinite or below 2^-126 although a and b are neither.
__device__ __forceinline__ bool leaves_range(float a, float b) {
    const float size = fabsf(a * b);
    return !(size >= 0x1p-126f && size < INFINITY) && a != 0.f && b != 0.f && fabsf(a) < INFINITY && fabsf(b) < INFINITY;
}
// The range of scales that were looked at, zeros apart: bit patterns without the sign,
// times two.  Two scales inside [2^-63, 2^63) have a normal product.
struct ScaleRange {
    uint32_t most = 0u, least = 0xFFFFFFFFu;                 // the largest; the smallest, less one, so that zero is the largest of all
    __device__ __forceinline__ void add(float a) {
        const uint32_t size = 2u * __float_as_uint(a);
        most = max(most, size);
        least = min(least, size - 1u);
    }
    __device__ __forceinline__ void add(float4 a) { add(a.x); add(a.y); add(a.z); add(a.w); }
    __device__ __forceinline__ bool far() const { return most >= 2u * 0x5F000000u || least < 2u * 0x20000000u - 1u; }
};
// The outputs of `token` and the 128 rows of `row_block`, by one warp, if one of their
// products of scales leaves fp32's normal range.  The factor a b of a block's sum S is
// then g h with h a power of two, and S is multiplied by g first: S is zero or 2^-18 <=
// |S| < 2^25, so S g is exact to a rounding, and only S g h, the term itself, may
// leave fp32.  Such scales are rare: the warp that copies the scales only looks whether
// any could be in such a product (ScaleRange), and this plain loop makes the outputs
// good at the end of the kernel.  (Two steps in the summing loops took 3-25 % more of
// every product, whichever warp looked for them; this takes 0-3 %, 0.3 us at most.)
__device__ __forceinline__ void again_in_range(const Mm8Params &p, int token, int row_block) {
    const int lane = threadIdx.x & 31;
    const float *w_scales = p.weight_scales + (size_t)row_block * p.blocks;
    bool leaves = false;
    for (int b = lane; b < p.blocks; b += 32) leaves |= leaves_range(p.scales[(size_t)b * p.tokens + token], w_scales[b]);
    if (!__any_sync(0xffffffffu, leaves)) return;
    constexpr int AT_ONCE = 8;                                // rows on their way together
    const int row0 = row_block * ROWS, row1 = min(row0 + ROWS, p.rows);
    for (int row = row0; row < row1; row += AT_ONCE) {
        float out[AT_ONCE] = {};
        for (int b = 0; b < p.blocks; ++b) {
            const int c = b * KB + 4 * lane;                  // this lane's columns of the block
            const float s = p.scales[(size_t)b * p.tokens + token], v = w_scales[b];
            uint32_t xc = 0u, wc[AT_ONCE] = {};
            if (c < p.width) {
                xc = *reinterpret_cast<const uint32_t *>(p.codes + (size_t)token * p.width + c);
#pragma unroll
                for (int i = 0; i < AT_ONCE; ++i)
                    wc[i] = *reinterpret_cast<const uint32_t *>(p.weights + (size_t)min(row + i, row1 - 1) * p.width + c);
            }
            float x[4], w[4], sum[AT_ONCE];
            e4m3_values(xc, x);
#pragma unroll
            for (int i = 0; i < AT_ONCE; ++i) {
                e4m3_values(wc[i], w);
                sum[i] = (w[0] * x[0] + w[1] * x[1]) + (w[2] * x[2] + w[3] * x[3]);
            }
#pragma unroll
            for (int o = 16; o; o >>= 1)
#pragma unroll
                for (int i = 0; i < AT_ONCE; ++i) sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], o);
            float g = 1.f, h = s * v;
            if (leaves_range(s, v)) {
                if (fabsf(h) < 1.f) {                         // neither is above 2^23; a term of a g below 2^-126 is below 2^-200
                    g = (s * 0x1p50f) * (v * 0x1p50f);
                    h = 0x1p-100f;
                } else {                                      // both are above 1; a g of 2^100 is infinity for every sum but zero
                    g = (s * 0x1p-64f) * (v * 0x1p-63f);
                    g = copysignf(fminf(fabsf(g), 0x1p100f), g);
                    h = 0x1p127f;
                }
            }
#pragma unroll
            for (int i = 0; i < AT_ONCE; ++i) out[i] = fmaf(sum[i] * g, h, out[i]);
        }
#pragma unroll
        for (int i = 0; i < AT_ONCE; ++i)
            if (lane == 0 && row + i < row1) p.out[(size_t)token * p.rows + row + i] = out[i];
    }
}

// Tokens first, first + step, ... below `end`, by all warps of the CTA.
__device__ __noinline__ void few_again(Mm8Params p, int first, int step, int end, int row_block) {
    for (int t = first + step * (threadIdx.x >> 5); t < end; t += step * (blockDim.x >> 5)) again_in_range(p, t, row_block);
}

// ---------------------------------------------------------------- few tokens
template <int NT> struct Few {
    // Two CTAs per SM up to 64 tokens, one at 128: their rings hold 192 KB or more
    // in flight.  Four warps scale and add up to 32 tokens, eight beyond.
    static constexpr int CTAS = NT <= 64 ? 2 : 1;
    static constexpr int STAGES = NT == 16 ? 6 : NT == 32 ? 5 : NT == 64 ? 4 : 6;
    static constexpr int BUFS = NT <= 32 ? 4 : 2;            // TMEM accumulators
    static constexpr int SUM_WARPS = NT <= 32 ? 4 : 8, COLS = NT * 4 / SUM_WARPS;   // columns of a warp
    static constexpr int THREADS = 32 * (3 + SUM_WARPS), SCALE_WARP = 2 + SUM_WARPS;
    static constexpr int SLOTS = STAGES + BUFS;              // scale slots
    static constexpr int W_BYTES = ROWS * KB, X_BYTES = NT * KB, STAGE = W_BYTES + X_BYTES;
    static constexpr int SLOT_FLOATS = NT + 4;
    static constexpr int SM_SCALE = STAGES * STAGE;
    static constexpr int SM_BAR = SM_SCALE + SLOTS * SLOT_FLOATS * 4;
    static constexpr int SMEM = SM_BAR + 384;
    static_assert(NT * ROWS * 4 <= STAGES * STAGE, "partial sums exceed the ring");
    static_assert((2 * STAGES + 2 * BUFS + 2 * SLOTS + 1) * 8 + 12 <= 384, "barrier area");
};

template <int NT>
__global__ void __launch_bounds__(Few<NT>::THREADS, Few<NT>::CTAS)
few_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmX, const Mm8Params p) {
    using L = Few<NT>;
    extern __shared__ __align__(1024) uint8_t smem[];
    uint64_t *full = reinterpret_cast<uint64_t *>(smem + L::SM_BAR), *empty = full + L::STAGES;
    uint64_t *d_full = empty + L::STAGES, *d_empty = d_full + L::BUFS, *s_full = d_empty + L::BUFS;
    uint64_t *s_empty = s_full + L::SLOTS, *mma_done = s_empty + L::SLOTS;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(mma_done + 1);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1), *far_flag = abort_flag + 1;
    float *slots = reinterpret_cast<float *>(smem + L::SM_SCALE);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int split = blockIdx.x, rtile = blockIdx.y, t0 = blockIdx.z * NT;
    const int b0 = (int)((long long)p.blocks * split / p.splits), b1 = (int)((long long)p.blocks * (split + 1) / p.splits);
    const int n = b1 - b0;
    const bool bad_base = (smem_addr(smem) & 1023) != 0;      // 128B-swizzle atoms need a 1024-byte aligned base

    if (threadIdx.x == 0) {
        for (int i = 0; i < L::STAGES; ++i) { mbar_init(full + i, 1); mbar_init(empty + i, 1); }
        for (int i = 0; i < L::BUFS; ++i) { mbar_init(d_full + i, 1); mbar_init(d_empty + i, L::SUM_WARPS); }
        for (int i = 0; i < L::SLOTS; ++i) { mbar_init(s_full + i, 32); mbar_init(s_empty + i, L::SUM_WARPS); }
        mbar_init(mma_done, 1);
        *abort_flag = bad_base ? 1 : 0;
        *far_flag = 0;
        if (bad_base) raise_status(STATUS_BAD_ARGUMENT);
        fence_barrier_init();
        prefetch_tmap(&tmW);
        prefetch_tmap(&tmX);
        // The ring's first weights, while the kernel before still runs: into L2, where
        // what that kernel may yet write to them arrives too (behind a norm8, 8 x 5,120 x
        // 17,408: 22.4 -> 21.1 us for both, 1 x 5,120 x 6,144: 17.9 -> 16.8; with the
        // CTA's whole share asked for, 23.6 and 17.1).
        if (!bad_base)
            for (int j = 0; j < min(n, L::STAGES); ++j) prefetch_l2_2d(&tmW, (b0 + j) * KB, rtile * ROWS);
    }
    if (warp == 1) { tmem_alloc(tmem_slot, L::BUFS * NT); tmem_relinquish(); }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    grid_dependency_wait();
    if (threadIdx.x == 0) launch_dependents();

    float2 acc[L::COLS / 2];
#pragma unroll
    for (int c = 0; c < L::COLS / 2; ++c) acc[c] = make_float2(0.f, 0.f);
    const int col0 = (warp - 2) / 4 * L::COLS;                 // this warp's tokens of the tile
    bool ok = !bad_base;
    if (warp == 0) {
        // ------------------------------------------------ producer
        const uint32_t lead = elect_lane();
        int issued = 0;
        for (int j = 0, s = 0, lap = 0; j < n; ++j) {
            if (lap > 0 && !warp_wait8(empty + s, (lap - 1) & 1, abort_flag)) { ok = false; break; }
            if (lead) {
                uint8_t *w = smem + s * L::STAGE;
                mbar_expect_tx(full + s, L::STAGE);
                tma_load_2d(w, &tmW, full + s, (b0 + j) * KB, rtile * ROWS);
                tma_load_2d(w + L::W_BYTES, &tmX, full + s, (b0 + j) * KB, t0);
            }
            __syncwarp();
            issued = j + 1;
            if (++s == L::STAGES) { s = 0; ++lap; }
        }
        // Every issued load must land before the CTA may exit or reuse the ring.
        if (lead) {
            const long long start = clock64();
            for (int j = max(0, issued - L::STAGES); j < issued; ++j)
                while (!mbar_try_wait(full + j % L::STAGES, (j / L::STAGES) & 1) && clock64() - start < WAIT_LIMIT_CYCLES) {}
        }
    } else if (warp == L::SCALE_WARP) {
        // ------------------------------------------------ scales, by small copies
        constexpr int PER_LANE = (NT + 31) / 32;
        const float *src[PER_LANE], *w_src = p.weight_scales + (size_t)rtile * p.blocks + b0;
        bool live[PER_LANE];
#pragma unroll
        for (int i = 0; i < PER_LANE; ++i) {
            const int t = 32 * i + lane;
            live[i] = t < NT && t0 + t < p.tokens;
            src[i] = p.scales + (size_t)b0 * p.tokens + (live[i] ? t0 + t : 0);
        }
        ScaleRange range;
        auto look_at = [&](const float *d) {
            range.add(*reinterpret_cast<const float4 *>(d + 4 * lane % NT));
            range.add(d[NT]);
            __syncwarp();
        };
        for (int j = 0, slot = 0, lap = 0; j < n; ++j) {
            // A slot has barriers of its own: `empty` may go on by two phases while
            // this warp is late, and its parity would then seem not to have changed.
            if (lap > 0 && !warp_wait8(s_empty + slot, (lap - 1) & 1, abort_flag)) { ok = false; break; }
            float *d = slots + slot * L::SLOT_FLOATS;
            if (lap > 0) look_at(d);
#pragma unroll
            for (int i = 0; i < PER_LANE; ++i) {
                if (32 * i + lane < NT) copy_float(d + 32 * i + lane, src[i], live[i]);
                src[i] += p.tokens;
            }
            if (lane == 0) copy_float(d + NT, w_src + j, true);
            arrive_copies(s_full + slot);
            if (++slot == L::SLOTS) { slot = 0; ++lap; }
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
        __syncwarp();
        for (int slot = 0; slot < min(n, L::SLOTS) && ok; ++slot) look_at(slots + slot * L::SLOT_FLOATS);
        if (range.far()) *far_flag = 1;
    } else if (warp == 1) {
        // ------------------------------------------------ MMA issuer
        constexpr uint32_t idesc = idesc_e4m3(ROWS, NT);
        const uint32_t lead = elect_lane(), tm = __shfl_sync(0xffffffffu, tmem, 0);
        for (int j = 0, s = 0, d = 0, lap = 0, dlap = 0; j < n && ok; ++j) {
            if (!warp_wait8(full + s, lap & 1, abort_flag)) { ok = false; break; }
            if (j >= L::BUFS && !warp_wait8(d_empty + d, (dlap - 1) & 1, abort_flag)) { ok = false; break; }
            tc_fence_after();
            const uint64_t w = sw128_desc(smem_addr(smem + s * L::STAGE), 16, 1024);
            const uint64_t x = sw128_desc(smem_addr(smem + s * L::STAGE + L::W_BYTES), 16, 1024);
#pragma unroll
            for (int k = 0; k < KB / 32; ++k)
                mma_e4m3_ss_by(lead, tm + d * NT, w + 2 * k, x + 2 * k, idesc, k > 0 ? 1u : 0u);
            mma_commit_by(lead, empty + s);
            mma_commit_by(lead, d_full + d);
            if (++s == L::STAGES) { s = 0; ++lap; }
            if (++d == L::BUFS) { d = 0; ++dlap; }
        }
        mma_commit_by(lead, mma_done);
        const long long start = clock64();
        while (!mbar_try_wait(mma_done, 0) && clock64() - start < WAIT_LIMIT_CYCLES) {}
    } else {
        // ------------------------------------------------ scales and sums: thread = TMEM lane = weight row
        const uint32_t t_lane = tmem + ((uint32_t)((warp & 3) * 32) << 16) + col0;
        for (int j = 0; j < n; ++j) {
            const int d = j % L::BUFS, slot = j % L::SLOTS;
            if (!warp_wait8(s_full + slot, (j / L::SLOTS) & 1, abort_flag) ||
                !warp_wait8(d_full + d, (j / L::BUFS) & 1, abort_flag)) { ok = false; break; }
            tc_fence_after();
            const float *sc = slots + slot * L::SLOT_FLOATS;
            const float2 ws = make_float2(sc[NT], sc[NT]);
#pragma unroll
            for (int c0 = 0; c0 < L::COLS; c0 += 16) {
                float x[16];
                tmem_ld16(t_lane + d * NT + c0, x);
                tmem_wait_ld();
#pragma unroll
                for (int c = 0; c < 16; c += 4) {
                    const float4 f = *reinterpret_cast<const float4 *>(sc + col0 + c0 + c);
                    float2 &a0 = acc[(c0 + c) / 2], &a1 = acc[(c0 + c) / 2 + 1];
                    a0 = ffma2(make_float2(x[c], x[c + 1]), fmul2(make_float2(f.x, f.y), ws), a0);
                    a1 = ffma2(make_float2(x[c + 2], x[c + 3]), fmul2(make_float2(f.z, f.w), ws), a1);
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) { mbar_arrive(d_empty + d); mbar_arrive(s_empty + slot); }
        }
    }
    __syncwarp();
    tc_fence_before();
    const int all_ok = __syncthreads_and(ok);
    tc_fence_after();
    if (warp == 1) tmem_dealloc(tmem, L::BUFS * NT);

    const int lrow = (warp & 3) * 32 + lane, row = rtile * ROWS + lrow;
    const int live = min(NT, p.tokens - t0);
    if (p.splits == 1) {
        if (warp >= 2 && warp < L::SCALE_WARP && all_ok && row < p.rows) {
#pragma unroll
            for (int t = 0; t < L::COLS; ++t)
                if (col0 + t < live) p.out[(size_t)(t0 + col0 + t) * p.rows + row] = t & 1 ? acc[t / 2].y : acc[t / 2].x;
        }
        if (*far_flag && all_ok) {
            __syncthreads();
            few_again(p, t0, 1, t0 + live, rtile);
        }
        return;
    }
    // Partial sums of the splits meet in shared memory (the idle ring); CTA q
    // of the cluster adds the tokens q, q + splits, ... in the order of the
    // splits.  Every CTA of the cluster passes both barriers.
    float *part = reinterpret_cast<float *>(smem);
    int *good = reinterpret_cast<int *>(slots);               // this CTA's partial sums are complete
    const bool sums = warp >= 2 && warp < L::SCALE_WARP;
    if (sums) {
#pragma unroll
        for (int t = 0; t < L::COLS; ++t) part[(col0 + t) * ROWS + lrow] = t & 1 ? acc[t / 2].y : acc[t / 2].x;
    }
    if (threadIdx.x == 0) *good = all_ok;
    cluster_sync();
    if (threadIdx.x == 0 && *far_flag)                        // every CTA of the cluster has outputs of this one's blocks
        for (int q = 0; q < p.splits; ++q) st_cluster_f32(cluster_map(const_cast<int *>(far_flag), q), 1.f);
    if (sums) {
        bool fine = true;
        for (int q = 0; q < p.splits; ++q) fine = fine && __float_as_int(ld_cluster_f32(cluster_map(good, q))) != 0;
        // a warp adds one token's 128 rows at a time, four rows a lane
        const int row4 = rtile * ROWS + 4 * lane;
        const bool vec = p.rows % 4 == 0 && (reinterpret_cast<uintptr_t>(p.out) & 15) == 0;
        const uint32_t mine = smem_addr(part) + 16 * lane;
        for (int t = split + p.splits * (warp - 2); fine && t < live; t += p.splits * L::SUM_WARPS) {
            float4 v[MAX_SPLITS];
#pragma unroll
            for (int q = 0; q < MAX_SPLITS; ++q)
                if (q < p.splits) v[q] = ld_cluster_f32x4(cluster_rank(mine + t * ROWS * 4, q));
            float4 sum = v[0];
#pragma unroll
            for (int q = 1; q < MAX_SPLITS; ++q)
                if (q < p.splits) { sum.x += v[q].x; sum.y += v[q].y; sum.z += v[q].z; sum.w += v[q].w; }
            float *dst = p.out + (size_t)(t0 + t) * p.rows + row4;
            if (vec) {
                if (row4 < p.rows) *reinterpret_cast<float4 *>(dst) = sum;
            } else {
                if (row4 < p.rows) dst[0] = sum.x;
                if (row4 + 1 < p.rows) dst[1] = sum.y;
                if (row4 + 2 < p.rows) dst[2] = sum.z;
                if (row4 + 3 < p.rows) dst[3] = sum.w;
            }
        }
    }
    cluster_sync();
    if (*far_flag) few_again(p, t0 + split, p.splits, min(t0 + NT, p.tokens), rtile);
}

// ---------------------------------------------------------------- many tokens
// A block's MMAs take 513 cycles, scaling and adding its 128 x 256 sums 256 cycles of
// every FMA lane, and TMEM holds the sums of two blocks.  A block takes 800 cycles:
// its sums' way from the MMA through two barriers and back, halved; the output of a
// tile, which waits for the stores, takes 7,000.  Measured and not faster (4,001 x 5,120
// x 17,408, beside this form's 390 us): pairs of CTAs on 256 x 256 tiles (cta_group::2)
// 410-460, sixteen summing warps 400, halves of the weight rows handed over separately
// 410, registers moved to the summing warps for two chunks in flight 410-450, rows of
// the output by bulk copies 457.  Without the sums the MMAs of this shape run at 590
// cycles a block.
struct Many {
    static constexpr int MT = 128, NT = 256;                 // tokens, weight rows of a tile
    static constexpr int STAGES = 4, BUFS = 2, SLOTS = STAGES + BUFS, SUM_WARPS = 8, SCALE_WARP = 10, THREADS = 352;
    static constexpr int X_BYTES = MT * KB, W_BYTES = NT * KB, STAGE = X_BYTES + W_BYTES;
    static constexpr int SLOT_FLOATS = MT + 4;
    static constexpr int OUT_ROW = 20;                       // floats of a staged row: 16 columns and a pad
    static constexpr int SM_OUT = STAGES * STAGE;            // [8 warps][32 rows][OUT_ROW]
    static constexpr int SM_SCALE = SM_OUT + 8 * 32 * OUT_ROW * 4;
    static constexpr int SM_BAR = SM_SCALE + SLOTS * SLOT_FLOATS * 4;
    static constexpr int SMEM = SM_BAR + 384;
    static_assert(SMEM <= 227 * 1024, "shared memory of a CTA");
};

// again_in_range over the tiles of this CTA; apart, so that nothing has to be kept for it.
__device__ __noinline__ void many_again(Mm8Params p) {
    const int row_blocks = (p.rows + ROWS - 1) / ROWS;
    for (int tile = blockIdx.x; tile < p.tiles; tile += gridDim.x) {
        const int m0 = tile % p.m_tiles * Many::MT, r0 = tile / p.m_tiles * (Many::NT / ROWS);
        for (int q = threadIdx.x >> 5; q < 2 * min(Many::MT, p.tokens - m0); q += Many::THREADS / 32)
            if (r0 + (q & 1) < row_blocks) again_in_range(p, m0 + (q >> 1), r0 + (q & 1));
    }
}

__global__ void __launch_bounds__(Many::THREADS, 1)
many_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmX, const Mm8Params p) {
    using L = Many;
    extern __shared__ __align__(1024) uint8_t smem[];
    uint64_t *full = reinterpret_cast<uint64_t *>(smem + L::SM_BAR), *empty = full + L::STAGES;
    uint64_t *d_full = empty + L::STAGES, *d_empty = d_full + L::BUFS, *s_full = d_empty + L::BUFS;
    uint64_t *s_empty = s_full + L::SLOTS, *mma_done = s_empty + L::SLOTS;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(mma_done + 1);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1), *far_flag = abort_flag + 1;
    float *slots = reinterpret_cast<float *>(smem + L::SM_SCALE);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const bool bad_base = (smem_addr(smem) & 1023) != 0;
    if (threadIdx.x == 0) {
        for (int i = 0; i < L::STAGES; ++i) { mbar_init(full + i, 1); mbar_init(empty + i, 1); }
        for (int i = 0; i < L::BUFS; ++i) { mbar_init(d_full + i, 1); mbar_init(d_empty + i, L::SUM_WARPS); }
        for (int i = 0; i < L::SLOTS; ++i) { mbar_init(s_full + i, 32); mbar_init(s_empty + i, L::SUM_WARPS); }
        mbar_init(mma_done, 1);
        *abort_flag = bad_base ? 1 : 0;
        *far_flag = 0;
        if (bad_base) raise_status(STATUS_BAD_ARGUMENT);
        fence_barrier_init();
        prefetch_tmap(&tmW);
        prefetch_tmap(&tmX);
    }
    if (warp == 1) { tmem_alloc(tmem_slot, 512); tmem_relinquish(); }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    grid_dependency_wait();
    if (threadIdx.x == 0) launch_dependents();

    // Tiles in order of the token tile first: the CTAs that run together share
    // a few weight tiles and all of X in L2.
    const int mine = p.tiles > (int)blockIdx.x ? (p.tiles - (int)blockIdx.x + (int)gridDim.x - 1) / (int)gridDim.x : 0;
    const int row_blocks = (p.rows + ROWS - 1) / ROWS;
    if (bad_base) {
    } else if (warp == 0) {
        // ------------------------------------------------ producer
        const uint32_t lead = elect_lane();
        int j = 0, s = 0, lap = 0;                           // j: blocks since the start, over all tiles
        bool ok = true;
        for (int i = 0; i < mine && ok; ++i) {
            const int tile = blockIdx.x + i * gridDim.x, m0 = tile % p.m_tiles * L::MT, n0 = tile / p.m_tiles * L::NT;
            for (int b = 0; b < p.blocks; ++b, ++j) {
                if (lap > 0 && !warp_wait8(empty + s, (lap - 1) & 1, abort_flag)) { ok = false; break; }
                if (lead) {
                    uint8_t *x = smem + s * L::STAGE;
                    mbar_expect_tx(full + s, L::STAGE);
                    tma_load_2d(x, &tmX, full + s, b * KB, m0);
                    tma_load_2d(x + L::X_BYTES, &tmW, full + s, b * KB, n0);
                }
                __syncwarp();
                if (++s == L::STAGES) { s = 0; ++lap; }
            }
        }
        // Every issued load must land before the CTA may exit.
        if (lead) {
            const long long start = clock64();
            for (int q = max(0, j - L::STAGES); q < j; ++q)
                while (!mbar_try_wait(full + q % L::STAGES, (q / L::STAGES) & 1) && clock64() - start < WAIT_LIMIT_CYCLES) {}
        }
    } else if (warp == L::SCALE_WARP) {
        // ------------------------------------------------ scales, by small copies
        int slot = 0, lap = 0;
        bool ok = true;
        ScaleRange range;
        auto look_at = [&](const float *d) {
            range.add(*reinterpret_cast<const float4 *>(d + 4 * lane));
            range.add(d[L::MT + (lane & 1)]);
            __syncwarp();
        };
        for (int i = 0; i < mine && ok; ++i) {
            const int tile = blockIdx.x + i * gridDim.x, m0 = tile % p.m_tiles * L::MT, n0 = tile / p.m_tiles * L::NT;
            bool live[4];
            const float *src[4];
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                live[t] = m0 + 32 * t + lane < p.tokens;
                src[t] = p.scales + (live[t] ? m0 + 32 * t + lane : 0);
            }
            const bool w_live = n0 / ROWS + lane < row_blocks;
            const float *w_src = p.weight_scales + (size_t)(w_live ? n0 / ROWS + lane : 0) * p.blocks;
            for (int b = 0; b < p.blocks; ++b) {
                if (lap > 0 && !warp_wait8(s_empty + slot, (lap - 1) & 1, abort_flag)) { ok = false; break; }
                float *d = slots + slot * L::SLOT_FLOATS;
                if (lap > 0) look_at(d);
#pragma unroll
                for (int t = 0; t < 4; ++t) {
                    copy_float(d + 32 * t + lane, src[t], live[t]);
                    src[t] += p.tokens;
                }
                if (lane < 2) copy_float(d + L::MT + lane, w_src + b, w_live);
                arrive_copies(s_full + slot);
                if (++slot == L::SLOTS) { slot = 0; ++lap; }
            }
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
        __syncwarp();
        for (int q = 0; q < min(mine * p.blocks, L::SLOTS) && ok; ++q) look_at(slots + q * L::SLOT_FLOATS);
        if (range.far()) *far_flag = 1;
    } else if (warp == 1) {
        constexpr uint32_t idesc = idesc_e4m3(L::MT, L::NT);
        const uint32_t lead = elect_lane(), tm = __shfl_sync(0xffffffffu, tmem, 0);
        const int n = mine * p.blocks;
        for (int j = 0, s = 0, lap = 0; j < n; ++j) {
            const int d = j & 1;
            if (!warp_wait8(full + s, lap & 1, abort_flag)) break;
            if (j >= 2 && !warp_wait8(d_empty + d, ((j >> 1) - 1) & 1, abort_flag)) break;
            tc_fence_after();
            const uint64_t x = sw128_desc(smem_addr(smem + s * L::STAGE), 16, 1024);
            const uint64_t w = sw128_desc(smem_addr(smem + s * L::STAGE + L::X_BYTES), 16, 1024);
#pragma unroll
            for (int k = 0; k < KB / 32; ++k)
                mma_e4m3_ss_by(lead, tm + d * L::NT, x + 2 * k, w + 2 * k, idesc, k > 0 ? 1u : 0u);
            mma_commit_by(lead, empty + s);
            mma_commit_by(lead, d_full + d);
            if (++s == L::STAGES) { s = 0; ++lap; }
        }
        mma_commit_by(lead, mma_done);
        const long long start = clock64();
        while (!mbar_try_wait(mma_done, 0) && clock64() - start < WAIT_LIMIT_CYCLES) {}
    } else {
        // Warps 2-5 take the tile's columns [0, 128), warps 6-9 [128, 256);
        // thread = TMEM lane = token.
        const int half = (warp - 2) >> 2, lrow = (warp & 3) * 32;
        const uint32_t t_col = tmem + ((uint32_t)lrow << 16) + half * 128;
        float *stage = reinterpret_cast<float *>(smem + L::SM_OUT) + (warp - 2) * 32 * L::OUT_ROW;
        int j = 0;
        bool ok = true;
        for (int i = 0; i < mine && ok; ++i) {
            const int tile = blockIdx.x + i * gridDim.x, m0 = tile % p.m_tiles * L::MT, n0 = tile / p.m_tiles * L::NT;
            float2 acc[64];
#pragma unroll
            for (int c = 0; c < 64; ++c) acc[c] = make_float2(0.f, 0.f);
            for (int b = 0; b < p.blocks; ++b, ++j) {
                const int d = j % L::BUFS, slot = j % L::SLOTS;
                if (!warp_wait8(s_full + slot, (j / L::SLOTS) & 1, abort_flag) ||
                    !warp_wait8(d_full + d, (j / L::BUFS) & 1, abort_flag)) { ok = false; break; }
                tc_fence_after();
                const float *sc = slots + slot * L::SLOT_FLOATS;
                const float f = sc[lrow + lane] * sc[L::MT + half];
                const float2 f2 = make_float2(f, f);
                float x[2][16];
#pragma unroll
                for (int c0 = 0; c0 < 128; c0 += 32) {
                    tmem_ld16(t_col + d * L::NT + c0, x[0]);
                    tmem_ld16(t_col + d * L::NT + c0 + 16, x[1]);
                    tmem_wait_ld();
#pragma unroll
                    for (int q = 0; q < 2; ++q)
#pragma unroll
                        for (int c = 0; c < 8; ++c)
                            acc[c0 / 2 + q * 8 + c] = ffma2(make_float2(x[q][2 * c], x[q][2 * c + 1]), f2, acc[c0 / 2 + q * 8 + c]);
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) { mbar_arrive(d_empty + d); mbar_arrive(s_empty + slot); }
            }
            if (!ok) break;
            // 16 columns at a time through shared memory: 64-byte pieces of eight rows per store.
            const bool vec = p.rows % 4 == 0 && (reinterpret_cast<uintptr_t>(p.out) & 15) == 0;
#pragma unroll
            for (int c0 = 0; c0 < 128; c0 += 16) {
#pragma unroll
                for (int c = 0; c < 16; c += 4) {
                    const float2 a = acc[(c0 + c) / 2], e = acc[(c0 + c) / 2 + 1];
                    *reinterpret_cast<float4 *>(stage + lane * L::OUT_ROW + c) = make_float4(a.x, a.y, e.x, e.y);
                }
                __syncwarp();
                const int col = n0 + half * 128 + c0 + (lane & 3) * 4;
#pragma unroll
                for (int r0 = 0; r0 < 32; r0 += 8) {
                    const int r = r0 + (lane >> 2), token = m0 + lrow + r;
                    const float4 v = *reinterpret_cast<const float4 *>(stage + r * L::OUT_ROW + (lane & 3) * 4);
                    if (token >= p.tokens) continue;
                    float *dst = p.out + (size_t)token * p.rows + col;
                    if (vec) {
                        if (col < p.rows) *reinterpret_cast<float4 *>(dst) = v;
                    } else {
                        if (col < p.rows) dst[0] = v.x;
                        if (col + 1 < p.rows) dst[1] = v.y;
                        if (col + 2 < p.rows) dst[2] = v.z;
                        if (col + 3 < p.rows) dst[3] = v.w;
                    }
                }
                __syncwarp();
            }
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 1) tmem_dealloc(tmem, 512);
    if (*far_flag && !*abort_flag) many_again(p);
}

// ---------------------------------------------------------------- host
// Map over [count][width] codes: box = 128 columns x `box_rows`, 128B swizzle; past the edges zeros are read.
CUtensorMap codes_map(const void *base, int width, int count, int box_rows) {
    CUtensorMap m;
    cuuint64_t dims[2] = {(cuuint64_t)width, (cuuint64_t)count};
    cuuint64_t strides[1] = {(cuuint64_t)width};
    cuuint32_t box[2] = {KB, (cuuint32_t)box_rows};
    cuuint32_t estr[2] = {1, 1};
    const CUresult r = tensor_map_encoder()(&m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void *>(base), dims, strides,
                                            box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                                            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) throw std::runtime_error("cuTensorMapEncodeTiled failed: " + std::to_string((int)r));
    return m;
}

PerDeviceOnce g_configured;
template <class K> void reserve(K *kernel, int bytes) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess)
        throw std::runtime_error("cannot reserve shared memory for the e4m3 product");
}

template <class K>
void launch_cluster(K *kernel, dim3 grid, int threads, int smem, int cluster, cudaStream_t st, const CUtensorMap &mw,
                    const CUtensorMap &mx, const Mm8Params &p) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = cluster;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, mw, mx, p);
    if (e != cudaSuccess) throw std::runtime_error(std::string("e4m3 product: ") + cudaGetErrorString(e));
}

template <int NT> void launch_few(Mm8Params p, const void *weights, const void *x, int width, cudaStream_t st) {
    using L = Few<NT>;
    const int row_tiles = (p.rows + ROWS - 1) / ROWS, token_tiles = (p.tokens + NT - 1) / NT;
    // Split the width as far as the CTAs fit the SMs at once and every CTA keeps four
    // blocks, but not over clusters of more than six: seven and eight pack badly (1 x
    // 6,144 x 5,120: four 9.6, six 10.0, seven 16.3, eight 15.6 us; 64 x 5,120 x
    // 10,240: two 17.6, three 15.6; 100 x 5,120 x 5,120: two 16.0, three 13.4; all
    // before far scales were looked for, which adds up to 0.3).
    const long long slots = 148LL * L::CTAS, tiles = (long long)row_tiles * token_tiles;
    const int splits = (int)std::max(1LL, std::min<long long>({MAX_SPLITS, slots / tiles, p.blocks / 4}));
    p.splits = splits;
    const CUtensorMap mw = codes_map(weights, width, p.rows, ROWS), mx = codes_map(x, width, p.tokens, NT);
    launch_cluster(few_kernel<NT>, dim3(splits, row_tiles, token_tiles), L::THREADS, L::SMEM, splits, st, mw, mx, p);
}

}  // namespace

void mm8(float *out, const void *weights, const float *weight_scales, const void *x, const float *scales, int tokens,
         int width, int rows, cudaStream_t st) {
    g_configured.run([] {
        reserve(few_kernel<16>, Few<16>::SMEM); reserve(few_kernel<32>, Few<32>::SMEM);
        reserve(few_kernel<64>, Few<64>::SMEM); reserve(few_kernel<128>, Few<128>::SMEM);
        reserve(many_kernel, Many::SMEM);
    });
    Mm8Params p{out, weight_scales, scales, static_cast<const uint8_t *>(weights), static_cast<const uint8_t *>(x),
                tokens, rows, width, (width + KB - 1) / KB, 1, 0, 0};
    const int m_tiles = (tokens + Many::MT - 1) / Many::MT;
    const long long tiles = (long long)m_tiles * ((rows + Many::NT - 1) / Many::NT);
    // Beyond 128 tokens few_kernel<128> is still the faster one while all its tiles
    // run at once (384 x 5,120 x 5,120: 23.3 against 27.1 us, 256 x 17,408 x 5,120: 65
    // against 72; two waves of it, 256 x 5,120 x 10,240: 42 against 28).
    const long long few_tiles = (long long)((tokens + 127) / 128) * ((rows + ROWS - 1) / ROWS);
    if (tokens > 128 && few_tiles > 148) {
        p.m_tiles = m_tiles;
        p.tiles = (int)tiles;
        int dev = 0, sms = 148;
        if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
        const CUtensorMap mw = codes_map(weights, width, rows, Many::NT), mx = codes_map(x, width, tokens, Many::MT);
        launch_cluster(many_kernel, dim3((unsigned)std::min<long long>(tiles, sms)), Many::THREADS, Many::SMEM, 1, st, mw, mx, p);
    } else if (tokens <= 16) {
        launch_few<16>(p, weights, x, width, st);
    } else if (tokens <= 32) {
        launch_few<32>(p, weights, x, width, st);
    } else if (tokens <= 64) {
        launch_few<64>(p, weights, x, width, st);
    } else {
        launch_few<128>(p, weights, x, width, st);
    }
}

}  // namespace qv
