// What the decode attention kernels share (attention.cu over the fp16 cache,
// attention8.cu over the 8-bit cache): the shapes and TMEM map of a decode CTA,
// the rotary embedding, the prepare step and append, the split epilogue, the
// split plan and workspace, and the tail that combines the splits.
#pragma once
#include "common.cuh"

#include <algorithm>

namespace qv {

constexpr int NQ = 24, NKV = 4, HD = 256, GROUP = NQ / NKV;
constexpr int BN = 64;           // cache positions per K/V tile
constexpr int TILE_BYTES = 4 * BN * 128;                      // one K or V tile, 4 boxes of 64 rows x 128 B
constexpr int DECODE_ROWS = 64;                               // logical rows of a decode CTA
constexpr float SCORE_LOG2 = 0.0625f * 1.4426950408889634f;   // (1/16) * log2(e)
constexpr float RESCALE_THRESHOLD = 8.f;                      // lazy O rescale, log2 units
constexpr int MAX_DECODE_T = DECODE_ROWS / GROUP;             // largest decode / verify batch (10)
// Rotary inverse frequencies 1e7^(-i/32), i = 0..31, as exact doubles (the
// values Python's 10000000 ** (-i / 32) yields).
static __constant__ double kRopeInvFreq[32] = {
    0x1.0000000000000p+0,  0x1.3566562253c7ep-1, 0x1.75f034d79e965p-2, 0x1.c3f06b4e265cep-3,
    0x1.111aedafb9a9dp-3,  0x1.4a12ad8379eb8p-4, 0x1.8eec7def5d56cp-5, 0x1.e222ec75094e2p-6,
    0x1.235a71c5ee5ccp-6,  0x1.6020a364b1284p-7, 0x1.a99428b3d26b3p-8, 0x1.012cfaad0da13p-8,
    0x1.36d219065ac0cp-9,  0x1.77a7d87ee61b0p-10, 0x1.c603c39630446p-11, 0x1.125c04ab2d71fp-11,
    0x1.4b96be9c2da2cp-12, 0x1.90c181b38fe22p-13, 0x1.e459c57e28a47p-14, 0x1.24b0fd0e890d4p-14,
    0x1.61bea2721385fp-15, 0x1.ab88830de4ad5p-16, 0x1.025b57369650bp-16, 0x1.383f8796f72a9p-17,
    0x1.7961810874a9fp-18, 0x1.c8198c91f9fccp-19, 0x1.139e9527f964ep-19, 0x1.4d1c97f4e952fp-20,
    0x1.9298ace36f12ep-21, 0x1.e69338f8adcd3p-22, 0x1.26091b11c8665p-22, 0x1.635e883bbc816p-23,
};

// (cos, sin) of the rotary angle pos * 1e7^(-i/32).  The angle is formed in
// double precision (it reaches ~1.4e5 rad, where float would lose ~1e-2 rad)
// and reduced by 2*pi with a two-part Cody-Waite split (a 33-bit head, so
// k * head is exact for |k| < 2^20, and a tail); the reduced |x| <= pi is then
// rounded to float and evaluated with single-precision sincosf, within a few
// float ulps of cos / sin of the double angle.
__device__ __forceinline__ float2 rope_angle(int pos, int i) {
    const double theta = (double)pos * kRopeInvFreq[i];
    const double k = rint(theta * 0.15915494309189535);          // 1 / (2 pi)
    const double x = fma(-k, 0x1.0b4611a626331p-32, fma(-k, 0x1.921fb54400000p+2, theta));
    float sf, cf;
    sincosf((float)x, &sf, &cf);
    return make_float2(cf, sf);
}

// Rotary embedding of one 256-wide row spread over a warp, lane l holding
// dims [4l, 4l+4) in v (dims [0,64) live in lanes 0..15): pairs (i, i+32),
// i < 32, rotate by the angle whose (cos, sin) is cs[i].
// Branch-free, so that consecutive rows interleave: lanes that do not
// rotate use the identity (cos 1, sin 0).
__device__ __forceinline__ void rope_row(float (&v)[4], const float2 *cs, int lane, bool apply) {
    const bool rot = apply && lane < 16;
    const float sign = lane < 8 ? -1.f : 1.f;      // lane < 8: a*c - b*s;  8..15: b*c + a*s
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const float partner = __shfl_xor_sync(0xffffffffu, v[e], 8);
        const float2 r = cs[4 * (lane & 7) + e];
        const float c = rot ? r.x : 1.f, sn = rot ? sign * r.y : 0.f;
        v[e] = fmaf(partner, sn, v[e] * c);
    }
}
__device__ __forceinline__ uint32_t half2_bits(__half2 h) { return *reinterpret_cast<const uint32_t *>(&h); }
// TMEM columns: S double buffer [0,128), O [128,384), Q (A operand) [384,512).
constexpr uint32_t TM_S = 0, TM_O = 128, TM_Q = 384;

// What a decode launch does with its rows once every split is done (the
// kernel tail, after a barrier over the CTAs of each KV head).
enum DecodeTail : int {
    TAIL_GATED = 0,      // out = softmax(...) V * sigmoid(gate)
    TAIL_SHARD = 1,      // out = normalised partial of this cache shard, lse = its natural-log LSE
    TAIL_EXCHANGE = 2,   // shard partial pushed to every rank's buffer, all ranks' partials merged, gated
};

struct FaParams {
    const float *q_gate;    // [T][24][512]: q = [0:256), gate = [256:512)
    float *out;             // [T][24][256]
    float *lse;             // natural-log LSE [T][24] (TAIL_SHARD)
    float *part_o;          // [4][64 rows][splits][256] unnormalised partial O of every split
    float *part_ml;         // [4][64 rows][MAXS][2] (running max in log2 units, sum)
    unsigned long long *sync;  // [4] per-KV-head barrier words (generation : arrivals)
    int T, position;        // tokens and absolute position of token 0
    int kv_begin;           // absolute position of cache row 0
    int kv_rows;            // valid cache rows
    int split_tiles, splits;
    int tail;               // DecodeTail
    const uint64_t *peers;  // TAIL_EXCHANGE: every rank's receive buffer
    int world, rank, seq;
    // The prepare step folded in: the CTA normalises and rotates its own query
    // rows from q_gate and, when its tiles hold the block's new cache rows,
    // writes their keys / values before loading them.
    const float *key, *value, *qn, *kn;
    __half *kc, *vc;        // the caches, for the append
    int append_row0;        // local cache row of token 0's key / value, or -1
    float eps;
};

// Logical query row -> (token, head): the rows of a CTA pack the 6 query heads
// of its KV head (blockIdx.y) and the T tokens.
__device__ __forceinline__ bool row_token_head(const FaParams &p, int r, int &t, int &h) {
    t = r / GROUP;
    h = blockIdx.y * GROUP + r % GROUP;
    return r < p.T * GROUP;
}

// Warp-uniform bounded wait (all lanes agree on the outcome).
__device__ __forceinline__ bool warp_wait(uint64_t *bar, uint32_t parity, volatile int *abort_flag) {
    return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag));
}

// ---------------------------------------------------------------- decode tail
// After its split of the cache, a decode CTA waits at a barrier over the CTAs
// of its KV head, then combines a share of the head's rows from all splits'
// partials (rows blockIdx.x, blockIdx.x + splits, ...): the split combine
// runs inside the attention launch, on every SM, with no second kernel.
constexpr float LN2 = 0.6931471805599453f;
constexpr int MAXS = 40;                               // splits a tail combine handles (plans use <= 37)

// Peer exchange (TAIL_EXCHANGE, multi-GPU verify).  Each rank's receive
// buffer holds [2 slots][world][EX_ROWS][EX_WORDS] 64-bit words (256 O, lse,
// padding) per row t*24 + h.  Every value travels as a word {value bits,
// tag}: the reader spins on each of its words until the tag of this call
// appears, so no fence or separate flag write is needed, and it zeroes each
// word after reading it.  `seq` counts the calls on these buffers (the same
// on every rank, +1 per call): its parity picks the slot and its low 24 bits
// are in the tag.  A rank writes into a slot again two calls later, after it
// has received this rank's partials of the call in between, and that call
// started only after this one (and its zeroing) completed.  A word that
// arrives after its reader gave up (a timeout) stays behind unread, but it
// carries the tag of its own call and the next call on that slot waits for a
// different tag, so it is never taken for new data.
constexpr int EX_ROWS = MAX_DECODE_T * NQ;       // rows of the largest decode batch
constexpr int EX_WORDS = 264;                    // words per row: 256 O + lse, padded to 64 bytes
constexpr int EX_MAX_WORLD = 8;
__host__ __device__ constexpr uint32_t ex_tag(int seq) {   // high half of a filled word; never 0
    return 0x51000000u | ((uint32_t)seq & 0x00FFFFFFu);
}
__host__ __device__ constexpr size_t ex_bytes(int world) {
    return (size_t)2 * world * EX_ROWS * EX_WORDS * sizeof(uint64_t);
}

// Barrier over the `splits` CTAs of one KV head, on one 64-bit word of the
// workspace: arrivals in the low half, a generation count in the high half.
// The arrivals must be zero before the first launch on a workspace.  A CTA
// waits until the arrivals reach `splits` or the generation moves on; the
// last CTA to arrive then resets the arrivals and advances the generation in
// one atomic add (off the others' critical path: they may leave as soon as
// its arrival shows), so every launch leaves the arrivals zero, also after a
// timeout (every CTA arrives; only a waiter gives up).  A launch has at most
// (SMs / 4) CTAs per head and one CTA per SM, so all CTAs of a head are
// resident together.  Bounded: a wait past the limit raises STATUS_TIMEOUT.
static __device__ bool head_barrier(unsigned long long *word, int splits, volatile int *flag) {
    fence_async_global();                              // the partials are read back by bulk copies
    __syncthreads();                                   // this CTA's partials are written
    if (threadIdx.x == 0) {
        __threadfence();                               // release them
        const unsigned long long old = atomicAdd(word, 1ull);
        bool ok = true;
        if ((uint32_t)old == (uint32_t)splits - 1) {
            atomicAdd(word, (1ull << 32) - (unsigned long long)splits);   // arrivals -> 0, generation + 1
        } else {
            const uint32_t gen = (uint32_t)(old >> 32);
            const long long start = clock64();
            while (true) {
                const unsigned long long v = ld_acquire_gpu_u64(word);
                if ((uint32_t)v >= (uint32_t)splits || (uint32_t)(v >> 32) != gen) break;
                if (clock64() - start > WAIT_LIMIT_CYCLES) { raise_status(STATUS_TIMEOUT); ok = false; break; }
            }
        }
        __threadfence();                               // acquire the other CTAs' partials
        *flag = ok ? 1 : 0;
    }
    __syncthreads();
    return *flag != 0;
}

// Bulk copy global -> shared (no tensor map), completion on the mbarrier's
// transaction count: addresses 16-byte aligned, size a multiple of 16.
__device__ __forceinline__ void bulk_load(void *dst, const void *src, uint32_t bytes, uint64_t *bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 :: "r"(smem_addr(dst)), "l"(src), "r"(bytes), "r"(smem_addr(bar)) : "memory");
}

// Split combine of decode rows ra and rb (rb < 0: ra only) of KV head g (row r
// = token r / 6, head 6g + r % 6).  A row's partials of all splits are one
// contiguous block (splits x 1 KB), and so are its splits' (max, sum) pairs
// (MAXS x 8 bytes): thread 0 brings both rows' blocks into shared memory
// (`buf`, the idle K/V ring) with bulk copies on `bar` (phase parity
// `phase`).  o[k] receives the normalised value of row k in dimension
// threadIdx.x, lse[k] its natural-log LSE.  `sh` holds 1280 floats of shared
// memory (weights and maxima in the first 2 MAXS + 8, the exchange's words
// after them, the rows' halves from float 256 on); the call ends with a CTA
// barrier.
static __device__ bool combine_rows(const FaParams &p, int g, int ra, int rb, float *sh, float *buf, uint64_t *bar,
                             uint32_t phase, volatile int *abort_flag, float (&o)[2], float (&lse)[2]) {
    const int d = threadIdx.x, S = p.splits;
    const bool two = rb >= 0;
    const size_t row_a = (size_t)g * DECODE_ROWS + ra, row_b = (size_t)g * DECODE_ROWS + (two ? rb : ra);
    float *xa = buf, *xb = buf + (size_t)S * HD;                    // partials [split][256]
    float *mla = buf + 2 * (size_t)S * HD, *mlb = mla + 2 * MAXS;   // (max, sum) [MAXS][2]
    if (threadIdx.x == 0) {
        // The partials were written through the generic proxy (and acquired
        // at the barrier); the bulk copies read them through the async proxy,
        // and overwrite shared memory the CTA last used through the generic one.
        fence_async_global();
        fence_async_shared();
        const uint32_t bytes = (uint32_t)S * HD * sizeof(float), ml_bytes = 2 * MAXS * sizeof(float);
        mbar_expect_tx(bar, two ? 2 * (bytes + ml_bytes) : bytes + ml_bytes);
        bulk_load(xa, p.part_o + row_a * S * HD, bytes, bar);
        bulk_load(mla, p.part_ml + row_a * 2 * MAXS, ml_bytes, bar);
        if (two) {
            bulk_load(xb, p.part_o + row_b * S * HD, bytes, bar);
            bulk_load(mlb, p.part_ml + row_b * 2 * MAXS, ml_bytes, bar);
        }
    }
    const bool ok = mbar_wait(bar, phase, abort_flag);
    if (threadIdx.x == 0 && phase == 0) QV_STAMP(14);
    // (max, sum) of split e of row a on threads [0, S), of row b on [64, 64 + S)
    const int e = d < 64 ? d : d - 64;
    float m = -INFINITY, l = 0.f;
    if (ok && e < S && (d < 64 || (two && d < 128))) {
        const float *ml = d < 64 ? mla : mlb;
        m = ml[2 * e]; l = ml[2 * e + 1];
    }
    float *wa = sh, *wb = sh + MAXS, *red = sh + 2 * MAXS;   // red: maxima [0..3], sums [4..7]
    float M = m;
#pragma unroll
    for (int k = 16; k; k >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, k));
    if (d < 128 && (d & 31) == 0) red[d >> 5] = M;
    __syncthreads();
    const float Ma = fmaxf(red[0], red[1]), Mb = fmaxf(red[2], red[3]);
    const float w = (e < S && d < 128 && m != -INFINITY) ? exp2f(m - (d < 64 ? Ma : Mb)) : 0.f;
    if (d < MAXS) wa[d] = w;
    else if (d >= 64 && d < 64 + MAXS) wb[d - 64] = w;
    const float den_part = warp_sum(w * l);
    if (d < 128 && (d & 31) == 0) red[4 + (d >> 5)] = den_part;
    __syncthreads();
    const float den_a = red[4] + red[5], den_b = red[6] + red[7];
    // The weighted sum over the splits: thread (row, half, quad) reads four
    // dimensions of its row with 16-byte loads over half of the splits; the
    // two halves meet in shared memory.
    const int rsel = d >> 7, hsel = (d >> 6) & 1, quad = d & 63;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    if (ok && (rsel == 0 || two)) {
        const float *x = rsel ? xb : xa, *w = rsel ? wb : wa;
        const int k0 = hsel ? S / 2 : 0, k1 = hsel ? S : S / 2;
        for (int k = k0; k < k1; ++k) {
            const float4 v = *reinterpret_cast<const float4 *>(x + (size_t)k * HD + 4 * quad);
            const float wk = w[k];
            acc.x = fmaf(wk, v.x, acc.x); acc.y = fmaf(wk, v.y, acc.y);
            acc.z = fmaf(wk, v.z, acc.z); acc.w = fmaf(wk, v.w, acc.w);
        }
    }
    float4 *part = reinterpret_cast<float4 *>(sh + 768);   // [2 rows][64 quads], the second halves
    float *res = sh + 256;                                   // [2 rows][256], the normalised rows
    if (hsel) part[rsel * 64 + quad] = acc;
    __syncthreads();
    if (!hsel) {
        const float4 b = part[rsel * 64 + quad];
        const float den = rsel ? den_b : den_a, inv = den > 0.f ? 1.f / den : 0.f;
        *reinterpret_cast<float4 *>(res + rsel * HD + 4 * quad) =
            make_float4((acc.x + b.x) * inv, (acc.y + b.y) * inv, (acc.z + b.z) * inv, (acc.w + b.w) * inv);
    }
    __syncthreads();
    o[0] = res[d];
    o[1] = res[HD + d];
    lse[0] = den_a > 0.f ? (Ma + log2f(den_a)) * LN2 : -INFINITY;
    lse[1] = den_b > 0.f ? (Mb + log2f(den_b)) * LN2 : -INFINITY;
    __syncthreads();                                   // sh and buf are free again
    return ok;
}

// Peer exchange of up to two rows (global row indices grow[k] = t*24 + h, k <
// nr): this shard's normalised values o[k] (dimension threadIdx.x) and LSEs go
// into slot [rank] of every other rank's buffer, then the other ranks' words
// of the rows are read from this rank's own buffer (all peers and both rows
// at once, so their latencies overlap; a word without this call's tag is
// re-read until it has it, bounded) and merged: sum_g exp(lse_g - LSE) o_g,
// written back into o[k].  `sh` holds 2 EX_MAX_WORLD floats; the call ends
// with a CTA barrier.
static __device__ void exchange_rows(const FaParams &p, const int (&grow)[2], int nr, float (&o)[2], const float (&lse)[2],
                              float *sh) {
    const int d = threadIdx.x, world = p.world, rank = p.rank, slot = p.seq & 1;
    const uint32_t tag32 = ex_tag(p.seq);
    const uint64_t tag = (uint64_t)tag32 << 32;
    for (int k = 0; k < nr; ++k)
        for (int q = 0; q < world; ++q) {
            if (q == rank) continue;
            uint64_t *dst = reinterpret_cast<uint64_t *>(p.peers[q]) +
                            (((size_t)slot * world + rank) * EX_ROWS + grow[k]) * EX_WORDS;
            st_word_sys(dst + d, tag | __float_as_uint(o[k]));
            if (d == 0) st_word_sys(dst + HD, tag | __float_as_uint(lse[k]));
        }
    uint64_t *own = reinterpret_cast<uint64_t *>(p.peers[rank]);
    auto word_of = [&](int q, int k, int col) {
        return own + (((size_t)slot * world + q) * EX_ROWS + grow[k]) * EX_WORDS + col;
    };
    // Every word this thread needs (its dimension of the other ranks' rows, and
    // on threads 32k + q the LSE of rank q's row k) is re-read together until all
    // carry this call's tag, so the waits for the peers overlap: one round trip
    // per pass, not one per word.
    const int lk = d >> 5, lq = d & 31;
    const bool lse_reader = lk < nr && lq < world && lq != rank;
    uint64_t w[2][EX_MAX_WORLD], wl = lse_reader ? ld_word_sys(word_of(lq, lk, HD)) : 0;
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int q = 0; q < EX_MAX_WORLD; ++q)
            w[k][q] = (k < nr && q < world && q != rank) ? ld_word_sys(word_of(q, k, d)) : ((uint64_t)tag32 << 32);
    const long long t0 = clock64();
    bool ok = true;
    while (true) {
        bool ready = !lse_reader || (uint32_t)(wl >> 32) == tag32;
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int q = 0; q < EX_MAX_WORLD; ++q) ready = ready && (uint32_t)(w[k][q] >> 32) == tag32;
        if (ready) break;
        if (clock64() - t0 > WAIT_LIMIT_CYCLES) { raise_status(STATUS_TIMEOUT); ok = false; break; }
        if (lse_reader && (uint32_t)(wl >> 32) != tag32) wl = ld_word_sys(word_of(lq, lk, HD));
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int q = 0; q < EX_MAX_WORLD; ++q)
                if (k < nr && q < world && q != rank && (uint32_t)(w[k][q] >> 32) != tag32) w[k][q] = ld_word_sys(word_of(q, k, d));
    }
    // read words are cleared (a late word of a timed-out call keeps its own tag)
    if (ok) {
        if (lse_reader) *word_of(lq, lk, HD) = 0;
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int q = 0; q < EX_MAX_WORLD; ++q)
                if (k < nr && q < world && q != rank) *word_of(q, k, d) = 0;
    }
    if (lk < nr && lq < world) sh[lk * EX_MAX_WORLD + lq] = lse_reader ? (ok ? __uint_as_float((uint32_t)wl) : 0.f) : lse[lk];
    float val[2][EX_MAX_WORLD];
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int q = 0; q < EX_MAX_WORLD; ++q) {
            val[k][q] = 0.f;
            if (k < nr && q < world) val[k][q] = q == rank ? o[k] : (ok ? __uint_as_float((uint32_t)w[k][q]) : 0.f);
        }
    const int all_ok = __syncthreads_and(ok);
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        float res = 0.f;
        if (all_ok && k < nr) {
            const float *ls = sh + k * EX_MAX_WORLD;
            float Mx = -INFINITY;
            for (int q = 0; q < world; ++q) Mx = fmaxf(Mx, ls[q]);
            float num = 0.f, den = 0.f;
            if (Mx != -INFINITY) {
#pragma unroll
                for (int q = 0; q < EX_MAX_WORLD; ++q) {
                    if (q >= world || ls[q] == -INFINITY) continue;
                    const float wq = expf(ls[q] - Mx);
                    den += wq;
                    num += wq * val[k][q];
                }
            }
            res = den > 0.f ? num / den : 0.f;
        }
        o[k] = res;
    }
    __syncthreads();                                   // sh is free again
}

// The decode tail of one CTA (all 256 threads): barrier over the KV head,
// then this CTA's rows of the head (blockIdx.x, blockIdx.x + splits, ...),
// two at a time, combined and written as p.tail says.  `scratch` is a little
// shared memory, `buf` room for two rows' partials of every split, `bar` an
// mbarrier (count 1) that no earlier phase of this launch used.
static __device__ void decode_tail(const FaParams &p, int g, uint8_t *scratch, float *buf, uint64_t *bar,
                            volatile int *abort_flag) {
    float *sh = reinterpret_cast<float *>(scratch);
    volatile int *flag = reinterpret_cast<volatile int *>(sh + 2 * MAXS + 8 + 2 * EX_MAX_WORLD);
    const int nrows = p.T * GROUP, d = threadIdx.x;
    auto global_row = [&](int r) { return (r / GROUP) * NQ + g * GROUP + r % GROUP; };
    // The gates of this CTA's first two rows load while the CTA waits at the barrier.
    auto load_gates = [&](int ra, int rb, float (&gate)[2]) {
        gate[0] = gate[1] = 0.f;
        if (p.tail == TAIL_SHARD) return;
        if (ra < nrows) gate[0] = p.q_gate[(size_t)global_row(ra) * 2 * HD + HD + d];
        if (rb >= 0) gate[1] = p.q_gate[(size_t)global_row(rb) * 2 * HD + HD + d];
    };
    float gate[2];
    {
        const int ra = blockIdx.x, rb = ra + p.splits < nrows ? ra + p.splits : -1;
        load_gates(ra, rb, gate);
    }
    if (!head_barrier(p.sync + g, p.splits, flag)) return;
    if (threadIdx.x == 0) QV_STAMP(7);
    uint32_t phase = 0;
    for (int ra = blockIdx.x; ra < nrows; ra += 2 * p.splits, phase ^= 1) {
        const int rb = ra + p.splits < nrows ? ra + p.splits : -1;
        const int nr = rb >= 0 ? 2 : 1;
        if (ra != (int)blockIdx.x) load_gates(ra, rb, gate);
        float o[2], lse[2];
        if (!combine_rows(p, g, ra, rb, sh, buf, bar, phase, abort_flag, o, lse)) return;
        const int grow[2] = {global_row(ra), nr == 2 ? global_row(rb) : 0};
        if (p.tail == TAIL_EXCHANGE) exchange_rows(p, grow, nr, o, lse, sh + 2 * MAXS + 8);
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            if (k >= nr) break;
            if (p.tail == TAIL_SHARD) {
                p.out[(size_t)grow[k] * HD + d] = o[k];
                if (d == 0) p.lse[grow[k]] = lse[k];
            } else {
                p.out[(size_t)grow[k] * HD + d] = o[k] * sigmoidf_(gate[k]);
            }
        }
    }
    if (threadIdx.x == 0) QV_STAMP(8);
}

// ---------------------------------------------------------------- decode phases
// The prepare step of a decode launch (its first 8 warps): the query rows are
// loaded, normalised, rotated and placed in TMEM as the A operand of the QK
// MMA.  Thread 0 calls `rows_arrived` once every warp's rows have arrived;
// `qstage` is 32 KB of shared memory that is idle until the first softmax (128
// A rows x 256 bytes); every warp arrives on q_ready at the end.
constexpr int QR = DECODE_ROWS / 8;              // query rows of a warp
template <class F>
__device__ __forceinline__ void prepare_queries(const FaParams &p, int kv_head, float2 *rope, uint8_t *qstage,
                                                uint32_t tmem, uint64_t *q_ready, F &&rows_arrived) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    float4 xa[QR], xb[QR], n0, n1;
    {
#pragma unroll
        for (int j = 0; j < QR; ++j) {
            const int rr = warp + 8 * j;
            if (rr < p.T * GROUP) {
                const float *src = p.q_gate + ((size_t)(rr / GROUP) * NQ + kv_head * GROUP + rr % GROUP) * 2 * HD;
                xa[j] = *reinterpret_cast<const float4 *>(src + 4 * lane);
                xb[j] = *reinterpret_cast<const float4 *>(src + 128 + 4 * lane);
            } else {
                xa[j] = xb[j] = make_float4(0.f, 0.f, 0.f, 0.f);
            }
        }
        n0 = *reinterpret_cast<const float4 *>(p.qn + 4 * lane);
        n1 = *reinterpret_cast<const float4 *>(p.qn + 128 + 4 * lane);
    }


    // Query rows r = warp + 8j: RMSNorm with weight, rotary on dims
    // [0,64), split into fp16 hi + lo (hi: the value truncated to fp16's
    // 11 significant bits, so that lo = x - hi is exact), placed in TMEM
    // A-row order (hi of row 16g+i at A row 32g+i, lo at 32g+16+i).  The
    // rows go to TMEM through the two P buffers (idle until the first
    // softmax, which needs these queries), in two rounds of 64 columns:
    // dims [0,128) then [128,256).  A staged A row is 256 bytes, 16-byte
    // chunks XOR-swizzled by the row's low 3 bits; in each round every
    // warp copies half the columns of its TMEM lane quarter.  Lane l of a row holds dims [4l,4l+4) and [128+4l,128+4l+4).
    // Rotary (cos, sin) of every (token, dim pair) while the loads are in flight.
    for (int e = threadIdx.x; e < p.T * 32; e += 256) rope[e] = rope_angle(p.position + (e >> 5), e & 31);
    float ss[QR];
#pragma unroll
    for (int j = 0; j < QR; ++j)
        ss[j] = xa[j].x * xa[j].x + xa[j].y * xa[j].y + xa[j].z * xa[j].z + xa[j].w * xa[j].w +
                xb[j].x * xb[j].x + xb[j].y * xb[j].y + xb[j].z * xb[j].z + xb[j].w * xb[j].w;
    named_barrier(1, 256);                                    // the rotary table is complete
    // Every warp has its query rows by now (it summed their squares before
    // the barrier), so the K/V tiles no longer queue in front of them.
    if (threadIdx.x == 0) rows_arrived();
#pragma unroll
    for (int o = 16; o; o >>= 1) {
#pragma unroll
        for (int j = 0; j < QR; ++j) ss[j] += __shfl_xor_sync(0xffffffffu, ss[j], o);
    }
    auto split = [](float a, float b, uint32_t &hi, uint32_t &lo) {
        const float ha = __uint_as_float(__float_as_uint(a) & 0xFFFFE000u);
        const float hb = __uint_as_float(__float_as_uint(b) & 0xFFFFE000u);
        hi = half2_bits(__floats2half2_rn(ha, hb));
        lo = half2_bits(__floats2half2_rn(a - ha, b - hb));
    };
    uint32_t hw[QR][2][4];                    // [row][round] {hi0, hi1, lo0, lo1}
#pragma unroll
    for (int j = 0; j < QR; ++j) {
        const int rr = warp + 8 * j;
        const bool live = rr < p.T * GROUP;
        const float inv = rsqrtf(ss[j] / HD + p.eps);
        const float4 a = xa[j], b = xb[j];
        float x0[4] = {a.x * inv * n0.x, a.y * inv * n0.y, a.z * inv * n0.z, a.w * inv * n0.w};
        const float x1[4] = {b.x * inv * n1.x, b.y * inv * n1.y, b.z * inv * n1.z, b.w * inv * n1.w};
        rope_row(x0, rope + (live ? rr / GROUP : 0) * 32, lane, live);
        split(x0[0], x0[1], hw[j][0][0], hw[j][0][2]);
        split(x0[2], x0[3], hw[j][0][1], hw[j][0][3]);
        split(x1[0], x1[1], hw[j][1][0], hw[j][1][2]);
        split(x1[2], x1[3], hw[j][1][1], hw[j][1][3]);
    }
    const int sub = (lane & 1) * 8;
    const int arow = (warp & 3) * 32 + lane, col_half = warp >> 2;
    const uint32_t qdst = tmem + ((uint32_t)((warp & 3) * 32) << 16) + TM_Q + col_half * 32;
#pragma unroll
    for (int round = 0; round < 2; ++round) {
#pragma unroll
        for (int j = 0; j < QR; ++j) {
            const int rr = warp + 8 * j;
            const int ahi = 32 * (rr >> 4) + (rr & 15);
            const int p0 = (((lane >> 1) ^ (ahi & 7)) << 4) + sub;
            *reinterpret_cast<uint2 *>(qstage + ahi * 256 + p0) = make_uint2(hw[j][round][0], hw[j][round][1]);
            *reinterpret_cast<uint2 *>(qstage + (ahi + 16) * 256 + p0) = make_uint2(hw[j][round][2], hw[j][round][3]);
        }
        named_barrier(2, 256);
        // Warp w: TMEM lanes 32*(w%4).., columns 64*round + [32*(w/4), 32*(w/4)+32).
        const uint8_t *mine = qstage + arow * 256;
#pragma unroll
        for (int m = 0; m < 2; ++m) {
            uint4 u[4];
#pragma unroll
            for (int e = 0; e < 4; ++e)
                u[e] = *reinterpret_cast<const uint4 *>(mine + (((col_half * 8 + 4 * m + e) ^ (lane & 7)) << 4));
            tmem_st16(qdst + round * 64 + m * 16, *reinterpret_cast<const float(*)[16]>(u));
        }
        if (round == 0) named_barrier(3, 256);    // every warp has read round 0 before it is overwritten
    }
    {
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(q_ready);
        if (threadIdx.x == 128) QV_STAMP(3);
    }
}

// The rows a decode launch appends: RMSNorm + rotary of the new keys, fp16 keys /
// values of the cache rows [lo, hi) of this CTA's tiles, one of two warps (k = 0 or 1).
__device__ __forceinline__ void append_rows(const FaParams &p, int kv_head, int k, int lo, int hi, const float2 *rope) {
    const int lane = threadIdx.x & 31;
    const float4 k0 = *reinterpret_cast<const float4 *>(p.kn + 4 * lane);
    const float4 k1 = *reinterpret_cast<const float4 *>(p.kn + 128 + 4 * lane);
    for (int row = lo + k; row < hi; row += 2) {
        const int tt = row - p.append_row0;
        const float *ks = p.key + ((size_t)tt * NKV + kv_head) * HD;
        const float *vs = p.value + ((size_t)tt * NKV + kv_head) * HD;
        const float4 a = *reinterpret_cast<const float4 *>(ks + 4 * lane);
        const float4 b = *reinterpret_cast<const float4 *>(ks + 128 + 4 * lane);
        const float4 va = *reinterpret_cast<const float4 *>(vs + 4 * lane);
        const float4 vb = *reinterpret_cast<const float4 *>(vs + 128 + 4 * lane);
        float sk = a.x * a.x + a.y * a.y + a.z * a.z + a.w * a.w + b.x * b.x + b.y * b.y + b.z * b.z +
                   b.w * b.w;
        sk = warp_sum(sk);
        const float inv = rsqrtf(sk / HD + p.eps);
        float x0[4] = {a.x * inv * k0.x, a.y * inv * k0.y, a.z * inv * k0.z, a.w * inv * k0.w};
        rope_row(x0, rope + tt * 32, lane, true);
        __half *kd = p.kc + ((size_t)row * NKV + kv_head) * HD;
        __half *vd = p.vc + ((size_t)row * NKV + kv_head) * HD;
        *reinterpret_cast<uint2 *>(kd + 4 * lane) =
            make_uint2(half2_bits(__floats2half2_rn(x0[0], x0[1])), half2_bits(__floats2half2_rn(x0[2], x0[3])));
        *reinterpret_cast<uint2 *>(kd + 128 + 4 * lane) =
            make_uint2(half2_bits(__floats2half2_rn(b.x * inv * k1.x, b.y * inv * k1.y)),
                       half2_bits(__floats2half2_rn(b.z * inv * k1.z, b.w * inv * k1.w)));
        *reinterpret_cast<uint2 *>(vd + 4 * lane) =
            make_uint2(half2_bits(__floats2half2_rn(va.x, va.y)), half2_bits(__floats2half2_rn(va.z, va.w)));
        *reinterpret_cast<uint2 *>(vd + 128 + 4 * lane) =
            make_uint2(half2_bits(__floats2half2_rn(vb.x, vb.y)), half2_bits(__floats2half2_rn(vb.z, vb.w)));
    }
}

// Epilogue of a decode CTA (its first 8 warps), once O is complete and the K/V
// ring idle.  Warps w and w+4 share TMEM lane quarter w%4 (O_hi of row
// 16(w%4)+i in lane i, O_lo in lane 16+i) and take O columns [0,128) (warps 4-7) and [128,256) (warps 0-3): each lane
// puts its lane's columns into a padded staging row, then the warp stores each
// of its rows, the sum of its hi and lo staging rows, as 512-byte pieces of
// this split's unnormalised partial.  `ring`: EPILOGUE_BYTES of shared memory.
constexpr int EPILOGUE_BYTES = 8 * 32 * (128 * 4 + 16);
__device__ __forceinline__ void store_partials(const FaParams &p, int kv_head, uint32_t tmem, uint8_t *ring) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, wq = warp & 3;
    const uint32_t t_lane = tmem + ((uint32_t)(wq * 32) << 16);
    tc_fence_after();
    if (threadIdx.x == 128) QV_STAMP(12);
    const int chalf = warp < 4 ? 1 : 0;
    constexpr int RS = 128 * 4 + 16;                       // staging row bytes (padded)
    uint8_t *stage = ring + warp * 32 * RS;
    uint8_t *myrow = stage + lane * RS;
    const uint32_t ocol = t_lane + TM_O + chalf * 128;
#pragma unroll
    for (int c4 = 0; c4 < 2; ++c4) {                       // 64 columns per TMEM round trip
        float o[4][16];
#pragma unroll
        for (int q = 0; q < 4; ++q) tmem_ld16(ocol + c4 * 64 + q * 16, o[q]);
        tmem_wait_ld();
#pragma unroll
        for (int q = 0; q < 4; ++q)
#pragma unroll
            for (int e = 0; e < 16; e += 4)
                *reinterpret_cast<float4 *>(myrow + (c4 * 64 + q * 16 + e) * 4) =
                    make_float4(o[q][e], o[q][e + 1], o[q][e + 2], o[q][e + 3]);
    }
    __syncwarp();
    if (threadIdx.x == 128) QV_STAMP(13);
    // The valid logical rows of a CTA are a prefix, so are this warp's.
    const int row0 = wq * 16;
    const int nvalid = max(0, min(16, p.T * GROUP - row0));
    const int col = 4 * lane;
#pragma unroll 4
    for (int i = 0; i < nvalid; ++i) {
        const int rr = row0 + i;
        float4 v = *reinterpret_cast<const float4 *>(stage + i * RS + col * 4);
        const float4 w = *reinterpret_cast<const float4 *>(stage + (i + 16) * RS + col * 4);
        v.x += w.x; v.y += w.y; v.z += w.z; v.w += w.w;
        float *dst = p.part_o + (((size_t)kv_head * DECODE_ROWS + rr) * p.splits + blockIdx.x) * HD;
        *reinterpret_cast<float4 *>(dst + chalf * 128 + col) = v;
    }
    if (threadIdx.x == 128) QV_STAMP(6);
}

// ---------------------------------------------------------------- host: split plan, workspace
namespace {
struct Split { int tiles, splits; };
// CTAs per KV head of a decode launch: a quarter of the SMs (37 on B200), so
// that the four heads fill one wave with one CTA per SM and the CTAs of a
// head, which meet at the tail barrier, are all resident at once.  Without a
// device (host-side size queries) the B200 figure is used.
inline int decode_ctas_per_head() {
    int dev = -1, sms = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) {
        cudaGetLastError();
        sms = 148;
    }
    return std::max(1, std::min(37, sms / NKV));
}
// Split-KV plan: whole tiles per split, at most decode_ctas_per_head() splits.
inline Split decode_split(int kv_rows) {
    const int total = std::max(1, (kv_rows + BN - 1) / BN);
    const int ctas = decode_ctas_per_head();
    const int per = (total + ctas - 1) / ctas;
    static_assert(37 <= MAXS, "the tail combine handles up to MAXS splits");
    return {per, (total + per - 1) / per};
}
inline size_t align256(size_t x) { return (x + 255) & ~size_t(255); }
inline bool decode_regime(int T) { return T * GROUP <= DECODE_ROWS; }

// Decode workspace: the tail barrier's words (256 bytes: one 64-bit word per
// KV head, generation : arrivals; the arrivals must be zero before the first
// launch on the workspace and every launch leaves them zero), then the split
// partials.
constexpr size_t SYNC_BYTES = 256;
struct DecodeParts { unsigned long long *sync; float *o, *ml; };
inline size_t decode_parts_bytes(const Split &sp) {
    return SYNC_BYTES + align256((size_t)NKV * sp.splits * DECODE_ROWS * HD * sizeof(float)) +
           align256((size_t)NKV * DECODE_ROWS * MAXS * 2 * sizeof(float));
}
inline DecodeParts decode_parts(void *ws, const Split &sp) {
    uint8_t *w = static_cast<uint8_t *>(ws);
    float *o = reinterpret_cast<float *>(w + SYNC_BYTES);
    float *ml = reinterpret_cast<float *>(w + SYNC_BYTES + align256((size_t)NKV * sp.splits * DECODE_ROWS * HD * sizeof(float)));
    return {reinterpret_cast<unsigned long long *>(w), o, ml};
}
}  // namespace

}  // namespace qv
