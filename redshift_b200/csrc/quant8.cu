// Quantisation into the two 8-bit forms of the serving path, and back.
//
//   cache8: int8 codes of fp16 K/V rows with a scale for every 64 tokens and
//     head, scale = max|x| / 127 and code = x / scale rounded to the nearest
//     integer (ties to even).  Codes are laid out [block][4 heads][64][256], so
//     that a block of one head, the tile attention reads, is 16 KB in a row.
//   norm8: e4m3 codes of fp32 rows with a scale for every row and 128 columns,
//     scale = max|y| / 448, y either the row itself or its RMSNorm after the
//     addition of a residual.  Scales are laid out [column block][row], the
//     order in which the product (mm8.cu) reads them.
//
// A block that holds a value which is not finite gets the scale NaN (and codes
// of zero): whatever is computed from it is NaN, as it would be without codes.
// All four kernels are bound by memory; every value is read and written once.
#include "common.cuh"
#include "hotpath.h"

#include <stdexcept>
#include <string>

namespace qv {
namespace {

constexpr int KV = 4, HD8 = 256, BLK = CACHE8_BLOCK;
constexpr int CODES = BLK * HD8;                 // codes of one (block, head)

__device__ __forceinline__ __half2 as_half2(uint32_t v) { return *reinterpret_cast<const __half2 *>(&v); }
__device__ __forceinline__ uint32_t half2_word(__half2 h) { return *reinterpret_cast<const uint32_t *>(&h); }

// x / s rounded to the nearest integer, ties to even, exactly: the product
// with the approximate reciprocal is off by one at most, and the sign of
// x - (q +- 1/2) s, which one fused multiply-add gives without error, says
// which side of the border x lies on.
__device__ __forceinline__ int nearest_code(float x, float s, float inv) {
    const float q = rintf(x * inv);
    const float above = fmaf(-(q + 0.5f), s, x), below = fmaf(-(q - 0.5f), s, x);
    const int n = (int)q, odd = n & 1;
    return n + ((above > 0.f || (above == 0.f && odd)) ? 1 : 0) - ((below < 0.f || (below == 0.f && odd)) ? 1 : 0);
}

struct Cache8Side {
    int8_t *codes;
    float *scales;
    __half *rows;
};
struct Cache8Params {
    Cache8Side k, v;
    int begin, end, ring;       // rows [begin, end); source row r at r % ring
};

// One CTA of 256 threads per (block, head, K or V): warp w takes rows w + 8 i,
// lane l the dims [8 l, 8 l + 8), all 64 rows in registers between the maximum
// and the codes, so the 32 KB are read once.
__global__ void __launch_bounds__(256) cache8_pack_kernel(const Cache8Params p) {
    const Cache8Side side = blockIdx.z ? p.v : p.k;
    const int head = blockIdx.y, block = p.begin / BLK + blockIdx.x;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    __shared__ uint32_t red[8];
    grid_dependency_wait();
    if (threadIdx.x == 0) launch_dependents();
    const int first = (int)((size_t)block * BLK % p.ring);      // a block never wraps inside the ring
    const __half *src = side.rows + ((size_t)first * KV + head) * HD8 + 8 * lane;
    uint4 x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = *reinterpret_cast<const uint4 *>(src + (size_t)(warp + 8 * i) * KV * HD8);
    // The magnitudes' bit patterns order like the values, infinity and NaN above all others.
    __half2 m = as_half2(0u);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        m = __hmax2_nan(m, __hmax2_nan(__hmax2_nan(__habs2(as_half2(x[i].x)), __habs2(as_half2(x[i].y))),
                                       __hmax2_nan(__habs2(as_half2(x[i].z)), __habs2(as_half2(x[i].w)))));
    }
    const uint32_t mb = half2_word(m);
    uint32_t bits = __reduce_max_sync(0xffffffffu, max(mb & 0x7FFFu, (mb >> 16) & 0x7FFFu));
    if (lane == 0) red[warp] = bits;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; ++i) bits = max(bits, red[i]);
    const bool finite = bits < 0x7C00u;
    const float scale = finite ? __fdiv_rn(__half2float(__ushort_as_half((unsigned short)bits)), 127.f)
                               : __int_as_float(0x7FC00000);
    const size_t tile = (size_t)block * KV + head;
    if (threadIdx.x == 0) side.scales[tile] = scale;
    const bool live = finite && bits != 0;
    const float inv = live ? __frcp_rn(scale) : 0.f;
    int8_t *dst = side.codes + tile * CODES + 8 * lane;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        uint32_t out[2] = {0u, 0u};
        if (live) {
            const uint32_t w[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float2 f = __half22float2(as_half2(w[e]));
                const uint32_t a = (uint32_t)nearest_code(f.x, scale, inv) & 0xFFu;
                const uint32_t b = (uint32_t)nearest_code(f.y, scale, inv) & 0xFFu;
                out[e >> 1] |= (a | b << 8) << (16 * (e & 1));
            }
        }
        *reinterpret_cast<uint2 *>(dst + (size_t)(warp + 8 * i) * HD8) = make_uint2(out[0], out[1]);
    }
}

// One CTA per (block, head, K or V) that [begin, end) touches: thread =
// 16 codes of a row, four rows each; fp16(code * scale).
__global__ void __launch_bounds__(256) cache8_unpack_kernel(const Cache8Params p) {
    const Cache8Side side = blockIdx.z ? p.v : p.k;
    const int head = blockIdx.y, block = p.begin / BLK + blockIdx.x;
    grid_dependency_wait();
    if (threadIdx.x == 0) launch_dependents();
    const size_t tile = (size_t)block * KV + head;
    const float scale = side.scales[tile];
    const int col = (threadIdx.x & 15) * 16, row0 = threadIdx.x >> 4;
    const int8_t *src = side.codes + tile * CODES + col;
    uint4 c[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int r = block * BLK + row0 + 16 * i;
        c[i] = r >= p.begin && r < p.end ? *reinterpret_cast<const uint4 *>(src + (size_t)(row0 + 16 * i) * HD8)
                                         : make_uint4(0u, 0u, 0u, 0u);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int r = block * BLK + row0 + 16 * i;
        if (r < p.begin || r >= p.end) continue;
        const uint32_t w[4] = {c[i].x, c[i].y, c[i].z, c[i].w};
        uint32_t h[8];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float a = (float)(int8_t)(w[e] & 0xFFu), b = (float)(int8_t)(w[e] >> 8 & 0xFFu);
            const float d = (float)(int8_t)(w[e] >> 16 & 0xFFu), f = (float)(int8_t)(w[e] >> 24);
            h[2 * e] = half2_word(__floats2half2_rn(a * scale, b * scale));
            h[2 * e + 1] = half2_word(__floats2half2_rn(d * scale, f * scale));
        }
        uint4 *dst = reinterpret_cast<uint4 *>(side.rows + ((size_t)(r - p.begin) * KV + head) * HD8 + col);
        dst[0] = make_uint4(h[0], h[1], h[2], h[3]);
        dst[1] = make_uint4(h[4], h[5], h[6], h[7]);
    }
}

// ---------------------------------------------------------------- norm8
struct Norm8Params {
    uint8_t *codes;
    float *scales, *sum_out, *normed;
    const float *x, *residual, *weights;
    int tokens, width, blocks;
    float eps;
};

// Four e4m3 codes, round to nearest even, of four floats.
__device__ __forceinline__ uint32_t e4m3x4(float a, float b, float c, float d) {
    uint16_t lo, hi;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b), "f"(a));
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d), "f"(c));
    return (uint32_t)lo | (uint32_t)hi << 16;
}

// One CTA per row.  A warp takes every (warps)-th block of 128 columns, lane l
// the columns [4 l, 4 l + 4) of it, up to PER_WARP blocks in registers, so the
// row is read once, its sum of squares meets in shared memory, and a block's
// maximum is a reduction inside one warp.  VEC: rows are 16-byte aligned.
constexpr int PER_WARP = 5, MAX_WARPS = 28;   // 140 blocks: 17,920 columns
template <bool NORM, bool VEC>
__global__ void __launch_bounds__(32 * MAX_WARPS) norm8_kernel(const Norm8Params p) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
    const int token = blockIdx.x;
    const size_t row = (size_t)token * p.width;
    __shared__ float red[32];
    grid_dependency_wait();
    if (threadIdx.x == 0) launch_dependents();
    float v[PER_WARP][4];
    auto load = [&](const float *src, int c, float (&d)[4]) {
        if (VEC) {
            const float4 f = c < p.width ? *reinterpret_cast<const float4 *>(src + c) : make_float4(0.f, 0.f, 0.f, 0.f);
            d[0] = f.x; d[1] = f.y; d[2] = f.z; d[3] = f.w;
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) d[e] = c + e < p.width ? src[c + e] : 0.f;
        }
    };
    auto store = [&](float *dst, int c, const float (&d)[4]) {
        if (VEC) {
            if (c < p.width) *reinterpret_cast<float4 *>(dst + c) = make_float4(d[0], d[1], d[2], d[3]);
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (c + e < p.width) dst[c + e] = d[e];
        }
    };
#pragma unroll
    for (int i = 0; i < PER_WARP; ++i) load(p.x + row, (warp + i * warps) * 128 + 4 * lane, v[i]);
    if (NORM) {
        if (p.residual) {
            float r[PER_WARP][4];
#pragma unroll
            for (int i = 0; i < PER_WARP; ++i) load(p.residual + row, (warp + i * warps) * 128 + 4 * lane, r[i]);
#pragma unroll
            for (int i = 0; i < PER_WARP; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) v[i][e] += r[i][e];
        }
        float w[PER_WARP][4], ss[PER_WARP];
#pragma unroll
        for (int i = 0; i < PER_WARP; ++i) load(p.weights, (warp + i * warps) * 128 + 4 * lane, w[i]);
#pragma unroll
        for (int i = 0; i < PER_WARP; ++i)
            ss[i] = (v[i][0] * v[i][0] + v[i][1] * v[i][1]) + (v[i][2] * v[i][2] + v[i][3] * v[i][3]);
        const float s = warp_sum((ss[0] + ss[1]) + (ss[2] + ss[3]) + ss[4]);
        if (lane == 0) red[warp] = s;
        __syncthreads();
        const float all = warp_sum(lane < warps ? red[lane] : 0.f);
        const float inv = __frsqrt_rn(__fdiv_rn(all, (float)p.width) + p.eps);
#pragma unroll
        for (int i = 0; i < PER_WARP; ++i) {
            const int c = (warp + i * warps) * 128 + 4 * lane;
            if (p.sum_out) store(p.sum_out + row, c, v[i]);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[i][e] = v[i][e] * inv * w[i][e];
            if (p.normed) store(p.normed + row, c, v[i]);
        }
    }
#pragma unroll
    for (int i = 0; i < PER_WARP; ++i) {
        const int block = warp + i * warps, c = block * 128 + 4 * lane;
        if (block >= p.blocks) continue;                       // the same for the whole warp
        // The magnitudes' bits order like the values, infinity and NaN above all others.
        const uint32_t own = max(max(__float_as_uint(v[i][0]) & 0x7FFFFFFFu, __float_as_uint(v[i][1]) & 0x7FFFFFFFu),
                                 max(__float_as_uint(v[i][2]) & 0x7FFFFFFFu, __float_as_uint(v[i][3]) & 0x7FFFFFFFu));
        const uint32_t bits = __reduce_max_sync(0xffffffffu, own);
        const bool finite = bits < 0x7F800000u;
        const float scale = finite ? __fdiv_rn(__uint_as_float(bits), 448.f) : __int_as_float(0x7FC00000);
        if (lane == 0) p.scales[(size_t)block * p.tokens + token] = scale;
        uint32_t codes = 0u;
        if (finite && scale > 0.f)
            codes = e4m3x4(__fdiv_rn(v[i][0], scale), __fdiv_rn(v[i][1], scale), __fdiv_rn(v[i][2], scale),
                           __fdiv_rn(v[i][3], scale));
        if (VEC) {
            if (c < p.width) *reinterpret_cast<uint32_t *>(p.codes + row + c) = codes;
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (c + e < p.width) p.codes[row + c + e] = (uint8_t)(codes >> (8 * e));
        }
    }
}

void launched(cudaError_t e, const char *what) {
    if (e != cudaSuccess) throw std::runtime_error(std::string(what) + ": " + cudaGetErrorString(e));
}
bool aligned(const void *a, size_t to) { return reinterpret_cast<uintptr_t>(a) % to == 0; }

}  // namespace

void cache8_pack(int8_t *kc, float *ks, int8_t *vc, float *vs, const __half *k, const __half *v, int begin, int end,
                 int ring, cudaStream_t st) {
    if (begin == end) return;
    const Cache8Params p{{kc, ks, const_cast<__half *>(k)}, {vc, vs, const_cast<__half *>(v)}, begin, end, ring};
    launched(launch_chained(cache8_pack_kernel, dim3((end - begin) / BLK, KV, 2), dim3(256), 0, st, p), "cache pack");
}

void cache8_unpack(__half *k, __half *v, const int8_t *kc, const float *ks, const int8_t *vc, const float *vs, int begin,
                   int end, cudaStream_t st) {
    if (begin == end) return;
    const Cache8Params p{{const_cast<int8_t *>(kc), const_cast<float *>(ks), k},
                         {const_cast<int8_t *>(vc), const_cast<float *>(vs), v}, begin, end, 0};
    launched(launch_chained(cache8_unpack_kernel, dim3((end + BLK - 1) / BLK - begin / BLK, KV, 2), dim3(256), 0, st, p),
             "cache unpack");
}

void norm8(uint8_t *codes, float *scales, float *sum_out, float *normed, const float *x, const float *residual,
           const float *weights, int tokens, int width, float eps, cudaStream_t st) {
    Norm8Params p{codes, scales, sum_out, normed, x, residual, weights, tokens, width, (width + 127) / 128, eps};
    const bool vec = width % 4 == 0 && aligned(codes, 4) && aligned(x, 16) && aligned(residual, 16) && aligned(weights, 16) &&
                     aligned(sum_out, 16) && aligned(normed, 16);
    // warps that hold the row in registers: PER_WARP blocks of 128 columns each
    int warps = (p.blocks + PER_WARP - 1) / PER_WARP;
    if (warps > MAX_WARPS) throw std::invalid_argument("the row is wider than a block of threads holds");
    auto kernel = weights ? (vec ? norm8_kernel<true, true> : norm8_kernel<true, false>)
                          : (vec ? norm8_kernel<false, true> : norm8_kernel<false, false>);
    launched(launch_chained(kernel, dim3(tokens), dim3(32 * warps), 0, st, p), weights ? "norm8" : "quantize8");
}

}  // namespace qv
