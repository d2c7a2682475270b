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
// All four kernels are bound by memory; every value is read and written once:
// packing and unpacking 32,768 rows takes 74 us (402 MB, 5.4 TB/s; 6.5 is the
// rate of a plain copy), 64 rows 5.3 us, two launches of a latency each.
#include "common.cuh"
#include "hotpath.h"

#include <algorithm>
#include <stdexcept>
#include <string>

namespace qv {
namespace {

constexpr int KV = 4, HD8 = 256, BLK = CACHE8_BLOCK;
constexpr int CODES = BLK * HD8;                 // codes of one (block, head)

__device__ __forceinline__ __half2 as_half2(uint32_t v) { return *reinterpret_cast<const __half2 *>(&v); }
__device__ __forceinline__ uint32_t half2_word(__half2 h) { return *reinterpret_cast<const uint32_t *>(&h); }

// Four codes: x / s rounded to the nearest integer, ties to even, exactly.
// Adding 1.5 * 2^23 to x times the approximate reciprocal leaves the integer q
// in the low bits, at most one off.  x - q s is exact: it is a multiple of the
// last place of s and no larger than s (where the last place of x is finer, |x|
// < s / 2 and q = 0).  So |x - q s| >= s / 2 tells the few q that may be
// wrong, and its sign the side.
__device__ __forceinline__ uint32_t nearest_codes(float4 x, float s, float inv) {
    constexpr float magic = 12582912.f;
    const float v[4] = {x.x, x.y, x.z, x.w}, half = 0.5f * s;
    uint32_t t[4];
    float far = 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const float sum = fmaf(v[e], inv, magic);
        t[e] = __float_as_uint(sum);
        far = fmaxf(far, fabsf(fmaf(magic - sum, s, v[e])));
    }
    if (far >= half) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float rest = fmaf(magic - __uint_as_float(t[e]), s, v[e]);
            const bool odd = t[e] & 1u;
            if (rest > half || (rest == half && odd)) ++t[e];
            else if (rest < -half || (rest == -half && odd)) --t[e];
        }
    }
    return __byte_perm(__byte_perm(t[0], t[1], 0x0040), __byte_perm(t[2], t[3], 0x0040), 0x5410);
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
            const float2 a = __half22float2(as_half2(x[i].x)), b = __half22float2(as_half2(x[i].y));
            const float2 c = __half22float2(as_half2(x[i].z)), d = __half22float2(as_half2(x[i].w));
            out[0] = nearest_codes(make_float4(a.x, a.y, b.x, b.y), scale, inv);
            out[1] = nearest_codes(make_float4(c.x, c.y, d.x, d.y), scale, inv);
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
            // the byte code + 128 as the last byte of 2^23 + it; subtracting leaves the code
            const uint32_t u = w[e] ^ 0x80808080u;
            float f[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) f[k] = (__uint_as_float(__byte_perm(u, 0x4B000000u, 0x7540 + k)) - 8388736.f) * scale;
            h[2 * e] = half2_word(__floats2half2_rn(f[0], f[1]));
            h[2 * e + 1] = half2_word(__floats2half2_rn(f[2], f[3]));
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

// Columns [c, c + 4) of a row, zero past its end.  VEC: rows are 16-byte aligned.
template <bool VEC> __device__ __forceinline__ void load_columns(const float *src, int c, int width, float (&d)[4]) {
    if (VEC) {
        const float4 f = c < width ? *reinterpret_cast<const float4 *>(src + c) : make_float4(0.f, 0.f, 0.f, 0.f);
        d[0] = f.x; d[1] = f.y; d[2] = f.z; d[3] = f.w;
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) d[e] = c + e < width ? src[c + e] : 0.f;
    }
}
template <bool VEC> __device__ __forceinline__ void store_columns(float *dst, int c, int width, const float (&d)[4]) {
    if (VEC) {
        if (c < width) *reinterpret_cast<float4 *>(dst + c) = make_float4(d[0], d[1], d[2], d[3]);
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (c + e < width) dst[c + e] = d[e];
    }
}
// Scale and codes of one block of 128 columns, spread over a warp, lane l with [4 l, 4 l + 4).
template <bool VEC>
__device__ __forceinline__ void store_codes(const Norm8Params &p, int token, int block, int lane, const float (&v)[4]) {
    // The magnitudes' bits order like the values, infinity and NaN above all others.
    const uint32_t own = max(max(__float_as_uint(v[0]) & 0x7FFFFFFFu, __float_as_uint(v[1]) & 0x7FFFFFFFu),
                             max(__float_as_uint(v[2]) & 0x7FFFFFFFu, __float_as_uint(v[3]) & 0x7FFFFFFFu));
    const uint32_t bits = __reduce_max_sync(0xffffffffu, own);
    const bool finite = bits < 0x7F800000u;
    const float scale = finite ? __fdiv_rn(__uint_as_float(bits), 448.f) : __int_as_float(0x7FC00000);
    if (lane == 0) p.scales[(size_t)block * p.tokens + token] = scale;
    uint32_t codes = 0u;
    if (finite && scale > 0.f) {
        float q[4];
        if (scale > 0x1p-100f) {
            // Markstein's division: the quotient from the correctly rounded reciprocal, corrected
            // once by its exact remainder (P. Markstein, IBM J. Res. Dev. 34, 1990)
            const float inv = __frcp_rn(scale);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float near = v[e] * inv;
                q[e] = fmaf(fmaf(-near, scale, v[e]), inv, near);
            }
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) q[e] = __fdiv_rn(v[e], scale);
        }
        codes = e4m3x4(q[0], q[1], q[2], q[3]);
    }
    const int c = block * 128 + 4 * lane;
    uint8_t *dst = p.codes + (size_t)token * p.width + c;
    if (VEC) {
        if (c < p.width) *reinterpret_cast<uint32_t *>(dst) = codes;
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (c + e < p.width) dst[e] = (uint8_t)(codes >> (8 * e));
    }
}

// One CTA per row.  A warp takes every (warps)-th block of 128 columns, up to
// PER_WARP of them in registers, so the row is read once, its sum of squares
// meets in shared memory, and a block's maximum is a reduction inside one warp.
// 4,096 rows x 5,120 with a residual: 45 us (272 MB, 6.0 TB/s); one row 3.4 us.
constexpr int PER_WARP = 5, MAX_WARPS = 28;   // 140 blocks: 17,920 columns
// The row's sum of all lanes' values (`red`: one float of each warp).
__device__ __forceinline__ float row_sum(float *red, float v, int warp, int lane, int warps) {
    const float s = warp_sum(v);
    if (lane == 0) red[warp] = s;
    __syncthreads();
    return warp_sum(lane < warps ? red[lane] : 0.f);
}
template <bool VEC>
__global__ void __launch_bounds__(32 * MAX_WARPS) norm8_kernel(const Norm8Params p) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
    const int token = blockIdx.x;
    const size_t row = (size_t)token * p.width;
    __shared__ float red[2][32];
    grid_dependency_wait();
    if (threadIdx.x == 0) launch_dependents();
    float v[PER_WARP][4], w[PER_WARP][4];
#pragma unroll
    for (int i = 0; i < PER_WARP; ++i) load_columns<VEC>(p.x + row, (warp + i * warps) * 128 + 4 * lane, p.width, v[i]);
    if (p.residual) {
        float r[PER_WARP][4];
#pragma unroll
        for (int i = 0; i < PER_WARP; ++i)
            load_columns<VEC>(p.residual + row, (warp + i * warps) * 128 + 4 * lane, p.width, r[i]);
#pragma unroll
        for (int i = 0; i < PER_WARP; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) v[i][e] += r[i][e];
    }
#pragma unroll
    for (int i = 0; i < PER_WARP; ++i) load_columns<VEC>(p.weights, (warp + i * warps) * 128 + 4 * lane, p.width, w[i]);
    auto squares = [&](float f) {                 // of this lane's columns times f
        float ss[PER_WARP];
#pragma unroll
        for (int i = 0; i < PER_WARP; ++i) {
            const float a = v[i][0] * f, b = v[i][1] * f, c = v[i][2] * f, d = v[i][3] * f;
            ss[i] = (a * a + b * b) + (c * c + d * d);
        }
        return (ss[0] + ss[1]) + (ss[2] + ss[3]) + ss[4];
    };
    float all = row_sum(red[0], squares(1.f), warp, lane, warps), inv = __frsqrt_rn(__fdiv_rn(all, (float)p.width) + p.eps);
    if (all > 0x1p126f) {                         // squares beyond fp32: those of the row times 2^-64
        all = row_sum(red[1], squares(0x1p-64f), warp, lane, warps);
        inv = __frsqrt_rn(__fdiv_rn(all, (float)p.width)) * 0x1p-64f;
    }
#pragma unroll
    for (int i = 0; i < PER_WARP; ++i) {
        const int block = warp + i * warps, c = block * 128 + 4 * lane;
        if (p.sum_out) store_columns<VEC>(p.sum_out + row, c, p.width, v[i]);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[i][e] = v[i][e] * inv * w[i][e];
        if (p.normed) store_columns<VEC>(p.normed + row, c, p.width, v[i]);
        if (block < p.blocks) store_codes<VEC>(p, token, block, lane, v[i]);
    }
}

// The codes alone: every warp takes QUANT_BLOCKS blocks of 128 columns of a row,
// independent of all others.  1999 tokens x 17408: 34.0 us (5.2 TB/s) with two
// blocks a warp and eight CTAs on an SM, 35.1 with four, 43.8 with eight; a call of
// 8 tokens x 6144 takes 2.0, 2.5 and 3.5 us.
constexpr int QUANT_BLOCKS = 2;
template <bool VEC>
__global__ void __launch_bounds__(256, 8) quantize8_kernel(const Norm8Params p) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, token = blockIdx.x;
    const int block0 = (blockIdx.y * 8 + warp) * QUANT_BLOCKS;
    const size_t row = (size_t)token * p.width;
    grid_dependency_wait();
    if (threadIdx.x == 0) launch_dependents();
    float v[QUANT_BLOCKS][4];
#pragma unroll
    for (int i = 0; i < QUANT_BLOCKS; ++i) load_columns<VEC>(p.x + row, (block0 + i) * 128 + 4 * lane, p.width, v[i]);
#pragma unroll
    for (int i = 0; i < QUANT_BLOCKS; ++i)
        if (block0 + i < p.blocks) store_codes<VEC>(p, token, block0 + i, lane, v[i]);
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
    if (!weights) {
        const dim3 grid(tokens, (p.blocks + 8 * QUANT_BLOCKS - 1) / (8 * QUANT_BLOCKS));
        const int warps = std::min(8, (p.blocks + QUANT_BLOCKS - 1) / QUANT_BLOCKS);
        launched(launch_chained(vec ? quantize8_kernel<true> : quantize8_kernel<false>, grid, dim3(32 * warps), 0, st, p), "quantize8");
        return;
    }
    // warps that hold the row in registers: PER_WARP blocks of 128 columns each
    const int warps = (p.blocks + PER_WARP - 1) / PER_WARP;
    if (warps > MAX_WARPS) throw std::invalid_argument("the row is wider than a block of threads holds");
    launched(launch_chained(vec ? norm8_kernel<true> : norm8_kernel<false>, dim3(tokens), dim3(32 * warps), 0, st, p), "norm8");
}

}  // namespace qv
