// Residual addition, root-mean-square norm and MX quantiser in one pass over a row:
//   h = bf16(x + residual);   y = h / sqrt(mean(h^2) + eps) * weight;   codes, scales = MX(y)
// The norm reads h as it is stored (the next layer adds to the stored value, so both see the same stream); everything after
// it stays in fp32 and is rounded once, to the code.  Block rule as in mx_quant.cuh, on the fp32 values: E = biased exponent
// of the block's largest |y|, scale byte E - emax, code = RNE with saturation of y * 2^(127 - byte).
//
// Bound by memory: 4 bytes read and 3 + 1/32 written per element with a residual.  A row lives in the registers of the warps
// that share it (16 elements a lane and pass: one full-sector load each for x and the residual), so that nothing is read
// twice; the sum of squares crosses the warps through shared memory once.
#pragma once

#include <cuda_bf16.h>

#include "common.cuh"
#include "mx_quant.cuh"

namespace catccos {

constexpr uint32_t kNormColsPerWarp = 512;   // 32 lanes x 16 elements
constexpr uint32_t kNormMaxWarps = 16;       // of one row
constexpr uint32_t kNormMaxPasses = 4;
constexpr uint32_t kNormMaxCols = kNormColsPerWarp * kNormMaxWarps * kNormMaxPasses;
constexpr float kNormMinEps = 1e-30f;  // squares that fp32 holds as denormals do not count beside it

struct NormQuantParams {
    const uint8_t* x;          // bf16 [rows, n]
    const uint8_t* residual;   // bf16 [rows, n] or nullptr
    const uint8_t* weight;     // bf16 [n]
    uint8_t* residual_out;     // bf16 [rows, n], h (with a residual only; may be residual or x)
    uint8_t* norm_out;         // bf16 [rows, n] or nullptr
    uint8_t* codes;            // [rows, n]
    uint8_t* scales;           // [rows, n / 32]
    uint32_t rows, n;
    float eps, inv_n;
    uint32_t device_tiny;
};

__device__ __forceinline__ float2 bf16x2_to_f32(uint32_t v)
{
    return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xFFFF0000u));
}

// Scale byte and multiplier for a block whose largest |value| is the fp32 amax: block_scale() of the bf16 quantiser, with the
// fp32 exponent, which has the same bias.
__device__ __forceinline__ void block_scale_f32(float amax, bool device_tiny, uint32_t emax, uint32_t& byte, float& mul, bool& nonfinite)
{
    const uint32_t E = __float_as_uint(amax) >> 23;  // amax >= 0
    nonfinite = E == 0xFFu;
    if (device_tiny) {
        byte = E > emax ? E - emax : 0u;
        mul = byte == 0u ? 0.0f : __uint_as_float((254u - byte) << 23);
    } else {
        const bool tiny = amax < 1e-12f;
        byte = tiny ? 0x7Fu : E - emax;
        mul = tiny ? 0.0f : __uint_as_float((254u - byte) << 23);
    }
    if (nonfinite) {
        byte = 0xFFu;
    }
}

// |a| or |b|, whichever is larger, as ordered bits: a NaN counts as larger than any number
__device__ __forceinline__ uint32_t max_abs_bits(uint32_t m, float v) { return max(m, __float_as_uint(v) & 0x7FFFFFFFu); }

__device__ __forceinline__ void store_half_block(void* p, const uint32_t (&v)[8])
{
    if (((uintptr_t)p & 31u) == 0u) {
        st_global_v8(p, v);
    } else {
        static_cast<uint4*>(p)[0] = make_uint4(v[0], v[1], v[2], v[3]);
        static_cast<uint4*>(p)[1] = make_uint4(v[4], v[5], v[6], v[7]);
    }
}

// The sum over the lanes of the warps that share a row, the same on all of them.
__device__ __forceinline__ float row_sum(float sum, float* partial, uint32_t warps_per_row)
{
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
#pragma unroll
    for (uint32_t d = 16; d > 0; d >>= 1) {
        sum += __shfl_xor_sync(0xFFFFFFFFu, sum, d);
    }
    if (warps_per_row > 1u) {
        if (lane == 0) {
            partial[warp] = sum;
        }
        __syncthreads();
        sum = lane < warps_per_row ? partial[lane] : 0.0f;
#pragma unroll
        for (uint32_t d = 8; d > 0; d >>= 1) {
            sum += __shfl_xor_sync(0xFFFFFFFFu, sum, d);
        }
        sum = __shfl_sync(0xFFFFFFFFu, sum, 0);
    }
    return sum;
}

// kPasses passes of warps_per_row x 512 columns cover a row; blockDim.x = 32 * warps_per_row * rows_per_cta.  With several rows
// to a CTA each has one warp (rows_per_cta > 1 only then), and nothing crosses warps.
template <uint32_t kPasses, bool kE5m2>
__global__ void __launch_bounds__(32 * kNormMaxWarps) add_rms_norm_mx_quant_kernel(const NormQuantParams p, uint32_t warps_per_row)
{
    __shared__ float partial[kNormMaxWarps];
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
    const uint32_t rows_per_cta = (blockDim.x >> 5) / warps_per_row;
    const uint32_t row = blockIdx.x * rows_per_cta + warp / warps_per_row;
    const uint32_t row_warp = warp % warps_per_row;
    const bool live = row < p.rows;
    grid_dep_wait();
    grid_dep_launch();

    uint32_t h[kPasses][8];
    float sum = 0.0f;
#pragma unroll
    for (uint32_t i = 0; i < kPasses; ++i) {
        const uint32_t col = (i * warps_per_row + row_warp) * kNormColsPerWarp + lane * 16u;
        uint4 a[2] = {}, b[2] = {};
        const size_t at = ((size_t)row * p.n + col) * 2u;
        const bool inside = live && col < p.n;
        if (inside) {
            load_half_block(p.x + at, a[0], a[1]);
            if (p.residual != nullptr) {
                load_half_block(p.residual + at, b[0], b[1]);
            }
        }
        const uint32_t av[8] = {a[0].x, a[0].y, a[0].z, a[0].w, a[1].x, a[1].y, a[1].z, a[1].w};
        const uint32_t bv[8] = {b[0].x, b[0].y, b[0].z, b[0].w, b[1].x, b[1].y, b[1].z, b[1].w};
#pragma unroll
        for (uint32_t j = 0; j < 8; ++j) {
            h[i][j] = av[j];
            float2 f = bf16x2_to_f32(av[j]);
            if (p.residual != nullptr) {
                const float2 r = bf16x2_to_f32(bv[j]);
                const __nv_bfloat162 s = __floats2bfloat162_rn(f.x + r.x, f.y + r.y);
                h[i][j] = *reinterpret_cast<const uint32_t*>(&s);
                f = bf16x2_to_f32(h[i][j]);
            }
            sum = fmaf(f.x, f.x, fmaf(f.y, f.y, sum));
        }
        if (inside && p.residual != nullptr) {
            store_half_block(p.residual_out + at, h[i]);
        }
    }
    sum = row_sum(sum, partial, warps_per_row);
    float inv = 1.0f / sqrtf(fmaf(sum, p.inv_n, p.eps));
    if (isinf(sum)) {  // |h| beyond 1e16; the same on all warps of a row, and a CTA with several warps to a row has one row
        sum = 0.0f;
#pragma unroll
        for (uint32_t i = 0; i < kPasses; ++i) {
#pragma unroll
            for (uint32_t j = 0; j < 8; ++j) {
                const float2 f = bf16x2_to_f32(h[i][j]);
                sum = fmaf(f.x * 0x1p-72f, f.x * 0x1p-72f, fmaf(f.y * 0x1p-72f, f.y * 0x1p-72f, sum));
            }
        }
        if (warps_per_row > 1u) {
            __syncthreads();  // all have read partial
        }
        sum = row_sum(sum, partial, warps_per_row);
        inv = 0x1p-72f / sqrtf(sum * p.inv_n);  // eps is nothing beside it
    }

#pragma unroll
    for (uint32_t i = 0; i < kPasses; ++i) {
        const uint32_t col = (i * warps_per_row + row_warp) * kNormColsPerWarp + lane * 16u;
        const bool inside = live && col < p.n;
        uint4 w[2] = {};
        if (inside) {
            w[0] = *reinterpret_cast<const uint4*>(p.weight + col * 2u);
            w[1] = *(reinterpret_cast<const uint4*>(p.weight + col * 2u) + 1);
        }
        const uint32_t wv[8] = {w[0].x, w[0].y, w[0].z, w[0].w, w[1].x, w[1].y, w[1].z, w[1].w};
        float y[16];
        uint32_t top = 0;
#pragma unroll
        for (uint32_t j = 0; j < 8; ++j) {
            const float2 f = bf16x2_to_f32(h[i][j]), g = bf16x2_to_f32(wv[j]);
            y[2 * j] = f.x * inv * g.x;
            y[2 * j + 1] = f.y * inv * g.y;
            top = max_abs_bits(max_abs_bits(top, y[2 * j]), y[2 * j + 1]);
        }
        top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));  // two lanes share a block
        uint32_t byte;
        float mul;
        bool nonfinite;
        block_scale_f32(__uint_as_float(top), p.device_tiny != 0u, kE5m2 ? 15u : 8u, byte, mul, nonfinite);
        uint32_t o[4];
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j) {
            const float a = y[4 * j] * mul, b = y[4 * j + 1] * mul, c = y[4 * j + 2] * mul, d = y[4 * j + 3] * mul;
            o[j] = kE5m2 ? cvt_e5m2x2(a, b) | (cvt_e5m2x2(c, d) << 16) : cvt_e4m3x2(a, b) | (cvt_e4m3x2(c, d) << 16);
            if (nonfinite) {
                o[j] = 0x7F7F7F7Fu;
            }
        }
        if (inside) {
            const size_t at = (size_t)row * p.n + col;
            *reinterpret_cast<uint4*>(p.codes + at) = make_uint4(o[0], o[1], o[2], o[3]);
            if ((lane & 1u) == 0u) {
                p.scales[at / 32u] = (uint8_t)byte;  // n is a multiple of 32: blocks follow one another over the rows too
            }
            if (p.norm_out != nullptr) {
                uint32_t v[8];
#pragma unroll
                for (uint32_t j = 0; j < 8; ++j) {
                    const __nv_bfloat162 s = __floats2bfloat162_rn(y[2 * j], y[2 * j + 1]);
                    v[j] = *reinterpret_cast<const uint32_t*>(&s);
                }
                store_half_block(p.norm_out + at * 2u, v);
            }
        }
    }
}

}  // namespace catccos
