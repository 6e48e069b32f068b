// Quantiser to 8-bit codes with one fp32 scale for each block of 128 values, the operands of block_gemm.cuh.  For a block
//   top = max(largest |x|, 2^-100);   scale = top / F;   code = RNE with saturation of x * (F / top)     (F = 448 E4M3, 57344 E5M2)
// A block is 128 values of a row (1 x 128: activations, whose products run along the row), of a column (128 x 1: operands of a
// weight's gradient, whose products run along the rows) or 128 x 128 (weights).  Blocks at the edges have what is there.  2^-100
// keeps both quotients finite and normal; a block of zeros has codes of zero.  An infinity or a NaN makes its block's scale and
// codes NaN.
//
// Bound by memory: 2 bytes read and 1 + 4 / 128 written an element (with row_index: the written part for every route).  Measured:
// 4096 x 7168 to 8 routes each 51.7 us (5.8 TB/s, 90 % of a plain copy), 8190 x 2304 by column 13.7 (4.2 TB/s: 1152 CTAs that each load,
// meet once and store).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"
#include "mx_quant.cuh"

namespace catccos {

constexpr uint32_t kBlockSize = 128;
constexpr uint32_t kBlockQuantThreads = 256;
constexpr float kBlockLeast = 0x1p-100f;

struct BlockQuantParams {
    const uint8_t* x;
    size_t x_row_bytes;
    const int32_t* row_index;  // [rows, top_k] or nullptr
    uint8_t* codes;            // [rows or out_rows, k]
    float* scales;
    uint32_t rows, k, blocks;  // blocks of a row
    uint32_t top_k, out_rows;
    uint64_t units;            // row form: blocks of the matrix
};

// kChunks consecutive 16-byte pieces; p is 16-byte aligned
template <uint32_t kChunks>
__device__ __forceinline__ void load_pieces(const uint8_t* p, uint4 (&w)[kChunks])
{
    if (kChunks >= 2 && ((uintptr_t)p & 31u) == 0u) {
#pragma unroll
        for (uint32_t i = 0; i + 1 < kChunks; i += 2) {
            ld_global_stream_v8(p + 16u * i, w[i], w[i + 1]);
        }
    } else {
#pragma unroll
        for (uint32_t i = 0; i < kChunks; ++i) {
            w[i] = __ldcs(reinterpret_cast<const uint4*>(p) + i);
        }
    }
}

// Their values as fp32
template <typename T, uint32_t kChunks>
__device__ __forceinline__ void values_of(const uint4 (&w)[kChunks], float (&v)[kChunks * 16 / sizeof(T)])
{
    constexpr uint32_t kPer = 16 / sizeof(T);
#pragma unroll
    for (uint32_t i = 0; i < kChunks; ++i) {
        const uint32_t b[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j) {
            if constexpr (sizeof(T) == 4) {
                v[i * kPer + j] = __uint_as_float(b[j]);
            } else if constexpr (std::is_same<T, __half>::value) {
                const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&b[j]));
                v[i * kPer + 2 * j] = f.x;
                v[i * kPer + 2 * j + 1] = f.y;
            } else {
                v[i * kPer + 2 * j] = __uint_as_float(b[j] << 16);
                v[i * kPer + 2 * j + 1] = __uint_as_float(b[j] & 0xFFFF0000u);
            }
        }
    }
}

// |v| as ordered bits: a NaN counts as larger than any number
__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7FFFFFFFu; }

// A block's scale and multiplier from its largest |value| (as ordered bits); a block that is not finite gets NaN for both, and a
// NaN times anything is encoded as the NaN code.
template <bool kE5m2>
__device__ __forceinline__ void block_scale_128(uint32_t top_bits, float& scale, float& mul)
{
    constexpr float kMost = kE5m2 ? 57344.0f : 448.0f;
    const float top = fmaxf(__uint_as_float(top_bits), kBlockLeast);
    scale = top / kMost;
    mul = kMost / top;
    if (top_bits >= 0x7F800000u) {
        scale = mul = __uint_as_float(0x7FC00000u);
    }
}

template <bool kE5m2>
__device__ __forceinline__ uint32_t encode_4(float a, float b, float c, float d)
{
    return kE5m2 ? cvt_e5m2x2(a, b) | (cvt_e5m2x2(c, d) << 16) : cvt_e4m3x2(a, b) | (cvt_e4m3x2(c, d) << 16);
}

// Blocks of 1 x 128: eight lanes of 16 values each to a block, the blocks of the matrix one after the other; every lane does one
// load and ends.
template <typename T, bool kE5m2>
__global__ void __launch_bounds__(kBlockQuantThreads) block_quant_rows_kernel(const BlockQuantParams p)
{
    grid_dep_wait();
    grid_dep_launch();
    const uint64_t unit = (uint64_t)blockIdx.x * (kBlockQuantThreads / 8) + (threadIdx.x >> 3);
    const uint32_t row = (uint32_t)(unit / p.blocks), block = (uint32_t)(unit - (uint64_t)row * p.blocks);
    const uint32_t col = block * kBlockSize + (threadIdx.x & 7u) * 16u;
    const bool live = unit < p.units, inside = live && col < p.k;
    float v[16] = {};
    if (inside) {
        uint4 w[sizeof(T)];
        load_pieces(p.x + (size_t)row * p.x_row_bytes + (size_t)col * sizeof(T), w);
        values_of<T>(w, v);
    }
    uint32_t top = 0;
#pragma unroll
    for (uint32_t i = 0; i < 16; ++i) {
        top = max(top, abs_bits(v[i]));
    }
    top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
    top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
    top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 4));
    float scale, mul;
    block_scale_128<kE5m2>(top, scale, mul);
    uint4 o;
    o.x = encode_4<kE5m2>(v[0] * mul, v[1] * mul, v[2] * mul, v[3] * mul);
    o.y = encode_4<kE5m2>(v[4] * mul, v[5] * mul, v[6] * mul, v[7] * mul);
    o.z = encode_4<kE5m2>(v[8] * mul, v[9] * mul, v[10] * mul, v[11] * mul);
    o.w = encode_4<kE5m2>(v[12] * mul, v[13] * mul, v[14] * mul, v[15] * mul);
    auto store = [&](size_t to) {
        if (inside) {
            *reinterpret_cast<uint4*>(p.codes + to * p.k + col) = o;
            if ((threadIdx.x & 7u) == 0u) {
                p.scales[to * p.blocks + block] = scale;
            }
        }
    };
    if (p.row_index == nullptr) {
        store(row);
    } else if (live) {
        for (uint32_t r = 0; r < p.top_k; ++r) {
            const uint32_t to = (uint32_t)__ldcg(p.row_index + (size_t)row * p.top_k + r);
            if (to < p.out_rows) {  // a dropped route is negative: above any row
                store(to);
            }
        }
    }
}

// Blocks of 128 x 1 and of 128 x 128: a CTA has 128 rows of 128 columns in registers, as they are stored (as fp32 the 16-bit types
// would leave room for half as many CTAs: 8190 x 2304 by column 20.0 us), a thread 8 columns of every 16th row. Four CTAs an SM of the
// 16-bit types against three: bf16 8190 x 2304 by column 14.0 -> 13.2 us, 8192 x 7168 37.5 -> 36.1, but 512 x 2304 3.7 -> 3.9.
template <typename T, bool kE5m2, bool kSquare>
__global__ void __launch_bounds__(kBlockQuantThreads, sizeof(T) == 2 ? 4 : 2) block_quant_tiles_kernel(const BlockQuantParams p)
{
    __shared__ __align__(16) uint32_t tops[kBlockQuantThreads / 32][kBlockSize];
    grid_dep_wait();
    grid_dep_launch();
    const uint32_t tx = threadIdx.x & 15u, ty = threadIdx.x >> 4, warp = threadIdx.x >> 5;
    const uint32_t row0 = (uint32_t)(blockIdx.x / p.blocks) * kBlockSize, block = blockIdx.x % p.blocks;
    const uint32_t col = block * kBlockSize + tx * 8u;
    uint4 w[8][sizeof(T) / 2];
#pragma unroll
    for (uint32_t i = 0; i < 8; ++i) {
        const uint32_t row = row0 + ty + 16u * i;
        if (row < p.rows && col < p.k) {
            load_pieces(p.x + (size_t)row * p.x_row_bytes + (size_t)col * sizeof(T), w[i]);
        } else {
#pragma unroll
            for (uint32_t c = 0; c < sizeof(T) / 2; ++c) {
                w[i][c] = make_uint4(0, 0, 0, 0);
            }
        }
    }
    uint32_t top[8] = {};
#pragma unroll
    for (uint32_t i = 0; i < 8; ++i) {
        float v[8];
        values_of<T>(w[i], v);
#pragma unroll
        for (uint32_t j = 0; j < 8; ++j) {
            top[j] = max(top[j], abs_bits(v[j]));
        }
    }
    // the values are made from the stored ones again below: kept as fp32 they would not fit (fp16 by column 13.4 -> 18.8 us)
    if (sizeof(T) == 2) {
#pragma unroll
        for (uint32_t i = 0; i < 8; ++i) {
            asm volatile("" : "+r"(w[i][0].x), "+r"(w[i][0].y), "+r"(w[i][0].z), "+r"(w[i][0].w));
        }
    }
    if (kSquare) {
        uint32_t all = 0;
#pragma unroll
        for (uint32_t j = 0; j < 8; ++j) {
            all = max(all, top[j]);
        }
        all = __reduce_max_sync(0xFFFFFFFFu, all);
        if ((threadIdx.x & 31u) == 0u) {
            tops[warp][0] = all;
        }
        __syncthreads();
#pragma unroll
        for (uint32_t i = 0; i < kBlockQuantThreads / 32; ++i) {
            all = max(all, tops[i][0]);
        }
        top[0] = all;
    } else {
#pragma unroll
        for (uint32_t j = 0; j < 8; ++j) {
            top[j] = max(top[j], __shfl_xor_sync(0xFFFFFFFFu, top[j], 16));
        }
        if ((threadIdx.x & 16u) == 0u) {
#pragma unroll
            for (uint32_t h = 0; h < 2; ++h) {
                *reinterpret_cast<uint4*>(&tops[warp][tx * 8u + 4u * h]) = make_uint4(top[4 * h], top[4 * h + 1], top[4 * h + 2], top[4 * h + 3]);
            }
        }
        __syncthreads();
#pragma unroll
        for (uint32_t i = 0; i < kBlockQuantThreads / 32; ++i) {
#pragma unroll
            for (uint32_t h = 0; h < 2; ++h) {
                const uint4 o = *reinterpret_cast<const uint4*>(&tops[i][tx * 8u + 4u * h]);
                top[4 * h] = max(top[4 * h], o.x);
                top[4 * h + 1] = max(top[4 * h + 1], o.y);
                top[4 * h + 2] = max(top[4 * h + 2], o.z);
                top[4 * h + 3] = max(top[4 * h + 3], o.w);
            }
        }
    }
    float scale[8], mul[8];
#pragma unroll
    for (uint32_t j = 0; j < (kSquare ? 1u : 8u); ++j) {
        block_scale_128<kE5m2>(top[j], scale[j], mul[j]);
    }
    if (kSquare) {
        if (threadIdx.x == 0) {
            p.scales[blockIdx.x] = scale[0];
        }
    } else if (ty == 0 && col < p.k) {
#pragma unroll
        for (uint32_t j = 0; j < 8; ++j) {
            p.scales[(size_t)(row0 / kBlockSize) * p.k + col + j] = scale[j];
        }
    }
#pragma unroll
    for (uint32_t i = 0; i < 8; ++i) {
        const uint32_t row = row0 + ty + 16u * i;
        if (row < p.rows && col < p.k) {
            float v[8];
            values_of<T>(w[i], v);
            uint32_t o[2];
#pragma unroll
            for (uint32_t h = 0; h < 2; ++h) {
                o[h] = encode_4<kE5m2>(v[4 * h] * mul[kSquare ? 0 : 4 * h], v[4 * h + 1] * mul[kSquare ? 0 : 4 * h + 1],
                                       v[4 * h + 2] * mul[kSquare ? 0 : 4 * h + 2], v[4 * h + 3] * mul[kSquare ? 0 : 4 * h + 3]);
            }
            *reinterpret_cast<uint2*>(p.codes + (size_t)row * p.k + col) = make_uint2(o[0], o[1]);
        }
    }
}

}  // namespace catccos
