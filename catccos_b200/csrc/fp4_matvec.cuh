// Products of one or a few tokens with packed E2M1 weights, read where they lie: y[m, n] = x[m, k] x dequant(w[k, n]).
//   x   bf16 [m, k];   w packed E2M1 [k, n/2], low nibble = even column;   scales E8M0 [k/64, n, 2]
// With ids the weight is one of several: row r of the result is x[r / (routes / x_rows)] x dequant(w[ids[r]]).
//
// Bound by the weights' bytes (half a byte and 1/32 per element), then by the instructions that unpack them: an SM takes in 46
// weights a cycle at full memory rate.  So two weights are unpacked by one conversion (cvt.f16x2.e2m1x2, 64 lanes a cycle as
// any integer instruction) and the products run on mma.sync m16n8k16 (f16 in, fp32 sums), where they cost nothing here.
// That instruction wants two consecutive k in a register; a byte holds two columns of one k.  Instead of transposing, the
// two k slots of a register are given to the two columns, and the token's value takes the first slot in one column of the
// other operand and the second slot in the next, with a zero beside it: eight columns of it are four tokens.
//
// x goes in as f16 after a power of two per token and 64 k that brings its largest magnitude to 2^14 .. 2^15: every bf16
// within 2^-29 of the largest stays exact, smaller ones are off by at most 2^-40 of it, far below the fp32 sums' rounding.
// Sums of 32 products share a weight scale, which is applied to them in fp32.
#pragma once

#include <cuda_fp16.h>

#include "common.cuh"
#include "mx_gemm.cuh"
#include "mx_quant.cuh"

namespace catccos {

constexpr uint32_t kMatvecWarps = 8, kMatvecThreads = kMatvecWarps * 32;
constexpr uint32_t kMatvecCols = 128;  // of a CTA: 8 lane groups x 16
constexpr uint32_t kMatvecUnit = 64;   // k of a warp's step: the two scale groups that lie together
constexpr uint32_t kMatvecMaxCluster = 8;

struct MatvecParams {
    const uint8_t* x;       // bf16
    const uint8_t* w;       // packed E2M1
    const uint8_t* scales;  // E8M0
    const int32_t* ids;     // one weight per row of the result, or nullptr
    uint8_t* out;           // 16-bit floats [rows, n]
    uint32_t rows, n, k;
    uint32_t experts;
    uint32_t rows_per_x;    // rows of the result that share a row of x (with ids)
};

__device__ __forceinline__ uint32_t e2m1x2_to_f16x2(uint32_t word, uint32_t byte)
{
    uint32_t r;
    asm("{\n\t"
        ".reg .b8 b;\n\t"
        "cvt.u8.u32 b, %1;\n\t"
        "cvt.rn.f16x2.e2m1x2 %0, b;\n\t"
        "}"
        : "=r"(r)
        : "r"(word >> (8u * byte)));
    return r;
}

// two E8M0 bytes -> two bf16 (0xFF becomes NaN)
__device__ __forceinline__ uint32_t e8m0x2_to_bf16x2(uint32_t pair)
{
    uint32_t r;
    asm("{\n\t"
        ".reg .b16 h;\n\t"
        "cvt.u16.u32 h, %1;\n\t"
        "cvt.rn.bf16x2.ue8m0x2 %0, h;\n\t"
        "}"
        : "=r"(r)
        : "r"(pair));
    return r;
}

__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1)
{
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ float ld_cluster_f32(const float* p, uint32_t cta)
{
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(map_to_cta(smem_u32(p), cta)) : "memory");
    return v;
}

// kSets sets of four tokens.  A cluster is one block of 128 columns of one set of rows; its CTAs and their warps share the
// steps of 64 k.  The partial sums meet in shared memory, warp by warp and CTA by CTA in ascending order.
template <uint32_t kSets, typename OutT>
__global__ void __launch_bounds__(kMatvecThreads, 2) fp4_matvec_kernel(const MatvecParams p)
{
    constexpr uint32_t kTokens = 4 * kSets;
    __shared__ float part[kMatvecWarps][kTokens][kMatvecCols];
    __shared__ float total[kTokens][kMatvecCols];
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
    const uint32_t g = lane >> 2, tig = lane & 3u;
    uint32_t ctas, cta;
    asm("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(ctas));
    cta = cluster_ctarank();
    const uint32_t n0 = blockIdx.x / ctas * kMatvecCols;
    const uint32_t row0 = p.ids != nullptr ? blockIdx.y : blockIdx.y * kTokens;
    grid_dep_wait();
    grid_dep_launch();

    const uint8_t* w = p.w;
    const uint8_t* scales = p.scales;
    uint32_t tokens = min(kTokens, p.rows - row0), x_row = row0;
    bool live = true;
    if (p.ids != nullptr) {
        const uint32_t id = (uint32_t)p.ids[row0];
        tokens = 1u;
        x_row = row0 / p.rows_per_x;
        live = id < p.experts;  // a negative id is a dropped route: its row is zero
        if (live) {
            w += (size_t)id * p.k * (p.n / 2u);
            scales += (size_t)id * (p.k / 32u) * p.n;
        }
    }
    const uint32_t col = n0 + g * 16u;
    const bool col_ok = col < p.n;
    const uint32_t steps = live ? p.k / kMatvecUnit : 0u;
    // bytes of the other operand's registers: this lane's slot takes the token's value, the other one a zero
    const uint32_t sel_lo = (g & 1u) == 0u ? 0x4410u : 0x1044u, sel_hi = (g & 1u) == 0u ? 0x4432u : 0x3244u;

    float sum[kSets][4][4] = {};
    for (uint32_t step = cta * kMatvecWarps + warp; step < steps; step += ctas * kMatvecWarps) {
        uint2 q[2][8];
        uint4 f[2];
        f[0] = f[1] = make_uint4(0, 0, 0, 0);
#pragma unroll
        for (uint32_t h = 0; h < 2; ++h) {
#pragma unroll
            for (uint32_t r = 0; r < 8; ++r) {
                q[h][r] = make_uint2(0, 0);
                if (col_ok) {
                    q[h][r] = __ldcs(reinterpret_cast<const uint2*>(
                        w + (size_t)(step * kMatvecUnit + h * 32u + tig * 8u + r) * (p.n / 2u) + col / 2u));
                }
            }
        }
        if (col_ok) {
            const uint4* s = reinterpret_cast<const uint4*>(scales + ((size_t)step * p.n + col) * 2u);
            f[0] = s[0];
            f[1] = s[1];
        }
        // the tokens' values: lane (g, tig) holds token g / 2, k tig * 8 .. + 7 of both halves
        uint32_t xh[kSets][2][4];
        float back[kSets];
#pragma unroll
        for (uint32_t t = 0; t < kSets; ++t) {
            const uint32_t token = t * 4u + (g >> 1);
            uint4 v[2];
            v[0] = v[1] = make_uint4(0, 0, 0, 0);
            if (token < tokens) {
                const uint4* src = reinterpret_cast<const uint4*>(p.x + ((size_t)(x_row + token) * p.k + step * kMatvecUnit + tig * 8u) * 2u);
                v[0] = src[0];
                v[1] = src[4];
            }
            uint32_t top = max(absmax_bits8(v[0]), absmax_bits8(v[1]));
            if (__any_sync(0xFFFFFFFFu, top >= 0x7F80u)) {
                // an infinity or NaN does not set the scale: the finite values beside it must not become infinite
                top = 0;
                const uint32_t all[8] = {v[0].x, v[0].y, v[0].z, v[0].w, v[1].x, v[1].y, v[1].z, v[1].w};
#pragma unroll
                for (uint32_t i = 0; i < 8; ++i) {
                    const uint32_t lo = all[i] & 0x7FFFu, hi = (all[i] >> 16) & 0x7FFFu;
                    top = max(top, max(lo < 0x7F80u ? lo : 0u, hi < 0x7F80u ? hi : 0u));
                }
            }
            top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
            top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
            const int up = min(141 - (int)(top >> 7), 126);
            const float mul = __uint_as_float((uint32_t)(127 + up) << 23);
            // this lane's sums belong to token tig of the set
            back[t] = __uint_as_float((uint32_t)(127 - __shfl_sync(0xFFFFFFFFu, up, tig * 8u)) << 23);
#pragma unroll
            for (uint32_t h = 0; h < 2; ++h) {
                const uint32_t a[4] = {v[h].x, v[h].y, v[h].z, v[h].w};
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i) {
                    xh[t][h][i] = pack2<__half>(__uint_as_float(a[i] << 16) * mul, __uint_as_float(a[i] & 0xFFFF0000u) * mul);
                }
            }
        }
        const uint32_t fw[8] = {f[0].x, f[0].y, f[0].z, f[0].w, f[1].x, f[1].y, f[1].z, f[1].w};
#pragma unroll
        for (uint32_t h = 0; h < 2; ++h) {
            float d[kSets][4][4] = {};
#pragma unroll
            for (uint32_t s = 0; s < 4; ++s) {
                uint32_t b0[kSets], b1[kSets];
#pragma unroll
                for (uint32_t t = 0; t < kSets; ++t) {
                    b0[t] = __byte_perm(xh[t][h][s], 0u, sel_lo);
                    b1[t] = __byte_perm(xh[t][h][s], 0u, sel_hi);
                }
#pragma unroll
                for (uint32_t j = 0; j < 4; ++j) {
                    const uint32_t a0 = e2m1x2_to_f16x2(q[h][2 * s].x, j), a1 = e2m1x2_to_f16x2(q[h][2 * s].y, j);
                    const uint32_t a2 = e2m1x2_to_f16x2(q[h][2 * s + 1].x, j), a3 = e2m1x2_to_f16x2(q[h][2 * s + 1].y, j);
#pragma unroll
                    for (uint32_t t = 0; t < kSets; ++t) {
                        mma_f16(d[t][j], a0, a1, a2, a3, b0[t], b1[t]);
                    }
                }
            }
            // d[.][j][0..3]: columns 2j, 2j + 1, 8 + 2j, 9 + 2j of this lane's sixteen, token tig of the set
#pragma unroll
            for (uint32_t j = 0; j < 4; ++j) {
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i) {
                    const uint32_t pair = fw[(i >> 1) * 4u + j] >> (16u * (i & 1u));
                    const uint32_t both = e8m0x2_to_bf16x2(pair);
                    const float scale = __uint_as_float(h == 0u ? both << 16 : both & 0xFFFF0000u);
#pragma unroll
                    for (uint32_t t = 0; t < kSets; ++t) {
                        sum[t][j][i] = fmaf(d[t][j][i] * back[t], scale, sum[t][j][i]);
                    }
                }
            }
        }
    }
#pragma unroll
    for (uint32_t t = 0; t < kSets; ++t) {
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j) {
            float* dst = &part[warp][t * 4u + tig][g * 16u];
            *reinterpret_cast<float2*>(dst + 2u * j) = make_float2(sum[t][j][0], sum[t][j][1]);
            *reinterpret_cast<float2*>(dst + 8u + 2u * j) = make_float2(sum[t][j][2], sum[t][j][3]);
        }
    }
    __syncthreads();
    const uint32_t values = tokens * kMatvecCols;
    for (uint32_t i = threadIdx.x; i < values; i += kMatvecThreads) {
        float v = 0.0f;
#pragma unroll
        for (uint32_t o = 0; o < kMatvecWarps; ++o) {
            v += (&part[o][0][0])[i];
        }
        (&total[0][0])[i] = v;
    }
    __syncthreads();
    if (ctas > 1u) {
        cluster_sync_all();
    }
    // every CTA of the cluster writes its share of the pairs of columns
    for (uint32_t i = cta * kMatvecThreads + threadIdx.x; i < values / 2u; i += ctas * kMatvecThreads) {
        const float* src = &total[0][0] + 2u * i;
        float a = 0.0f, b = 0.0f;
        for (uint32_t o = 0; o < ctas; ++o) {
            a += ctas > 1u ? ld_cluster_f32(src, o) : src[0];
            b += ctas > 1u ? ld_cluster_f32(src + 1, o) : src[1];
        }
        const uint32_t token = 2u * i / kMatvecCols, c = n0 + (2u * i & (kMatvecCols - 1u));
        if (c < p.n) {
            *reinterpret_cast<uint32_t*>(p.out + ((size_t)(row0 + token) * p.n + c) * 2u) = pack2<OutT>(a, b);
        }
    }
    if (ctas > 1u) {
        __syncwarp();
        cluster_sync_all();  // no CTA leaves while another may still read its sums
    }
}

}  // namespace catccos
