// Products of one or a few tokens with packed E2M1 weights, read where they lie: y[m, n] = x[m, k] x dequant(w[k, n]).
//   x   bf16 [m, k];   w packed E2M1 [k, n/2], low nibble = even column;   scales E8M0 [k/64, n, 2]
// With ids the weight is one of several: row r of the result is x[r / (routes / x_rows)] x dequant(w[ids[r]]).
//
// Rows of the result that share a weight are multiplied together, four to a pass over it.
//
// Bound by the weights' bytes (half a byte and 1/32 per element), then by the instructions that unpack them: an SM takes in 46
// weights a cycle at full memory rate.  So two weights are unpacked by one conversion (cvt.f16x2.e2m1x2, 64 lanes a cycle as
// any integer instruction) and the products run on mma.sync m16n8k16 (f16 in, fp32 sums), where they cost nothing here.
// That instruction wants two consecutive k in a register; a byte holds two columns of one k.  Instead of transposing, the
// two k slots of a register are given to the two columns, and the token's value takes the first slot in one column of the
// other operand and the second slot in the next, with a zero beside it: eight columns of it are four tokens.
//
// x goes in as f16 after a power of two per token and 64 k that brings its largest magnitude to 2^14 .. 2^15: every bf16
// within 2^-29 of the largest stays exact, smaller ones are off by at most 2^-39 of it (half a step of f16's denormals, 2^-25, of
// 2^14), far below the fp32 sums' rounding.
// Sums of 32 products share a weight scale, which is applied to them in fp32, after the power of two is undone: what lies between
// may be larger than what comes out.  A sum of 32 is below 2^22.6 (values to 2^15, weights to 6), and for the largest bf16 2^113 is
// to be undone, so all sums are held at 2^-8 of their size up to the end and no step of a result that bf16 holds leaves fp32's
// range.  The additions of results near fp32's lowest normal number are off by up to 2^-142 for that, a 512th of bf16's lowest.
// (Deciding step by step costs 1 to 5 % with a branch, 7 % with a multiplication more.)
//
// Every warp has a ring of its own in shared memory, filled by asynchronous copies, two steps (10 KB) ahead; 150 KB an SM.  One
// token and a weight of 330 MB run at 5.5 TB/s; small ones are some 5 us of launch, first and last step around that (one token,
// 4096 x 7168: 7.1 us).  Half steps in rings of three, three CTAs an SM, took 10.0 us there, and the largest magnitude of x found
// ahead of the loop 9.5.
#pragma once

#include <cuda_fp16.h>

#include "common.cuh"
#include "mx_gemm.cuh"
#include "mx_quant.cuh"

namespace catccos {

constexpr uint32_t kMatvecWarps = 8, kMatvecThreads = kMatvecWarps * 32;
constexpr uint32_t kMatvecCols = 128;  // of a CTA: 8 lane groups x 16
constexpr uint32_t kMatvecUnit = 64;   // k of a warp's step: the two scale groups that lie together
constexpr uint32_t kMatvecDepth = 2;   // steps of a warp's ring
constexpr uint32_t kMatvecMaxCluster = 8;
constexpr int kMatvecHeadroom = 8;     // sums are held at 2^-8 of their size
constexpr uint32_t kMatvecPartRow = kMatvecCols + 8;
constexpr uint32_t kMatvecWindow = 1024;  // routes among which a weight's rows find one another

// One step in a warp's ring: 64 rows of 64 bytes of the weight, 128 columns' scales, four tokens' (times kSets) values
constexpr uint32_t kMatvecScalesOff = kMatvecUnit * kMatvecCols / 2;
constexpr uint32_t kMatvecXOff = kMatvecScalesOff + kMatvecCols * 2;
template <uint32_t kSets>
constexpr uint32_t kMatvecStage = kMatvecXOff + kSets * 4 * kMatvecUnit * 2;
template <uint32_t kSets>
constexpr uint32_t kMatvecSmem = kMatvecWarps * kMatvecDepth * kMatvecStage<kSets>;

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

// The two E2M1 values of byte `byte` of a word as f16, the low nibble's in the low half.  The byte is named by the instruction
// itself: shifting it down first made three of four conversions two instructions.
template <uint32_t kByte>
__device__ __forceinline__ uint32_t e2m1x2_to_f16x2(uint32_t word)
{
    uint32_t r;
    if constexpr (kByte == 0) {
        asm("{.reg .b8 b0, b1, b2, b3; mov.b32 {b0, b1, b2, b3}, %1; cvt.rn.f16x2.e2m1x2 %0, b0;}" : "=r"(r) : "r"(word));
    } else if constexpr (kByte == 1) {
        asm("{.reg .b8 b0, b1, b2, b3; mov.b32 {b0, b1, b2, b3}, %1; cvt.rn.f16x2.e2m1x2 %0, b1;}" : "=r"(r) : "r"(word));
    } else if constexpr (kByte == 2) {
        asm("{.reg .b8 b0, b1, b2, b3; mov.b32 {b0, b1, b2, b3}, %1; cvt.rn.f16x2.e2m1x2 %0, b2;}" : "=r"(r) : "r"(word));
    } else {
        asm("{.reg .b8 b0, b1, b2, b3; mov.b32 {b0, b1, b2, b3}, %1; cvt.rn.f16x2.e2m1x2 %0, b3;}" : "=r"(r) : "r"(word));
    }
    return r;
}

// A word of E8M0 bytes as four bf16, two to a register (0xFF becomes NaN)
__device__ __forceinline__ void e8m0x4_to_bf16(uint32_t word, uint32_t& lo, uint32_t& hi)
{
    asm("{.reg .b16 h0, h1; mov.b32 {h0, h1}, %2; cvt.rn.bf16x2.ue8m0x2 %0, h0; cvt.rn.bf16x2.ue8m0x2 %1, h1;}"
        : "=r"(lo), "=r"(hi)
        : "r"(word));
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

// 8-byte copy global -> shared; zeros when !inside (then nothing is read).
__device__ __forceinline__ void cp_async_8(uint32_t smem_dst, const void* gsrc, bool inside)
{
    asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(smem_dst), "l"(gsrc), "r"(inside ? 8u : 0u) : "memory");
}

__device__ __forceinline__ uint4 ld_shared_u4(uint32_t addr)
{
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
    return v;
}

__device__ __forceinline__ uint2 ld_shared_u2(uint32_t addr)
{
    uint2 v;
    asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr));
    return v;
}

// Half a step lies in slots of 64 bytes: slot s has row 8 (s & 3) + s / 4 (a load of the products takes rows r, 8 + r, 16 + r and
// 24 + r of the eight lane groups), the last two of four slots their 16-byte chunks the other way round.  So no two lanes of a
// half warp meet in a bank, and a copy, which fills slots that follow one another, none either.
__device__ __forceinline__ uint32_t matvec_row(uint32_t slot) { return ((slot & 3u) << 3) | (slot >> 2); }
__device__ __forceinline__ uint32_t matvec_chunk(uint32_t slot, uint32_t chunk) { return chunk ^ (slot & 2u); }

// kSets sets of four tokens.  A cluster is one block of 128 columns of one set of rows; its CTAs and their warps share the
// steps of 64 k.  The partial sums meet in shared memory, warp by warp and CTA by CTA in ascending order.
// kWhole: rows of the weight are multiples of 16 bytes.
template <uint32_t kSets, bool kWhole, typename OutT>
__global__ void __launch_bounds__(kMatvecThreads, 2) fp4_matvec_kernel(const MatvecParams p)
{
    constexpr uint32_t kTokens = 4 * kSets;
    constexpr uint32_t kAll = 0xFFFFFFFFu;
    extern __shared__ __align__(16) uint8_t matvec_smem[];
    __shared__ float total[kTokens][kMatvecCols];
    __shared__ uint32_t same[kMatvecWindow / 32];
    static_assert(kMatvecSmem<kSets> >= kMatvecWarps * kTokens * kMatvecPartRow * 4, "the partial sums take the rings' place");
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
    const uint32_t g = lane >> 2, tig = lane & 3u;
    uint32_t ctas;
    asm("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(ctas));
    const uint32_t cta = cluster_ctarank();
    const uint32_t n0 = blockIdx.x / ctas * kMatvecCols;
    grid_dep_wait();
    grid_dep_launch();

    const uint8_t* w = p.w;
    const uint8_t* scales = p.scales;
    uint32_t rows[kTokens];  // of the result
    uint32_t tokens;
    bool live = true;
    if (p.ids == nullptr) {
        tokens = min(kTokens, p.rows - blockIdx.y * kTokens);
#pragma unroll
        for (uint32_t t = 0; t < kTokens; ++t) {
            rows[t] = blockIdx.y * kTokens + t;
        }
    } else {
        // this row and the next three of the same weight; a row that one in front of it takes along has nothing to do
        const uint32_t row = blockIdx.y, base = row / kMatvecWindow * kMatvecWindow;
        const uint32_t id = (uint32_t)p.ids[row];
        live = id < p.experts;  // a negative id is a dropped route: its row is zero
#pragma unroll
        for (uint32_t i = 0; i < kMatvecWindow / kMatvecThreads; ++i) {
            const uint32_t at = base + i * kMatvecThreads + threadIdx.x;
            const uint32_t mask = __ballot_sync(kAll, at < p.rows && (uint32_t)p.ids[min(at, p.rows - 1u)] == id);
            if (lane == 0) {
                same[i * kMatvecWarps + warp] = mask;
            }
        }
        __syncthreads();
        uint32_t before = 0;
        const uint32_t word = (row - base) >> 5, bit = (row - base) & 31u;
        for (uint32_t i = 0; i < word; ++i) {
            before += (uint32_t)__popc(same[i]);
        }
        before += (uint32_t)__popc(same[word] & ((1u << bit) - 1u));
        if (live && before % kTokens != 0u) {
            return;  // the same answer for the whole cluster
        }
        tokens = 1;
        rows[0] = row;
        uint32_t i = word, left = same[word] & ~((2u << bit) - 1u);
#pragma unroll
        for (uint32_t t = 1; t < kTokens; ++t) {
            rows[t] = row;
            while (live && left == 0u && i + 1u < kMatvecWindow / 32u) {
                left = same[++i];
            }
            if (live && left != 0u) {
                rows[t] = base + i * 32u + (uint32_t)__ffs((int)left) - 1u;
                left &= left - 1u;
                tokens = t + 1u;
            }
        }
        if (live) {
            w += (size_t)id * p.k * (p.n / 2u);
            scales += (size_t)id * (p.k / 32u) * p.n;
        }
    }
    const uint32_t steps = live ? p.k / kMatvecUnit : 0u;
    // bytes of the other operand's registers: this lane's slot takes the token's value, the other one a zero
    const uint32_t sel_lo = (g & 1u) == 0u ? 0x4410u : 0x1044u, sel_hi = (g & 1u) == 0u ? 0x4432u : 0x3244u;
    const uint32_t ring = smem_u32(matvec_smem) + warp * (kMatvecDepth * kMatvecStage<kSets>);

    // where this lane copies from: token lane / 8 of each set
    const uint8_t* x_src[kSets];
    bool x_in[kSets];
#pragma unroll
    for (uint32_t t = 0; t < kSets; ++t) {
        uint32_t row = rows[t * 4u];
#pragma unroll
        for (uint32_t j = 1; j < 4; ++j) {
            row = (lane >> 3) == j ? rows[t * 4u + j] : row;
        }
        x_in[t] = t * 4u + (lane >> 3) < tokens;
        x_src[t] = p.x + ((size_t)(x_in[t] ? row / p.rows_per_x : 0u) * p.k + (lane & 7u) * 8u) * 2u;
    }
    auto copy = [&](uint32_t step, uint32_t stage) {
        const size_t pitch = p.n / 2u;
        const uint8_t* src = w + (size_t)step * kMatvecUnit * pitch;
        if constexpr (kWhole) {
            const uint32_t chunk = lane & 3u;
            const bool inside = n0 + chunk * 32u < p.n;
            const uint8_t* from = src + (inside ? n0 / 2u + chunk * 16u : 0u);
#pragma unroll
            for (uint32_t i = 0; i < 8; ++i) {
                const uint32_t half = i >> 2, slot = (i & 3u) * 8u + (lane >> 2);
                cp_async_16(stage + half * 2048u + slot * 64u + matvec_chunk(slot, chunk) * 16u,
                            from + (half * 32u + matvec_row(slot)) * pitch, inside);
            }
        } else {
            const uint32_t part = lane & 7u;
            const bool inside = n0 + part * 16u < p.n;
            const uint8_t* from = src + (inside ? n0 / 2u + part * 8u : 0u);
#pragma unroll
            for (uint32_t i = 0; i < 16; ++i) {
                const uint32_t half = i >> 3, slot = (i & 7u) * 4u + (lane >> 3);
                cp_async_8(stage + half * 2048u + slot * 64u + matvec_chunk(slot, part >> 1) * 16u + (part & 1u) * 8u,
                           from + (half * 32u + matvec_row(slot)) * pitch, inside);
            }
        }
        if (lane < 16u) {
            const bool inside = n0 + lane * 8u < p.n;
            cp_async_16(stage + kMatvecScalesOff + lane * 16u, scales + ((size_t)step * p.n + (inside ? n0 + lane * 8u : 0u)) * 2u, inside);
        }
#pragma unroll
        for (uint32_t t = 0; t < kSets; ++t) {
            cp_async_16(stage + kMatvecXOff + t * 512u + lane * 16u, x_src[t] + (size_t)step * (kMatvecUnit * 2u), x_in[t]);
        }
    };

    float sum[kSets][4][4] = {};
    const uint32_t first = cta * kMatvecWarps + warp, stride = ctas * kMatvecWarps;
#pragma unroll
    for (uint32_t d = 0; d < kMatvecDepth; ++d) {
        if (first + d * stride < steps) {
            copy(first + d * stride, ring + d * kMatvecStage<kSets>);
        }
        cp_async_commit();
    }
    uint32_t stage = ring;
    for (uint32_t step = first; step < steps; step += stride) {
        cp_async_wait<kMatvecDepth - 1>();
        __syncwarp();
        // the tokens' values: lane (g, tig) holds token g / 2, k tig * 8 .. + 7 of both halves
        uint32_t xh[kSets][2][4];
        float back[kSets];
#pragma unroll
        for (uint32_t t = 0; t < kSets; ++t) {
            const uint32_t at = stage + kMatvecXOff + t * 512u + (g >> 1) * 128u + tig * 16u;
            const uint4 v[2] = {ld_shared_u4(at), ld_shared_u4(at + 64u)};
            uint32_t top = max(absmax_bits8(v[0]), absmax_bits8(v[1]));
            if (__any_sync(kAll, top >= 0x7F80u)) {
                // an infinity or NaN does not set the scale: the finite values beside it must not become infinite
                top = 0;
                const uint32_t all[8] = {v[0].x, v[0].y, v[0].z, v[0].w, v[1].x, v[1].y, v[1].z, v[1].w};
#pragma unroll
                for (uint32_t i = 0; i < 8; ++i) {
                    const uint32_t lo = all[i] & 0x7FFFu, hi = (all[i] >> 16) & 0x7FFFu;
                    top = max(top, max(lo < 0x7F80u ? lo : 0u, hi < 0x7F80u ? hi : 0u));
                }
            }
            top = max(top, __shfl_xor_sync(kAll, top, 1));
            top = max(top, __shfl_xor_sync(kAll, top, 2));
            const int up = min(141 - (int)(top >> 7), 118);
            const float mul = __uint_as_float((uint32_t)(127 + up) << 23);
            // this lane's sums belong to token tig of the set
            back[t] = __uint_as_float((uint32_t)(127 - kMatvecHeadroom - __shfl_sync(kAll, up, tig * 8u)) << 23);
#pragma unroll
            for (uint32_t h = 0; h < 2; ++h) {
                const uint32_t a[4] = {v[h].x, v[h].y, v[h].z, v[h].w};
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i) {
                    xh[t][h][i] = pack2<__half>(__uint_as_float(a[i] << 16) * mul, __uint_as_float(a[i] & 0xFFFF0000u) * mul);
                }
            }
        }
        const uint4 f0 = ld_shared_u4(stage + kMatvecScalesOff + g * 32u), f1 = ld_shared_u4(stage + kMatvecScalesOff + g * 32u + 16u);
        const uint32_t fw[8] = {f0.x, f0.y, f0.z, f0.w, f1.x, f1.y, f1.z, f1.w};
        uint32_t scale[4][4];  // of columns 2j, 2j + 1, 8 + 2j, 9 + 2j, the first half's below, the second half's above
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j) {
            e8m0x4_to_bf16(fw[j], scale[j][0], scale[j][1]);
            e8m0x4_to_bf16(fw[4 + j], scale[j][2], scale[j][3]);
        }
#pragma unroll
        for (uint32_t h = 0; h < 2; ++h) {
            float d[kSets][4][4] = {};
#pragma unroll
            for (uint32_t s = 0; s < 4; ++s) {
                const uint32_t at = stage + h * 2048u + tig * 64u + matvec_chunk(tig, g >> 1) * 16u + (g & 1u) * 8u;
                const uint2 q0 = ld_shared_u2(at + 2u * s * 256u), q1 = ld_shared_u2(at + (2u * s + 1u) * 256u);
                uint32_t b0[kSets], b1[kSets];
#pragma unroll
                for (uint32_t t = 0; t < kSets; ++t) {
                    b0[t] = __byte_perm(xh[t][h][s], 0u, sel_lo);
                    b1[t] = __byte_perm(xh[t][h][s], 0u, sel_hi);
                }
#pragma unroll
                for (uint32_t t = 0; t < kSets; ++t) {
                    mma_f16(d[t][0], e2m1x2_to_f16x2<0>(q0.x), e2m1x2_to_f16x2<0>(q0.y), e2m1x2_to_f16x2<0>(q1.x),
                            e2m1x2_to_f16x2<0>(q1.y), b0[t], b1[t]);
                    mma_f16(d[t][1], e2m1x2_to_f16x2<1>(q0.x), e2m1x2_to_f16x2<1>(q0.y), e2m1x2_to_f16x2<1>(q1.x),
                            e2m1x2_to_f16x2<1>(q1.y), b0[t], b1[t]);
                    mma_f16(d[t][2], e2m1x2_to_f16x2<2>(q0.x), e2m1x2_to_f16x2<2>(q0.y), e2m1x2_to_f16x2<2>(q1.x),
                            e2m1x2_to_f16x2<2>(q1.y), b0[t], b1[t]);
                    mma_f16(d[t][3], e2m1x2_to_f16x2<3>(q0.x), e2m1x2_to_f16x2<3>(q0.y), e2m1x2_to_f16x2<3>(q1.x),
                            e2m1x2_to_f16x2<3>(q1.y), b0[t], b1[t]);
                }
            }
            // d[.][j][0..3]: columns 2j, 2j + 1, 8 + 2j, 9 + 2j of this lane's sixteen, token tig of the set
#pragma unroll
            for (uint32_t j = 0; j < 4; ++j) {
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i) {
                    const float f = __uint_as_float(h == 0u ? scale[j][i] << 16 : scale[j][i] & 0xFFFF0000u);
#pragma unroll
                    for (uint32_t t = 0; t < kSets; ++t) {
                        sum[t][j][i] = fmaf(d[t][j][i] * back[t], f, sum[t][j][i]);
                    }
                }
            }
        }
        __syncwarp();  // everybody has read the stage
        if (step + kMatvecDepth * stride < steps) {
            copy(step + kMatvecDepth * stride, stage);
        }
        cp_async_commit();
        stage = stage + kMatvecStage<kSets> == ring + kMatvecDepth * kMatvecStage<kSets> ? ring : stage + kMatvecStage<kSets>;
    }
    cp_async_wait<0>();
    __syncthreads();  // the rings are empty: their place takes the partial sums
    // [warp][token][pair of columns of a lane][lane group]: a row of eight floats more keeps the four tokens a half warp stores
    // out of one another's banks
    float* part = reinterpret_cast<float*>(matvec_smem);
#pragma unroll
    for (uint32_t t = 0; t < kSets; ++t) {
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j) {
            float* dst = part + (warp * kTokens + t * 4u + tig) * kMatvecPartRow + j * 16u + g * 2u;
            *reinterpret_cast<float2*>(dst) = make_float2(sum[t][j][0], sum[t][j][1]);
            *reinterpret_cast<float2*>(dst + 64u) = make_float2(sum[t][j][2], sum[t][j][3]);
        }
    }
    __syncthreads();
    const uint32_t values = tokens * kMatvecCols;
    for (uint32_t i = threadIdx.x; i < values; i += kMatvecThreads) {
        const uint32_t token = i / kMatvecCols, at = i & (kMatvecCols - 1u);
        float v = 0.0f;
#pragma unroll
        for (uint32_t o = 0; o < kMatvecWarps; ++o) {
            v += part[(o * kTokens + token) * kMatvecPartRow + at];
        }
        total[token][at] = v;
    }
    __syncthreads();
    if (ctas > 1u) {
        cluster_sync_all();
    }
    // every CTA of the cluster writes its share of the pairs of columns
    for (uint32_t i = cta * kMatvecThreads + threadIdx.x; i < values / 2u; i += ctas * kMatvecThreads) {
        const uint32_t token = i / (kMatvecCols / 2u), pair = i & (kMatvecCols / 2u - 1u);
        const float* src = &total[token][(pair & 7u) * 16u + (pair >> 3) * 2u];  // pair & 7 names half and j: columns 8 half + 2 j
        float a = 0.0f, b = 0.0f;
        for (uint32_t o = 0; o < ctas; ++o) {
            a += ctas > 1u ? ld_cluster_f32(src, o) : src[0];
            b += ctas > 1u ? ld_cluster_f32(src + 1, o) : src[1];
        }
        const uint32_t c = n0 + 2u * pair;
        uint32_t row = rows[0];
#pragma unroll
        for (uint32_t t = 1; t < kTokens; ++t) {
            row = token == t ? rows[t] : row;
        }
        if (c < p.n) {
            constexpr float kSize = (float)(1 << kMatvecHeadroom);
            *reinterpret_cast<uint32_t*>(p.out + ((size_t)row * p.n + c) * 2u) = pack2<OutT>(a * kSize, b * kSize);
        }
    }
    if (ctas > 1u) {
        __syncwarp();
        cluster_sync_all();  // no CTA leaves while another may still read its sums
    }
}

}  // namespace catccos
