// Products of 8-bit codes with one fp32 scale for each block of 128, for sm_100a, dense and per expert:
//   C[i, j] = sum over blocks t of K:  sa[i, t] * sb[t, j / 128] * (sum over k in block t of A[i, k] B[k, j])
// (or sb[t, j]: B scaled by column, a weight's gradient).  With offsets [experts + 1] on the device, rows offsets[e] ..
// offsets[e + 1] of A meet expert e's B.
//
// The scales are no powers of two, so the tensor core cannot apply them: every block's products are a tensor-memory tile of
// their own, which the promotion warps read, scale and add to sums in registers while the next blocks are multiplied into
// other tiles.  128 columns of K are four tcgen05.mma kind::f8f6f4 (K = 32).
//
// Either operand may be stored with K or with its other axis running fastest: both are operand layouts of the tensor core, so
// that x W, dy W^T and x^T dy read the same codes without a transposed copy.  K need not be a multiple of 128: TMA fills the
// last block with zeros.
//
// This file: what the two forms share, and the one for few rows (an expert); block_gemm_pair.cuh: the one for many.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "block_plan.hpp"
#include "common.cuh"
#include "mx_gemm_small.cuh"
#include "mx_grouped_gemm.cuh"

namespace catccos {

constexpr uint32_t kBlockFewThreads = 256;

struct BlockGemmParams {
    const uint8_t *a, *b;                                  // the codes, for block_few_again
    size_t a_line, b_line, b_matrix;                       // bytes from one line, one expert's matrix to the next
    const float* a_scales;
    size_t a_scale_row, a_scale_block;                     // floats from one row's (block's) scale to the next
    const float* b_scales;
    size_t b_scale_block, b_scale_col, b_scale_matrix;     // from one block of K, of columns (by column: 1), one expert to the next
    const int32_t* offsets;                                // nullptr: one matrix
    void* c;
    uint32_t rows, experts, N, K;
    uint32_t a_fmt, b_fmt;                                 // 0 = E4M3, 1 = E5M2
    uint32_t a_cols, b_rows;                               // 1: A is stored [K, rows]; B [N, K]
    uint32_t parts;                                        // few rows: CTAs of a cluster that share K (a power of two)
    uint64_t bar_timeout_ns;
    StatusBlock* status;
};

// mbar_wait_warp whose first polls do not look at the clock: reading it takes longer than what these barriers are waited for (a
// tile's way from the tensor core to the promotion and back counts in every block of K).
__device__ __forceinline__ bool mbar_wait_soon(uint64_t* bar, uint32_t parity, StatusBlock* st, uint32_t id, uint32_t stage, uint64_t limit_ns)
{
#pragma unroll 1
    for (uint32_t i = 0; i < 4096u; ++i) {
        if (__all_sync(0xFFFFFFFFu, mbar_try_wait(bar, parity))) {
            return true;
        }
    }
    return mbar_wait_warp(bar, parity, st, id, stage, limit_ns);
}

// Instruction descriptor of kind::f8f6f4 with fp32 accumulators: make_idesc_mxf8's fields without the scales' (bits 4, 5: fp32)
__host__ __device__ constexpr uint32_t make_idesc_f8(uint32_t M, uint32_t N, uint32_t a_fmt, uint32_t b_fmt, bool a_mn, bool b_mn)
{
    return (1u << 4) | (a_fmt << 7) | (b_fmt << 10) | ((a_mn ? 1u : 0u) << 15) | ((b_mn ? 1u : 0u) << 16) | ((N >> 3) << 17) | ((M >> 4) << 24);
}

// A tile load with the announcement of its bytes, by one lane of a converged warp: with a branch on the lane such instructions take
// several times as long to issue.
__device__ __forceinline__ void tma_expect_and_load_2d(void* smem_dst, const void* tmap, uint64_t* bar, uint32_t bytes, uint32_t x, uint32_t y)
{
    asm volatile(
        "{\n\t"
        ".reg .pred one;\n\t"
        "elect.sync _|one, 0xffffffff;\n\t"
        "@one mbarrier.arrive.expect_tx.shared::cta.b64 _, [%2], %5;\n\t"
        "@one cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];\n\t"
        "}"
        ::"r"(smem_u32(smem_dst)), "l"(tmap), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(bytes)
        : "memory");
}

__device__ __forceinline__ void tma_expect_and_load_3d(void* smem_dst, const void* tmap, uint64_t* bar, uint32_t bytes, uint32_t x, uint32_t y, uint32_t z)
{
    asm volatile(
        "{\n\t"
        ".reg .pred one;\n\t"
        "elect.sync _|one, 0xffffffff;\n\t"
        "@one mbarrier.arrive.expect_tx.shared::cta.b64 _, [%2], %6;\n\t"
        "@one cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];\n\t"
        "}"
        ::"r"(smem_u32(smem_dst)), "l"(tmap), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z), "r"(bytes)
        : "memory");
}

// 32 lanes x 16 consecutive 32-bit columns -> 16 registers per thread; they hold the values behind tmem_ld_fence of them
__device__ __forceinline__ void tmem_ld_16(uint32_t taddr, float (&r)[16])
{
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]), "=f"(r[7]), "=f"(r[8]),
          "=f"(r[9]), "=f"(r[10]), "=f"(r[11]), "=f"(r[12]), "=f"(r[13]), "=f"(r[14]), "=f"(r[15])
        : "r"(taddr)
        : "memory");
}

// Waits for this thread's tensor-memory loads; nothing that reads r moves in front of it.
__device__ __forceinline__ void tmem_ld_fence(float (&r)[16])
{
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+f"(r[0]), "+f"(r[1]), "+f"(r[2]), "+f"(r[3]), "+f"(r[4]), "+f"(r[5]), "+f"(r[6]), "+f"(r[7]), "+f"(r[8]),
                   "+f"(r[9]), "+f"(r[10]), "+f"(r[11]), "+f"(r[12]), "+f"(r[13]), "+f"(r[14]), "+f"(r[15])
                 :
                 : "memory");
}

// Sixteen columns of a row to global memory; p is aligned to their size or 32 bytes
template <typename OutT>
__device__ __forceinline__ void store_16(OutT* p, const float* v)
{
    if constexpr (sizeof(OutT) == 4) {
        uint32_t o[2][8];
#pragma unroll
        for (uint32_t i = 0; i < 16; ++i) {
            o[i / 8][i % 8] = __float_as_uint(v[i]);
        }
        st_global_v8(p, o[0]);
        st_global_v8(p + 8, o[1]);
    } else {
        uint32_t o[8];
#pragma unroll
        for (uint32_t i = 0; i < 8; ++i) {
            o[i] = pack2<OutT>(v[2 * i], v[2 * i + 1]);
        }
        st_global_v8(p, o);
    }
}

// (a0, a1) += (x0, x1) * (y0, y1), each rounded once, in one instruction
__device__ __forceinline__ void fma_2(float& a0, float& a1, float x0, float x1, float y0, float y1)
{
    asm("{\n\t"
        ".reg .b64 a, x, y;\n\t"
        "mov.b64 a, {%0, %1};\n\t"
        "mov.b64 x, {%2, %3};\n\t"
        "mov.b64 y, {%4, %5};\n\t"
        "fma.rn.f32x2 a, x, y, a;\n\t"
        "mov.b64 {%0, %1}, a;\n\t"
        "}"
        : "+f"(a0), "+f"(a1)
        : "f"(x0), "f"(x1), "f"(y0), "f"(y1));
}

// (x0, x1) *= (y0, y1)
__device__ __forceinline__ void mul_2(float& x0, float& x1, float y0, float y1)
{
    asm("{\n\t"
        ".reg .b64 x, y;\n\t"
        "mov.b64 x, {%0, %1};\n\t"
        "mov.b64 y, {%2, %3};\n\t"
        "mul.rn.f32x2 x, x, y;\n\t"
        "mov.b64 {%0, %1}, x;\n\t"
        "}"
        : "+f"(x0), "+f"(x1)
        : "f"(y0), "f"(y1));
}

// sixteen sums += f * the columns of this lane's row; by column: f * scale[column] * them (scale: address in shared memory, 16-byte
// aligned)
template <bool kByColumn>
__device__ __forceinline__ void add_scaled(float* acc, const float (&v)[16], float f, uint32_t scale)
{
#pragma unroll
    for (uint32_t c = 0; c < 16; c += 4) {
        float4 g = make_float4(f, f, f, f);
        if (kByColumn) {
            const float4 s = ld_shared_v4(scale + c * 4u);
            g = make_float4(f * s.x, f * s.y, f * s.z, f * s.w);
        }
        fma_2(acc[c], acc[c + 1], v[c], v[c + 1], g.x, g.y);
        fma_2(acc[c + 2], acc[c + 3], v[c + 2], v[c + 3], g.z, g.w);
    }
}

__device__ __forceinline__ float ld_shared_f32(uint32_t addr)
{
    float v;
    asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(addr));
    return v;
}

// 32 columns of row `lane` to a box of 32 rows in shared memory that TMA stores: 16-byte pieces in its swizzle of 64 (16-bit types) or
// 128 bytes.
template <typename OutT>
__device__ __forceinline__ void stage_out(uint8_t* box, uint32_t lane, const float* v)
{
    constexpr uint32_t kPieces = 2 * sizeof(OutT), kPer = 32 / kPieces;  // of a row; values of one
    const uint32_t turn = sizeof(OutT) == 4 ? lane & 7u : (lane >> 1) & 3u;
#pragma unroll
    for (uint32_t i = 0; i < kPieces; ++i) {
        uint4 o;
        if constexpr (sizeof(OutT) == 4) {
            o = make_uint4(__float_as_uint(v[i * kPer]), __float_as_uint(v[i * kPer + 1]), __float_as_uint(v[i * kPer + 2]), __float_as_uint(v[i * kPer + 3]));
        } else {
            o = make_uint4(pack2<OutT>(v[i * kPer], v[i * kPer + 1]), pack2<OutT>(v[i * kPer + 2], v[i * kPer + 3]),
                           pack2<OutT>(v[i * kPer + 4], v[i * kPer + 5]), pack2<OutT>(v[i * kPer + 6], v[i * kPer + 7]));
        }
        *reinterpret_cast<uint4*>(box + lane * (32u * sizeof(OutT)) + ((i ^ turn) << 4)) = o;
    }
}

// A line's scales of blocks kb .. kb + 3 of K (those behind the last: 1, an ordinary one); they are `step` floats apart.
__device__ __forceinline__ void load_scales(const float* line, size_t step, uint32_t kb, uint32_t blocks, float (&v)[4])
{
    const float* at = line + kb * step;
    if (step == 1 && kb + 4u <= blocks && ((uintptr_t)at & 15u) == 0u) {
        const float4 w = __ldcg(reinterpret_cast<const float4*>(at));
        v[0] = w.x, v[1] = w.y, v[2] = w.z, v[3] = w.w;
    } else {
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j) {
            v[j] = kb + j < blocks ? __ldcg(at + j * step) : 1.0f;
        }
    }
}

// ---- two scales whose product is not in fp32's range ----
// A block's sum v (with finite codes 0, or 2^-32 to 2^39 in size) is added as v * f, one product of the scales for many sums.  f is kHeld * sa *
// sb, and what is held is kHeld times the result: where f is below fp32's normal numbers, v * f is then off by 2^39 * 2^-150 / 2^40 of the
// result at most, less than half of fp32's smallest step.  (Without kHeld the product for a block of zeros, whose scale is 2^-109 or 2^-116,
// and small weights would be there already.)
//
// Upwards, f has to stay below 2^64, so that no sum of blocks overflows where the result does not, and that v = 0 stays 0 beside finite
// scales.  The warps that make the factors look for larger ones.
//   CTA pairs: the group of four blocks of K is marked; with it the promotion goes on to a second loop up to the end of the unit, which holds
//   the result itself and adds (v * g) * f with g = 2^64 or 2^-64 and f that much smaller or larger: v * g is exact, and what is then outside
//   of f's range is outside of the result's.  By column: ((v * near) * sb) * rest with sa = near * rest.
//   Few rows: before a CTA ends, rows with such a block are computed again from the codes in global memory.
// A row without such blocks gets the same result whatever the others have (by column: but for its last bit).  With such scales in 5 % of the
// rows 8192 x 2304 x 7168 takes 220 us (150), 16 x 4096 x 7168 with one such row 91 (10.9).  Other calls pay 0 to 2 %, short ones (5 to 20 us) 1 to
// 4, on pairs 4 to 10.  A choice inside one loop cost them 5 to 25 %, for few rows a second loop 2 to 7, on pairs the rows at the end 3 on large
// products.
constexpr float kHeld = 0x1p40f;
constexpr uint32_t kFactorLimit = 0x5F800000u;  // 2^64 as bits; a negative factor, an infinity and a NaN are above it, too, and looked at again

__device__ __forceinline__ bool is_finite(float f) { return __float_as_uint(f) * 2u < 0xFF000000u; }

__device__ __forceinline__ bool is_finite_and_not_zero(float f) { return __float_as_uint(f) * 2u - 1u < 0xFEFFFFFFu; }

// Whether f, as kHeld times the product of the two scales, does not stand for them (NaN may be 0 times kHeld * sb)
__device__ __forceinline__ bool needs_both_scales(float sa, float sb, float f)
{
    return !(fabsf(f) < 0x1p64f) && is_finite(sa) && is_finite(sb);
}

// The factor of a marked group: v * sa * sb is (v * g) * it.
__device__ __forceinline__ float wide_factor(float sa, float sb, float& g)
{
    float f = sa * sb;
    const float size = fabsf(f);
    g = 1.0f;
    if (!(size >= 0x1p-126f && size <= 0x1.fffffep127f) && is_finite_and_not_zero(sa) && is_finite_and_not_zero(sb)) {
        // of a product of 2^128 or more neither scale is below 1, of one below 2^-126 neither is above 2^23
        const bool large = size > 1.0f;
        const float shift = large ? 0x1p-32f : 0x1p32f;
        f = (sa * shift) * (sb * shift);
        f = fminf(fmaxf(f, -0x1.fffffep127f), 0x1.fffffep127f);  // above 2^192 in all: any v but 0 is infinite, and 0 is 0
        g = large ? 0x1p64f : 0x1p-64f;
    }
    return f;
}

// sums *= s
template <uint32_t kCount>
__device__ __forceinline__ void scale_sums(float (&sums)[kCount], float s)
{
#pragma unroll
    for (uint32_t i = 0; i < kCount; i += 2) {
        mul_2(sums[i], sums[i + 1], s, s);
    }
}

// s = near * rest, exactly: rest a power of two, near from 2^-86 to 2^65 (an infinity or a NaN stays in near)
__device__ __forceinline__ void split_scale(float s, float& near, float& rest)
{
    const int e = (int)((__float_as_uint(s) >> 23) & 0xFFu) - 127;
    const int shift = e - min(max(e, -64), 64);
    near = s * __uint_as_float((uint32_t)(127 - shift) << 23);
    rest = __uint_as_float((uint32_t)(127 + shift) << 23);
}

// By column, in the second loop: sixteen sums += f * scale[column] * the columns of this lane's row, as ((v * near) * scale) * rest with f =
// near * rest: the products on the way are outside of fp32's range only where the result is.
__device__ __forceinline__ void add_scaled_apart(float* acc, float (&v)[16], float f, uint32_t scale)
{
    float near, rest;
    split_scale(f, near, rest);
#pragma unroll
    for (uint32_t c = 0; c < 16; c += 4) {
        const float4 s = ld_shared_v4(scale + c * 4u);
        mul_2(v[c], v[c + 1], near, near);
        mul_2(v[c + 2], v[c + 3], near, near);
        mul_2(v[c], v[c + 1], s.x, s.y);
        mul_2(v[c + 2], v[c + 3], s.z, s.w);
        fma_2(acc[c], acc[c + 1], v[c], v[c + 1], rest, rest);
        fma_2(acc[c + 2], acc[c + 3], v[c + 2], v[c + 3], rest, rest);
    }
}

// One warp: where each expert's rows and row tiles begin (count_grouped_tiles), or the one matrix without offsets.
__device__ __forceinline__ void count_block_tiles(const BlockGemmParams& p, uint32_t tile_rows, uint32_t* tiles, uint32_t* row_begin,
                                                  uint32_t* row_end, uint32_t lane)
{
    if (p.offsets != nullptr) {
        GroupedParams g = {};
        g.offsets = p.offsets;
        g.rows = p.rows;
        g.experts = p.experts;
        count_grouped_tiles(g, tile_rows, tiles, row_begin, row_end, lane);
    } else if (lane == 0) {
        tiles[0] = 0;
        tiles[1] = (p.rows + tile_rows - 1u) / tile_rows;
        row_begin[0] = 0;
        row_end[0] = p.rows;
    }
}

// One block of K: four products (K = 32) into the tile at tmem_d, then arrivals on `done` and `empty` when they are finished.  Called
// by a converged warp, of which one lane issues everything: with a branch on the lane it takes three times as long.
__device__ __forceinline__ void umma_f8_block(uint32_t tmem_d, uint32_t a_lo, uint32_t a_hi, uint32_t a_step, uint32_t b_lo, uint32_t b_hi,
                                              uint32_t b_step, uint32_t idesc, uint64_t* done, uint64_t* empty)
{
    asm volatile(
        "{\n\t"
        ".reg .pred one, add;\n\t"
        ".reg .b64 da, db;\n\t"
        ".reg .b32 a, b;\n\t"
        "elect.sync _|one, 0xffffffff;\n\t"
        "setp.ne.b32 add, 0, 0;\n\t"
        "mov.b64 da, {%1, %2};\n\t"
        "mov.b64 db, {%4, %5};\n\t"
        "@one tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], da, db, %7, add;\n\t"
        "setp.eq.b32 add, 0, 0;\n\t"
        "add.u32 a, %1, %3;\n\t"
        "add.u32 b, %4, %6;\n\t"
        "mov.b64 da, {a, %2};\n\t"
        "mov.b64 db, {b, %5};\n\t"
        "@one tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], da, db, %7, add;\n\t"
        "add.u32 a, a, %3;\n\t"
        "add.u32 b, b, %6;\n\t"
        "mov.b64 da, {a, %2};\n\t"
        "mov.b64 db, {b, %5};\n\t"
        "@one tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], da, db, %7, add;\n\t"
        "add.u32 a, a, %3;\n\t"
        "add.u32 b, b, %6;\n\t"
        "mov.b64 da, {a, %2};\n\t"
        "mov.b64 db, {b, %5};\n\t"
        "@one tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], da, db, %7, add;\n\t"
        "@one tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%8];\n\t"
        "@one tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%9];\n\t"
        "}"
        ::"r"(tmem_d), "r"(a_lo), "r"(a_hi), "r"(a_step), "r"(b_lo), "r"(b_hi), "r"(b_step), "r"(idesc), "r"(smem_u32(done)), "r"(smem_u32(empty))
        : "memory");
}

// Both barriers, looked at together.
__device__ __forceinline__ bool mbar_wait_both(uint64_t* bar1, uint32_t parity1, uint64_t* bar2, uint32_t parity2, StatusBlock* st, uint32_t id,
                                               uint32_t stage, uint64_t limit_ns)
{
#pragma unroll 1
    for (uint32_t i = 0; i < 4096u; ++i) {
        const bool first = mbar_try_wait(bar1, parity1), second = mbar_try_wait(bar2, parity2);
        if (__all_sync(0xFFFFFFFFu, first && second)) {
            return true;
        }
    }
    return mbar_wait_warp(bar1, parity1, st, id, stage, limit_ns) && mbar_wait_warp(bar2, parity2, st, id + 1u, stage, limit_ns);
}

// ------------------------------------------------------------------------------------------
// few rows
// ------------------------------------------------------------------------------------------
// Up to 64 rows (of an expert) are bound by streaming the weights and by latencies, so the operands change sides: 128 columns of the
// weight are the rows of a tile, kRows rows of A its columns.  A lane then has one weight column and kRows sums, and every warp of
// the promotion has work however few the rows are.  (With the rows of A on the lanes the one warp that has 16 rows took 600 cycles a
// block and 16 x 4096 x 7168 12.9 us.)  Measured: 16 x 4096 x 7168 9.3 us in a caller's loop (3.2 TB/s; launch and set-up 3, the meeting 1.3,
// the weights alone 4.6), 10.8 back to back; 128 rows over 32 experts of 4096 x 7168 128 us: the used experts' weights at HBM's rate.
//
// K may be cut over the CTAs of a cluster (p.parts: 1, 2, 4 or 8), so that calls of few tiles stream their weights with every SM.
// Their sums meet in distributed shared memory: part d owns 128 / parts of the weight columns, the others push theirs into its idle
// ring, and it adds them in ascending order of the parts.  A launch with parts has a cluster for every unit there may be.
//
// 256 threads, two CTAs to an SM: warps 0-3 promotion and output (lane quarter = warp), 4 and 5 TMA for B and A, 6 MMA, 7 the factors:
// the scales of the rows times the weight's, for groups of four blocks of K (every unit begins with a group of its own).
template <uint32_t kRows>
struct BlockFewSmem {
    static constexpr uint32_t kStages = kRows == 64 ? 4 : 5;
    static constexpr uint32_t kWBytes = kBlockFewColumns * 128, kXBytes = kRows * 128;
    static constexpr uint32_t kTiles = 4, kTmemCols = kTiles * kRows;
    static constexpr uint32_t kGroups = 4;  // of factors, on their way
    static constexpr uint32_t kOffW = 0;
    static constexpr uint32_t kOffX = kOffW + kStages * kWBytes;
    static constexpr uint32_t kOffFactor = kOffX + kStages * kXBytes;  // [4 blocks][kRows] a group
    static constexpr uint32_t kOffBar = kOffFactor + kGroups * 4 * kRows * 4;
    static constexpr uint32_t kNumBars = 2 * kStages + 2 * kTiles + 2 * kGroups;
    static constexpr uint32_t kOffTmemPtr = kOffBar + kNumBars * 8;
    static constexpr uint32_t kOffDead = kOffTmemPtr + 4;  // a part of this cluster has given up
    static constexpr uint32_t kOffLarge = kOffTmemPtr + 8;  // some factor was too large, in this CTA or another part
    static constexpr uint32_t kOffTiles = kOffTmemPtr + 16;
    static constexpr uint32_t kPitch = kRows + 4;  // floats of a weight column's sums in the exchange
    static constexpr uint32_t dynamic_bytes(uint32_t experts) { return kOffTiles + (3u * experts + 1u) * 4u + 1024u; }
    static_assert(kBlockFewColumns * kPitch * 4 <= kOffX && kBlockFewThreads / 32 * kBlockFewColumns * 4 <= kOffX, "the sums of all parts fit the idle ring");
};

// The values of two codes
__device__ __forceinline__ float2 code_values(uint32_t two, uint32_t e5m2)
{
    uint32_t halves;
    if (e5m2) {
        asm("{\n\t.reg .b16 c;\n\tcvt.u16.u32 c, %1;\n\tcvt.rn.f16x2.e5m2x2 %0, c;\n\t}" : "=r"(halves) : "r"(two));
    } else {
        asm("{\n\t.reg .b16 c;\n\tcvt.u16.u32 c, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, c;\n\t}" : "=r"(halves) : "r"(two));
    }
    return __half22float2(*reinterpret_cast<const __half2*>(&halves));
}

// The units of a CTA once more (with parts, the columns that it owns), after a factor was too large: rows of which a block needs both
// scales are computed again.  All warps have a row together, a warp every eighth block of K, a lane four columns and sixteen steps of K at
// a time; sums: the idle ring.
template <uint32_t kRows, typename OutT>
__device__ __forceinline__ void block_few_again(const BlockGemmParams& p, const uint32_t* tiles, float* sums)
{
    constexpr uint32_t kWarps = kBlockFewThreads / 32;
    const uint32_t n_tiles = (p.N + kBlockFewColumns - 1) / kBlockFewColumns, k_blocks = (p.K + 127u) / 128u;
    const uint32_t own = kBlockFewColumns / p.parts, clusters = gridDim.x / p.parts, warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
    const uint32_t* row_begin = tiles + p.experts + 1u;
    const uint32_t num_units = p.parts > 1u ? min(tiles[p.experts] * n_tiles, clusters) : tiles[p.experts] * n_tiles;
    GroupedWalk walk;
    for (uint32_t unit = blockIdx.x / p.parts; unit < num_units; unit += clusters) {
        const TileCoord tc = walk.seek(tiles, n_tiles, unit);
        const uint32_t first = row_begin[walk.e] + tc.m_tile * kRows, rows = min(row_begin[p.experts + walk.e] - first, kRows);
        const uint32_t n0 = tc.n_tile * kBlockFewColumns + (blockIdx.x & (p.parts - 1u)) * own, n = n0 + 4u * lane;
        const uint32_t columns = n0 < p.N ? min(p.N - n0, own) : 0u;  // a multiple of 16
        const uint8_t* b_codes = p.b + walk.e * p.b_matrix;
        const float* sb_of = p.b_scales + walk.e * p.b_scale_matrix + tc.n_tile * p.b_scale_col;
        for (uint32_t r = 0; r < rows; ++r) {
            const size_t row = first + r;
            const float* sa_of = p.a_scales + row * p.a_scale_row;
            bool both = false;
            for (uint32_t kb = threadIdx.x; kb < k_blocks; kb += kBlockFewThreads) {
                const float sa = __ldcg(sa_of + kb * p.a_scale_block), sb = __ldcg(sb_of + kb * p.b_scale_block);
                both = both || needs_both_scales(sa, sb, sa * (sb * kHeld));
            }
            if (!__syncthreads_or(both)) {
                continue;
            }
            float acc[4] = {};
            for (uint32_t kb = warp; kb < k_blocks && 4u * lane < columns; kb += kWarps) {
                float v[4] = {}, near, rest;
                const uint32_t end = min(p.K, kb * 128u + 128u);  // a multiple of 16
#pragma unroll 2
                for (uint32_t k = kb * 128u; k < end; k += 16u) {
                    const uint4 x = *reinterpret_cast<const uint4*>(p.a + row * p.a_line + k);
                    const uint32_t a[4] = {x.x, x.y, x.z, x.w};
                    uint32_t b[16];  // four steps of each of four columns, four times
                    if (p.b_rows) {
#pragma unroll
                        for (uint32_t c = 0; c < 4; ++c) {
                            const uint4 w = *reinterpret_cast<const uint4*>(b_codes + (n + c) * p.b_line + k);
                            b[c] = w.x, b[4 + c] = w.y, b[8 + c] = w.z, b[12 + c] = w.w;
                        }
                    } else {
#pragma unroll
                        for (uint32_t i = 0; i < 16; i += 4) {
                            uint32_t w[4];
#pragma unroll
                            for (uint32_t j = 0; j < 4; ++j) {
                                w[j] = *reinterpret_cast<const uint32_t*>(b_codes + (k + i + j) * p.b_line + n);
                            }
#pragma unroll
                            for (uint32_t c = 0; c < 4; ++c) {
                                b[i + c] = __byte_perm(__byte_perm(w[0], w[1], c | ((4u + c) << 4)), __byte_perm(w[2], w[3], c | ((4u + c) << 4)), 0x5410u);
                            }
                        }
                    }
#pragma unroll
                    for (uint32_t i = 0; i < 16; i += 2) {
                        const float2 xs = code_values(a[i / 4] >> (8u * (i & 3u)) & 0xFFFFu, p.a_fmt);
#pragma unroll
                        for (uint32_t c = 0; c < 4; ++c) {
                            const float2 ws = code_values(b[i / 4 * 4 + c] >> (8u * (i & 3u)) & 0xFFFFu, p.b_fmt);
                            v[c] = fmaf(xs.y, ws.y, fmaf(xs.x, ws.x, v[c]));
                        }
                    }
                }
                split_scale(__ldcg(sa_of + kb * p.a_scale_block), near, rest);
                const float sb = __ldcg(sb_of + kb * p.b_scale_block);
#pragma unroll
                for (uint32_t c = 0; c < 4; ++c) {
                    acc[c] = fmaf(v[c] * near * sb, rest, acc[c]);
                }
            }
            *reinterpret_cast<float4*>(sums + warp * kBlockFewColumns + 4u * lane) = make_float4(acc[0], acc[1], acc[2], acc[3]);
            __syncthreads();
            if (threadIdx.x < columns) {
                float sum = sums[threadIdx.x];
                for (uint32_t w = 1; w < kWarps; ++w) {
                    sum += sums[w * kBlockFewColumns + threadIdx.x];
                }
                static_cast<OutT*>(p.c)[row * p.N + n0 + threadIdx.x] = static_cast<OutT>(sum);
            }
        }
    }
}

template <uint32_t kRows, typename OutT>
__global__ void __launch_bounds__(kBlockFewThreads, 2)
block_gemm_few_kernel(const __grid_constant__ CUtensorMap tmap_x, const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ BlockGemmParams p)
{
    using S = BlockFewSmem<kRows>;
    constexpr uint32_t kStages = S::kStages, kTiles = S::kTiles;

    grid_dep_launch();
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + S::kOffBar);
    uint64_t* empty = full + kStages;
    uint64_t* tmem_full = empty + kStages;
    uint64_t* tmem_empty = tmem_full + kTiles;
    uint64_t* scale_full = tmem_empty + kTiles;
    uint64_t* scale_empty = scale_full + S::kGroups;
    uint32_t* tmem_ptr_smem = reinterpret_cast<uint32_t*>(smem + S::kOffTmemPtr);
    uint32_t* dead = reinterpret_cast<uint32_t*>(smem + S::kOffDead);
    volatile uint32_t* large = reinterpret_cast<volatile uint32_t*>(smem + S::kOffLarge);
    uint32_t* tiles = reinterpret_cast<uint32_t*>(smem + S::kOffTiles);
    uint32_t* row_begin = tiles + p.experts + 1u;
    uint32_t* row_end = row_begin + p.experts;

    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
    const uint32_t n_tiles = (p.N + kBlockFewColumns - 1) / kBlockFewColumns;
    const uint32_t k_blocks = (p.K + 127u) / 128u;
    const uint32_t part = blockIdx.x & (p.parts - 1u), first_unit = blockIdx.x / p.parts, stride = gridDim.x / p.parts;
    const uint32_t kb0 = (uint32_t)((uint64_t)part * k_blocks / p.parts), kb1 = (uint32_t)((uint64_t)(part + 1u) * k_blocks / p.parts);
    const uint64_t bar_ns = p.bar_timeout_ns;

    if (threadIdx.x == 128) {
        for (uint32_t s = 0; s < kStages; ++s) {
            mbar_init(&full[s], 2);  // both producers (expect_tx)
            mbar_init(&empty[s], 1);
        }
        for (uint32_t b = 0; b < kTiles; ++b) {
            mbar_init(&tmem_full[b], 1);
            mbar_init(&tmem_empty[b], 4);
        }
        for (uint32_t i = 0; i < S::kGroups; ++i) {
            mbar_init(&scale_full[i], 1);
            mbar_init(&scale_empty[i], 4);
        }
        *dead = 0u;
        *large = 0u;
        mbar_fence_init();
        tma_prefetch_desc(&tmap_x);
        tma_prefetch_desc(&tmap_w);
    }
    if (warp == 6) {
        tmem_alloc(tmem_ptr_smem, S::kTmemCols);
        tmem_relinquish();
    }
    grid_dep_wait();
    if (warp == 0) {
        count_block_tiles(p, kRows, tiles, row_begin, row_end, lane);
    }
    tcgen05_fence_before();
    __syncthreads();
    tcgen05_fence_after();
    const uint32_t tmem_base = *tmem_ptr_smem;
    // Offsets that do not ascend may give more units than the host reckoned with: with parts a cluster meets for one unit, no more.
    const uint32_t num_units = p.parts > 1u ? min(tiles[p.experts] * n_tiles, stride) : tiles[p.experts] * n_tiles;
    bool alive = true;  // false once a wait of this role has given up
    GroupedWalk walk;

    if (warp == 4 || warp == 5) {
        // ------------------------------- TMA producers ------------------------------------
        uint32_t s = 0, ph = 1;
        for (uint32_t unit = first_unit; alive && unit < num_units; unit += stride) {
            const TileCoord tc = walk.seek(tiles, n_tiles, unit);
            const uint32_t m0 = row_begin[walk.e] + tc.m_tile * kRows, n0 = tc.n_tile * kBlockFewColumns;
            for (uint32_t kb = kb0; kb < kb1; ++kb) {
                const uint32_t k = kb * 128u;
                alive = mbar_wait_soon(&empty[s], ph, p.status, 400, s, bar_ns);
                if (!alive) {
                    break;
                }
                if (warp == 4) {
                    tma_expect_and_load_3d(smem + S::kOffW + s * S::kWBytes, &tmap_w, &full[s], S::kWBytes, p.b_rows ? k : n0, p.b_rows ? n0 : k, walk.e);
                } else {  // rows behind the expert's last come along: their products are not looked at
                    tma_expect_and_load_2d(smem + S::kOffX + s * S::kXBytes, &tmap_x, &full[s], S::kXBytes, k, m0);
                }
                s = s + 1u == kStages ? 0u : s + 1u;
                ph ^= s == 0u ? 1u : 0u;
            }
        }
    } else if (warp == 6) {
        // ------------------------------- MMA issuer ---------------------------------------
        const uint32_t idesc = make_idesc_f8(kBlockFewColumns, kRows, p.b_fmt, p.a_fmt, p.b_rows == 0u, false);
        const uint64_t desc_k = make_smem_desc(0, 16, 1024, 2), desc_w = p.b_rows ? desc_k : make_smem_desc(0, 16384, 1024, 2);
        const uint32_t hi_w = (uint32_t)(desc_w >> 32), hi_x = (uint32_t)(desc_k >> 32);
        const uint32_t w_lo0 = (uint32_t)desc_w | (smem_u32(smem + S::kOffW) >> 4);
        const uint32_t x_lo0 = (uint32_t)desc_k | (smem_u32(smem + S::kOffX) >> 4);
        const uint32_t step_w = (p.b_rows ? 32u : 4096u) >> 4;
        uint32_t it = 0, s = 0, ph = 0;
        for (uint32_t unit = first_unit; alive && unit < num_units; unit += stride) {
            for (uint32_t kb = kb0; kb < kb1; ++kb, ++it) {
                const uint32_t b = it % kTiles;
                alive = mbar_wait_both(&full[s], ph, &tmem_empty[b], ((it / kTiles) & 1u) ^ 1u, p.status, 401, s, bar_ns);
                if (!alive) {
                    break;  // nothing is issued, and no tile reported, after a wait has given up
                }
                tcgen05_fence_after();
                umma_f8_block(tmem_base + b * kRows, w_lo0 + s * (S::kWBytes >> 4), hi_w, step_w, x_lo0 + s * (S::kXBytes >> 4), hi_x, 32u >> 4, idesc,
                              &tmem_full[b], &empty[s]);
                s = s + 1u == kStages ? 0u : s + 1u;
                ph ^= s == 0u ? 1u : 0u;
            }
        }
    } else if (warp == 7) {
        // ------------------------------- factors ------------------------------------------
        constexpr uint32_t kPerLane = (kRows + 31) / 32;
        uint32_t group = 0;
        for (uint32_t unit = first_unit; alive && unit < num_units; unit += stride) {
            const TileCoord tc = walk.seek(tiles, n_tiles, unit);
            const uint32_t row = row_begin[walk.e] + tc.m_tile * kRows + lane, end = row_end[walk.e];
            const float* w_scales = p.b_scales + walk.e * p.b_scale_matrix + tc.n_tile * p.b_scale_col;
            for (uint32_t kb = kb0; kb < kb1; kb += 4u, ++group) {
                float x[kPerLane][4], w[4];
                load_scales(w_scales, p.b_scale_block, kb, kb1, w);
#pragma unroll
                for (uint32_t i = 0; i < kPerLane; ++i) {
                    load_scales(p.a_scales + min(row + 32u * i, end - 1u) * p.a_scale_row, p.a_scale_block, kb, kb1, x[i]);
                }
                const uint32_t slot = group % S::kGroups;
                alive = mbar_wait_soon(&scale_empty[slot], ((group / S::kGroups) & 1u) ^ 1u, p.status, 405, slot, bar_ns);
                if (!alive) {
                    break;
                }
                float* factor = reinterpret_cast<float*>(smem + S::kOffFactor) + slot * (4u * kRows) + lane;
                uint32_t most = 0;
#pragma unroll
                for (uint32_t j = 0; j < 4; ++j) {
                    const float w_held = w[j] * kHeld;
#pragma unroll
                    for (uint32_t i = 0; i < kPerLane; ++i) {
                        const float f = x[i][j] * w_held;
                        most = max(most, __float_as_uint(f));
                        if (lane < kRows) {
                            factor[j * kRows + 32u * i] = f;
                        }
                    }
                }
                if (__builtin_expect(most >= kFactorLimit, 0)) {
#pragma unroll
                    for (uint32_t i = 0; i < kPerLane * 4; ++i) {
                        if (needs_both_scales(x[i / 4][i % 4], w[i % 4], x[i / 4][i % 4] * (w[i % 4] * kHeld))) {
                            *large = 1u;
                        }
                    }
                }
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(&scale_full[slot]);
                }
            }
        }
    } else {
        // ------------------------------- promotion and output -----------------------------
        const uint32_t tmem = tmem_base + ((warp * 32u) << 16), column = warp * 32u + lane;
        uint32_t it = 0, group = 0;
        for (uint32_t unit = first_unit; alive && unit < num_units; unit += stride) {
            const TileCoord tc = walk.seek(tiles, n_tiles, unit);
            const uint32_t first = row_begin[walk.e] + tc.m_tile * kRows, rows = min(row_end[walk.e] - first, kRows);
            const uint32_t n0 = tc.n_tile * kBlockFewColumns;
            float acc[kRows] = {};
            for (uint32_t kb = kb0; kb < kb1; ++kb, ++it) {
                const uint32_t b = it % kTiles, slot = group % S::kGroups, j = (kb - kb0) & 3u;
                alive = j == 0u ? mbar_wait_both(&tmem_full[b], (it / kTiles) & 1u, &scale_full[slot], (group / S::kGroups) & 1u, p.status, 406, b, bar_ns)
                                : mbar_wait_soon(&tmem_full[b], (it / kTiles) & 1u, p.status, 406, b, bar_ns);
                if (!alive) {
                    break;  // a tile that never filled is not written out
                }
                tcgen05_fence_after();
                const float4* factor = reinterpret_cast<const float4*>(smem + S::kOffFactor) + (slot * 4u + j) * (kRows / 4);
#pragma unroll
                for (uint32_t c = 0; c < kRows; c += 16) {
                    if (c < rows) {
                        float v[16];
                        tmem_ld_16(tmem + b * kRows + c, v);
                        tmem_ld_fence(v);
#pragma unroll
                        for (uint32_t i = 0; i < 16; i += 4) {
                            const float4 f = factor[(c + i) / 4];
                            fma_2(acc[c + i], acc[c + i + 1], v[i], v[i + 1], f.x, f.y);
                            fma_2(acc[c + i + 2], acc[c + i + 3], v[i + 2], v[i + 3], f.z, f.w);
                        }
                    }
                }
                tcgen05_fence_before();
                __syncwarp();
                const bool group_end = j == 3u || kb + 1u == kb1;
                if (lane == 0) {
                    mbar_arrive(&tmem_empty[b]);
                    if (group_end) {
                        mbar_arrive(&scale_empty[slot]);
                    }
                }
                group += group_end ? 1u : 0u;
            }
            scale_sums(acc, 1.0f / kHeld);
            OutT* out = static_cast<OutT*>(p.c) + (size_t)first * p.N + n0;
            if (p.parts == 1u) {
                if (alive && n0 + column < p.N) {
#pragma unroll
                    for (uint32_t t = 0; t < kRows; ++t) {
                        if (t < rows) {
                            out[(size_t)t * p.N + column] = static_cast<OutT>(acc[t]);
                        }
                    }
                }
                continue;
            }
            // The sums of all parts.  Every CTA of the cluster has multiplied its last block: the rings are idle.
            const uint32_t shift = __ffs(kBlockFewColumns / p.parts) - 1;  // of a part's columns
            cluster_sync_all();
            if (lane == 0 && (!alive || *large != 0u)) {
                for (uint32_t d = 0; d < p.parts; ++d) {
                    st_shared_cluster_u32(map_to_cta(smem_u32(smem) + (alive ? S::kOffLarge : S::kOffDead), d), 1u);
                }
            }
            __syncwarp();
            if (alive) {
                const uint32_t to = column >> shift, line = (part << shift) + (column - (to << shift));
                const uint32_t at = map_to_cta(smem_u32(smem) + line * (S::kPitch * 4u), to);
#pragma unroll
                for (uint32_t t = 0; t < kRows; t += 4) {
                    if (t < rows) {
                        st_shared_cluster_v4(at + t * 4u, __float_as_uint(acc[t]), __float_as_uint(acc[t + 1]), __float_as_uint(acc[t + 2]),
                                             __float_as_uint(acc[t + 3]));
                    }
                }
            }
            __syncwarp();
            cluster_sync_all();
            if (*reinterpret_cast<volatile uint32_t*>(dead) != 0u) {
                alive = false;
            }
            for (uint32_t i = threadIdx.x; alive && i < rows << shift; i += 128u) {
                const uint32_t t = i >> shift, c = i - (t << shift), n = (part << shift) + c;
                const float* at = reinterpret_cast<const float*>(smem) + c * S::kPitch + t;
                float sum = *at;
                for (uint32_t src = 1; src < p.parts; ++src) {
                    sum += at[(src << shift) * S::kPitch];
                }
                if (n0 + n < p.N) {
                    out[(size_t)t * p.N + n] = static_cast<OutT>(sum);
                }
            }
        }
    }
    if (warp >= 4 && p.parts > 1u && first_unit < num_units) {
        __syncwarp();
        cluster_sync_all();  // the two meetings of the promotion warps
        cluster_sync_all();
    }

    tcgen05_fence_before();
    if (__syncthreads_or(alive ? 0 : 1)) {
        drain_after_abort(p.status);
    } else if (__builtin_expect(*large != 0u, 0)) {
        block_few_again<kRows, OutT>(p, tiles, reinterpret_cast<float*>(smem));
    }
    if (warp == 6) {
        tcgen05_fence_after();
        tmem_dealloc(tmem_base, S::kTmemCols);
    }
}

}  // namespace catccos
