// Products of 8-bit codes with one fp32 scale for each block of 128, for sm_100a, dense and per expert:
//   C[i, j] = sum over blocks t of K:  sa[i, t] * sb[t, j / 128] * (sum over k in block t of A[i, k] B[k, j])
// (or sb[t, j]: B scaled by column, a weight's gradient).  With offsets [experts + 1] on the device, rows offsets[e] ..
// offsets[e + 1] of A meet expert e's B.
//
// The scales are no powers of two, so the tensor core cannot apply them: every block's products are a tensor-memory tile of
// their own, which the promotion warps read, scale and add to sums in registers while the next block is multiplied into the
// other tile.  128 columns of K are four tcgen05.mma kind::f8f6f4 (K = 32).
//
// Either operand may be stored with K or with its other axis running fastest: both are operand layouts of the tensor core, so
// that x W, dy W^T and x^T dy read the same codes without a transposed copy.  K need not be a multiple of 128: TMA fills the
// last block with zeros.
//
// 320 threads: warps 0-7 promotion and output (warp w: lane quarter w % 4, column half w / 4), warp 8 TMA, warp 9 MMA.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"
#include "mx_gemm_small.cuh"
#include "mx_grouped_gemm.cuh"

namespace catccos {

constexpr uint32_t kBlockGemmThreads = 320;
constexpr uint32_t kBlockGemmM = 128;
constexpr uint32_t kBlockGemmMaxParts = 8;

struct BlockGemmParams {
    const float* a_scales;
    size_t a_scale_row, a_scale_block;                     // floats from one row's (block's) scale to the next
    const float* b_scales;
    size_t b_scale_block, b_scale_col, b_scale_matrix;     // from one block of K, of columns (by column: 1), one expert to the next
    const int32_t* offsets;                                // nullptr: one matrix
    void* c;
    uint32_t rows, experts, N, K;
    uint32_t a_fmt, b_fmt;                                 // 0 = E4M3, 1 = E5M2
    uint32_t a_cols, b_rows;                               // 1: A is stored [K, rows]; B [N, K]
    uint32_t parts;                                        // CTAs of a cluster that share K (a power of two)
    uint32_t stages, a_stage_rows, ring_bytes;             // of block_gemm_kernel's ring (BlockGemmSmem)
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

__device__ __forceinline__ void tma_load_3d(void* smem_dst, const void* tmap, uint64_t* bar, int32_t x, int32_t y, int32_t z)
{
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
        ::"r"(smem_u32(smem_dst)), "l"(tmap), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z)
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

// sixteen sums += f * the columns of this lane's row; by column: f * scale[column] * them (scale 16-byte aligned)
template <bool kByColumn>
__device__ __forceinline__ void add_scaled(float* acc, const float (&v)[16], float f, const float* scale)
{
#pragma unroll
    for (uint32_t c = 0; c < 16; c += 4) {
        float4 g = make_float4(f, f, f, f);
        if (kByColumn) {
            const float4 s = *reinterpret_cast<const float4*>(scale + c);
            g = make_float4(f * s.x, f * s.y, f * s.z, f * s.w);
        }
        fma_2(acc[c], acc[c + 1], v[c], v[c + 1], g.x, g.y);
        fma_2(acc[c + 2], acc[c + 3], v[c + 2], v[c + 3], g.z, g.w);
    }
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

// A line's scales of blocks kb .. kb + 3 of K (those behind the last: 0); they are `step` floats apart.
__device__ __forceinline__ void load_scales(const float* line, size_t step, uint32_t kb, uint32_t blocks, float (&v)[4])
{
    const float* at = line + kb * step;
    if (step == 1 && kb + 4u <= blocks && ((uintptr_t)at & 15u) == 0u) {
        const float4 w = __ldcg(reinterpret_cast<const float4*>(at));
        v[0] = w.x, v[1] = w.y, v[2] = w.z, v[3] = w.w;
    } else {
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j) {
            v[j] = kb + j < blocks ? __ldcg(at + j * step) : 0.0f;
        }
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

// Shared memory of block_gemm_kernel.  How many rows of A a stage holds, and with it how many stages there are, is the launch's
// choice: few rows leave more room for B on its way.  (The tensor core reads 128 rows whatever a stage holds; the others' products
// are not looked at.)
template <uint32_t BLOCK_N>
struct BlockGemmSmem {
    static constexpr uint32_t kMaxStages = 8;
    static constexpr uint32_t kBBytes = BLOCK_N * 128;
    static constexpr uint32_t kScaleSlots = 4;                                                  // by column: scales of a block
    static constexpr uint32_t kScaleBytes = kScaleSlots * BLOCK_N * 4;
    static constexpr uint32_t kNumBars = 2 * kMaxStages + 4 + 2 * kScaleSlots;                  // full[], empty[], tmem_full[2], tmem_empty[2], scale_full[], scale_empty[]
    static constexpr uint32_t kRest = kScaleBytes + kNumBars * 8 + 16;                          // behind the ring
    static constexpr uint32_t dynamic_bytes(uint32_t ring, uint32_t experts) { return ring + kRest + (3u * experts + 1u) * 4u + 1024u; }
    static constexpr uint32_t kRing = 106496;  // at most: two CTAs to an SM
    // the parts' sums meet in the ring: [part][128 rows][a part's columns, four more]
    static constexpr uint32_t sum_bytes(uint32_t parts) { return kBlockGemmM * (BLOCK_N + 4u * parts) * 4u; }
};

// K may be cut over the CTAs of a cluster (p.parts: 1, 2, 4 or 8), so that calls of few tiles stream their weights with every SM.
// Their sums meet in distributed shared memory: part d owns BLOCK_N / parts of the columns, the others push theirs into its idle
// ring, and it adds them in ascending order of the parts.  A launch with parts has a cluster for every unit there may be.
template <uint32_t BLOCK_N, typename OutT, bool kByColumn>
__global__ void __launch_bounds__(kBlockGemmThreads, 2)
block_gemm_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_a32,
                  const __grid_constant__ CUtensorMap tmap_b, const __grid_constant__ BlockGemmParams p)
{
    using S = BlockGemmSmem<BLOCK_N>;
    constexpr uint32_t kCols = BLOCK_N / 2;  // of a promotion warp
    constexpr uint32_t kTmemCols = 2 * BLOCK_N;

    grid_dep_launch();
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    const uint32_t stages = p.stages, a_bytes = p.a_stage_rows * 128u;
    uint8_t* smem_b = smem + stages * a_bytes;
    float* scales = reinterpret_cast<float*>(smem + p.ring_bytes);
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + p.ring_bytes + S::kScaleBytes);
    uint64_t* empty = full + S::kMaxStages;
    uint64_t* tmem_full = empty + S::kMaxStages;
    uint64_t* tmem_empty = tmem_full + 2;
    uint64_t* scale_full = tmem_empty + 2;
    uint64_t* scale_empty = scale_full + S::kScaleSlots;
    uint32_t* tmem_ptr_smem = reinterpret_cast<uint32_t*>(scale_empty + S::kScaleSlots);
    uint32_t* dead = tmem_ptr_smem + 1;  // a part of this cluster has given up
    uint32_t* tiles = tmem_ptr_smem + 4;
    uint32_t* row_begin = tiles + p.experts + 1u;
    uint32_t* row_end = row_begin + p.experts;

    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
    const uint32_t n_tiles = (p.N + BLOCK_N - 1) / BLOCK_N;
    const uint32_t k_blocks = (p.K + 127u) / 128u;
    const uint32_t part = blockIdx.x & (p.parts - 1u), first_unit = blockIdx.x / p.parts, stride = gridDim.x / p.parts;
    const uint32_t kb0 = (uint32_t)((uint64_t)part * k_blocks / p.parts), kb1 = (uint32_t)((uint64_t)(part + 1u) * k_blocks / p.parts);
    const uint64_t bar_ns = p.bar_timeout_ns;

    if (threadIdx.x == 256) {
        for (uint32_t s = 0; s < stages; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        for (uint32_t a = 0; a < 2; ++a) {
            mbar_init(&tmem_full[a], 1);
            mbar_init(&tmem_empty[a], 8);
        }
        for (uint32_t i = 0; i < S::kScaleSlots; ++i) {
            mbar_init(&scale_full[i], 1);
            mbar_init(&scale_empty[i], 8);
        }
        *dead = 0u;
        mbar_fence_init();
        tma_prefetch_desc(&tmap_a);
        tma_prefetch_desc(&tmap_a32);
        tma_prefetch_desc(&tmap_b);
    }
    if (warp == 9) {
        tmem_alloc(tmem_ptr_smem, kTmemCols);
        tmem_relinquish();
    }
    grid_dep_wait();
    if (warp == 0) {
        count_block_tiles(p, kBlockGemmM, tiles, row_begin, row_end, lane);
    }
    tcgen05_fence_before();
    __syncthreads();
    tcgen05_fence_after();
    const uint32_t tmem_base = *tmem_ptr_smem;
    const uint32_t num_units = tiles[p.experts] * n_tiles;
    bool alive = true;  // false once a wait of this role has given up
    GroupedWalk walk;

    if (warp == 8) {
        // ------------------------------- TMA producer -------------------------------------
        uint32_t it = 0, s = 0, ph = 1;
        for (uint32_t unit = first_unit; alive && unit < num_units; unit += stride) {
            const TileCoord tc = walk.seek(tiles, n_tiles, unit);
            const uint32_t m0 = row_begin[walk.e] + tc.m_tile * kBlockGemmM, n0 = tc.n_tile * BLOCK_N;
            const uint32_t boxes = (min(row_end[walk.e] - m0, kBlockGemmM) + 31u) / 32u;  // of 32 rows
            const uint32_t scale_bytes = min(p.N - n0, BLOCK_N) * 4u;
            const uint32_t tx_bytes = (p.a_cols ? kBlockGemmM * 128u : boxes * (32u * 128u)) + S::kBBytes;
            for (uint32_t kb = kb0; alive && kb < kb1; ++kb, ++it) {
                alive = mbar_wait_soon(&empty[s], ph, p.status, 400, s, bar_ns);
                if (!alive) {
                    break;
                }
                if (elect_one()) {
                    mbar_arrive_expect_tx(&full[s], tx_bytes);
                    const int32_t k = (int32_t)(kb * 128u);
                    tma_load_3d(smem_b + s * S::kBBytes, &tmap_b, &full[s], p.b_rows ? k : (int32_t)n0, p.b_rows ? (int32_t)n0 : k, (int32_t)walk.e);
                    uint8_t* a = smem + s * a_bytes;
                    if (p.a_cols) {
                        tma_load_2d(a, &tmap_a, &full[s], (int32_t)m0, k);
                    } else if (boxes == 4u) {
                        tma_load_2d(a, &tmap_a, &full[s], k, (int32_t)m0);
                    } else {
                        for (uint32_t i = 0; i < boxes; ++i) {
                            tma_load_2d(a + i * (32u * 128u), &tmap_a32, &full[s], k, (int32_t)(m0 + i * 32u));
                        }
                    }
                }
                __syncwarp();
                if (kByColumn) {
                    const uint32_t slot = it % S::kScaleSlots;
                    alive = mbar_wait_soon(&scale_empty[slot], ((it / S::kScaleSlots) & 1u) ^ 1u, p.status, 405, slot, bar_ns);
                    if (alive && elect_one()) {
                        mbar_arrive_expect_tx(&scale_full[slot], scale_bytes);
                        bulk_load(scales + slot * BLOCK_N, p.b_scales + (size_t)walk.e * p.b_scale_matrix + kb * p.b_scale_block + n0, scale_bytes, &scale_full[slot]);
                    }
                    __syncwarp();
                }
                s = s + 1u == stages ? 0u : s + 1u;
                ph ^= s == 0u ? 1u : 0u;
            }
        }
    } else if (warp == 9) {
        // ------------------------------- MMA issuer ---------------------------------------
        const uint32_t idesc0 = make_idesc_f8(kBlockGemmM, 0, p.a_fmt, p.b_fmt, p.a_cols != 0u, p.b_rows == 0u);
        const uint64_t desc_a = p.a_cols ? make_smem_desc(0, 16384, 1024, 2) : make_smem_desc(0, 16, 1024, 2);
        const uint64_t desc_b = p.b_rows ? make_smem_desc(0, 16, 1024, 2)
                                         : make_smem_desc(0, 16384, 8 * BLOCK_N, BLOCK_N == 64 ? 4 : 2);
        const uint32_t hi_a = (uint32_t)(desc_a >> 32), hi_b = (uint32_t)(desc_b >> 32);
        const uint32_t a_lo0 = (uint32_t)desc_a | (smem_u32(smem) >> 4);
        const uint32_t b_lo0 = (uint32_t)desc_b | (smem_u32(smem_b) >> 4);
        const uint32_t step_a = (p.a_cols ? 32u * 128u : 32u) >> 4, step_b = (p.b_rows ? 32u : 32u * BLOCK_N) >> 4;
        uint32_t it = 0, s = 0, ph = 0;
        for (uint32_t unit = first_unit; alive && unit < num_units; unit += stride) {
            // a ragged last column of tiles is multiplied as wide as it is (a multiple of 16)
            const uint32_t idesc = idesc0 | ((min(p.N - unit % n_tiles * BLOCK_N, BLOCK_N) >> 3) << 17);
            for (uint32_t kb = kb0; kb < kb1; ++kb, ++it) {
                const uint32_t buf = it & 1u;
                alive = mbar_wait_both(&full[s], ph, &tmem_empty[buf], ((it >> 1) & 1u) ^ 1u, p.status, 401, s, bar_ns);
                if (!alive) {
                    break;  // nothing is issued, and no tile reported, after a wait has given up
                }
                tcgen05_fence_after();
                umma_f8_block(tmem_base + buf * BLOCK_N, a_lo0 + s * (a_bytes >> 4), hi_a, step_a, b_lo0 + s * (S::kBBytes >> 4), hi_b, step_b, idesc,
                              &tmem_full[buf], &empty[s]);
                s = s + 1u == stages ? 0u : s + 1u;
                ph ^= s == 0u ? 1u : 0u;
            }
        }
    } else {
        // ------------------------------- promotion and output -----------------------------
        const uint32_t q = warp & 3u, half = warp >> 2;
        const uint32_t tmem = tmem_base + ((q * 32u) << 16) + half * kCols;
        uint32_t it = 0;
        for (uint32_t unit = first_unit; alive && unit < num_units; unit += stride) {
            const TileCoord tc = walk.seek(tiles, n_tiles, unit);
            const uint32_t first = row_begin[walk.e] + tc.m_tile * kBlockGemmM, end = row_end[walk.e];
            const uint32_t row0 = first + q * 32u, row = row0 + lane, n0 = tc.n_tile * BLOCK_N;
            const bool live = row0 < end && n0 + half * kCols < p.N;  // else there is nothing to fetch
            const float* a_line = p.a_scales + min(row, end - 1u) * p.a_scale_row;
            const float* b_line = p.b_scales + walk.e * p.b_scale_matrix + (n0 / 128u) * p.b_scale_col;
            float acc[kCols] = {};
            float a4[4], b4[4];  // scales of four blocks
            auto fetch = [&](uint32_t kb) {
                if (live) {
                    load_scales(a_line, p.a_scale_block, kb, kb1, a4);
                    if (!kByColumn) {
                        load_scales(b_line, p.b_scale_block, kb, kb1, b4);
                    }
                }
            };
            fetch(kb0);
            for (uint32_t kb = kb0; kb < kb1; ++kb, ++it) {
                const uint32_t buf = it & 1u, slot = it % S::kScaleSlots, j = (kb - kb0) & 3u;
                alive = kByColumn ? mbar_wait_both(&tmem_full[buf], (it >> 1) & 1u, &scale_full[slot], (it / S::kScaleSlots) & 1u, p.status, 406, buf, bar_ns)
                                  : mbar_wait_soon(&tmem_full[buf], (it >> 1) & 1u, p.status, 406, buf, bar_ns);
                if (!alive) {
                    break;  // a tile that never filled is not written out
                }
                tcgen05_fence_after();
                if (live) {
                    auto pick = [&](const float (&v)[4]) { return j == 0u ? v[0] : (j == 1u ? v[1] : (j == 2u ? v[2] : v[3])); };
                    const float f = kByColumn ? pick(a4) : pick(a4) * pick(b4);
                    if (j == 3u) {
                        fetch(kb + 1u);  // the next four, while this block is added
                    }
#pragma unroll
                    for (uint32_t c = 0; c < kCols; c += 16) {
                        float v[16];
                        tmem_ld_16(tmem + buf * BLOCK_N + c, v);
                        tmem_ld_fence(v);
                        add_scaled<kByColumn>(&acc[c], v, f, scales + slot * BLOCK_N + half * kCols + c);
                    }
                }
                tcgen05_fence_before();
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(&tmem_empty[buf]);
                    if (kByColumn) {
                        mbar_arrive(&scale_empty[slot]);
                    }
                }
            }
            if (p.parts == 1u) {
                if (alive && row < end) {
                    OutT* dst = static_cast<OutT*>(p.c) + (size_t)row * p.N + n0 + half * kCols;
#pragma unroll
                    for (uint32_t c = 0; c < kCols; c += 16) {
                        if (n0 + half * kCols + c < p.N) {
                            store_16(dst + c, &acc[c]);
                        }
                    }
                }
                continue;
            }
            // The sums of all parts.  Every CTA of the cluster has multiplied its last block: the rings are idle.
            const uint32_t cols = BLOCK_N / p.parts, shift = __ffs(cols) - 1, pitch = cols + 4u;  // a part's columns; four more keep lanes off one bank
            cluster_sync_all();
            if (!alive && lane == 0) {
                for (uint32_t d = 0; d < p.parts; ++d) {
                    st_shared_cluster_u32(map_to_cta(smem_u32(dead), d), 1u);
                }
            }
            __syncwarp();
            if (alive && row < end) {
                const uint32_t line = smem_u32(smem) + (part * 128u + q * 32u + lane) * pitch * 4u;
#pragma unroll
                for (uint32_t c = 0; c < kCols; c += 4) {
                    const uint32_t col = half * kCols + c, d = col >> shift;
                    st_shared_cluster_v4(map_to_cta(line + (col - (d << shift)) * 4u, d), __float_as_uint(acc[c]), __float_as_uint(acc[c + 1]),
                                         __float_as_uint(acc[c + 2]), __float_as_uint(acc[c + 3]));
                }
            }
            __syncwarp();
            cluster_sync_all();
            if (*reinterpret_cast<volatile uint32_t*>(dead) != 0u) {
                alive = false;
            }
            const uint32_t rows = min(end - first, kBlockGemmM);
            for (uint32_t i = threadIdx.x; alive && i < rows << (shift - 2u); i += 256u) {
                const uint32_t r = i >> (shift - 2u), c = (i & ((1u << (shift - 2u)) - 1u)) * 4u, n = n0 + part * cols + c;
                const float* at = reinterpret_cast<const float*>(smem) + r * pitch + c;
                float4 sum = *reinterpret_cast<const float4*>(at);
                for (uint32_t src = 1; src < p.parts; ++src) {
                    const float4 x = *reinterpret_cast<const float4*>(at + src * 128u * pitch);
                    sum.x += x.x;
                    sum.y += x.y;
                    sum.z += x.z;
                    sum.w += x.w;
                }
                if (n < p.N) {
                    OutT* dst = static_cast<OutT*>(p.c) + (size_t)(first + r) * p.N + n;
                    if constexpr (sizeof(OutT) == 4) {
                        *reinterpret_cast<float4*>(dst) = sum;
                    } else {
                        *reinterpret_cast<uint2*>(dst) = make_uint2(pack2<OutT>(sum.x, sum.y), pack2<OutT>(sum.z, sum.w));
                    }
                }
            }
        }
    }
    if (warp >= 8 && p.parts > 1u && first_unit < num_units) {
        __syncwarp();
        cluster_sync_all();  // the two meetings of the promotion warps
        cluster_sync_all();
    }

    tcgen05_fence_before();
    if (__syncthreads_or(alive ? 0 : 1)) {
        drain_after_abort(p.status);
    }
    if (warp == 9) {
        tcgen05_fence_after();
        tmem_dealloc(tmem_base, kTmemCols);
    }
}

}  // namespace catccos
