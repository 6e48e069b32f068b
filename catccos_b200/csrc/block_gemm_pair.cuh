// The products of block_gemm.cuh on CTA pairs (clusters of two SMs, tcgen05 cta_group::2), for calls that fill the GPU with 256 x 128
// tiles.
//
// CTA r of a pair loads rows [128 r, +128) of A and columns [64 r, +64) of B with plain TMA; the leader issues the products of both,
// and each CTA has the results for its own 128 rows and all 128 columns in its own tensor memory.
//
// A block's way from the tensor core through the promotion and back is far longer than its products (256 cycles at best): some 500
// cycles until a finished product is seen, 400 to load and add the tile, 300 until the issuer knows that it is free again.  So four
// tiles take turns (all that tensor memory holds), a tile goes back as soon as its last columns are in registers, and no warp that
// promotes looks at a barrier in shared memory, which takes some 150 cycles even if there is nothing to wait for: another warp does,
// and named barriers pass it on.  (With each promotion warp looking for itself 8192 x 2304 x 7168 takes 171 us.)
//
// What bounds it, at 8192 x 2304 x 7168: 153 us back to back on two sets of operands (1.77 PFLOP/s; 177 in a caller's loop with new operands,
// 1.53), 0.34 us a block of K.  With the promotion left out it is 127, with its loads alone 135: operands come at 24 KB a block and SM, 85 GB/s, about what a K tile of 192 rows takes in mx_gemm_pair.cuh.  256 x
// 256 tiles read a third less of A and B, but have room for two tiles only, and came to 153; at 3001 x 7168 x 2304 to 84 against 78.
// Sixteen promotion warps of 32 columns: 160.  By column (the scales of 128 columns in shared memory, one more product a value): 7168
// x 2304 x 4096 127 to 134 us, bound by the promotion.  (All figures back to back.)
//
//   full[s], tmem_empty[b]    live in the leader; both CTAs' TMA bytes, and the other CTA's word that it has read a tile, go there
//   empty[s], tmem_full[b]    live in each CTA; the leader's tcgen05.commit arrives on both copies
//   tile_read[b]              lives in each CTA: its promotion warps have read a tile
//   scale_full[i], scale_empty[i]   live in each CTA: the factors of its rows (and, by column, of the columns) for a group of four
//                             blocks of K (every unit begins with a group of its own)
//   named barriers 1 + b      tile b may be read; 5: the first group's factors are there (the warp that arrives on them always does, and nothing
//                             else waits on one: their waits have no limit)
//
// A role takes 300 to 600 cycles for a block whatever its size (a look at a barrier, then instructions of one lane), hence so many of
// them.  448 threads: warps 0-7 promotion and output (warp w: lane quarter w % 4, columns 64 (w / 4)), 8 and 9 TMA for A and B, 10
// and 11 MMA, each every second block (in the other CTA they pass on that tiles have been read), 12 tells the promotion of tiles and factors, 13 makes the factors, a row's scale times the columns'.
#pragma once

#include "block_gemm.cuh"
#include "mx_gemm_pair.cuh"

namespace catccos {

constexpr uint32_t kBlockPairThreads = 448;
constexpr uint32_t kBlockPairPromoters = 8;  // warps

template <typename OutT>
struct BlockPairSmem {
    static constexpr uint32_t kStages = sizeof(OutT) == 4 ? 5 : 6;
    static constexpr uint32_t kTiles = 4;           // in tensor memory
    static constexpr uint32_t kABytes = 128 * 128;  // this CTA's rows
    static constexpr uint32_t kBBytes = 64 * 128;   // this CTA's columns
    static constexpr uint32_t kOutBytes = 32 * 64 * sizeof(OutT);  // of a warp
    static constexpr uint32_t kScaleSlots = 4;                     // groups of four blocks
    static constexpr uint32_t kOffA = 0;
    static constexpr uint32_t kOffB = kOffA + kStages * kABytes;
    static constexpr uint32_t kOffOut = kOffB + kStages * kBBytes;
    static constexpr uint32_t kOffFactor = kOffOut + kBlockPairPromoters * kOutBytes;  // [128 rows][4 blocks] a slot
    static constexpr uint32_t kOffScale = kOffFactor + kScaleSlots * 128 * 16;         // by column: [4 blocks][128 columns] a slot; else g as the factors
    static constexpr uint32_t kOffBar = kOffScale + kScaleSlots * kBlockPairN * 16;
    static constexpr uint32_t kNumBars = 2 * kStages + 3 * kTiles + 2 * kScaleSlots;
    static constexpr uint32_t kOffTmemPtr = kOffBar + kNumBars * 8;
    static constexpr uint32_t kOffDead = kOffTmemPtr + 4;   // the step (counted from 1) whose wait has given up; ~0: before the first
    static constexpr uint32_t kOffLeave = kOffTmemPtr + 16;               // [tiles]: the step (from 1) with which the promotion leaves its loop
    static constexpr uint32_t kOffApart = kOffLeave + kTiles * 4;         // [slots] words: the group's products of scales leave fp32's range
    static constexpr uint32_t kOffTiles = kOffApart + kScaleSlots * 4;
    static constexpr uint32_t dynamic_bytes(uint32_t experts) { return kOffTiles + (3u * experts + 1u) * 4u + 1024u; }
    static_assert(kScaleSlots * 128 * 16 <= kOffBar - kOffScale, "a marked group's g lie where the columns' scales would");
};
static_assert(BlockPairSmem<float>::dynamic_bytes(kGroupedMaxExperts) <= 232448 && BlockPairSmem<__half>::dynamic_bytes(kGroupedMaxExperts) <= 232448,
              "one CTA's shared memory");

// One block of K: four products (K = 32) into the tile at tmem_d, then arrivals on both CTAs' `done` and `empty` when
// they are finished.  Called by a converged warp, of which one lane issues everything: a branch on the lane around each instruction would
// cost more than the instruction, and the next block's way through the promotion waits for this one.
__device__ __forceinline__ void umma_f8_pair_block(uint32_t tmem_d, uint32_t a_lo, uint32_t a_hi, uint32_t a_step, uint32_t b_lo, uint32_t b_hi,
                                                   uint32_t b_step, uint32_t idesc, uint64_t* done, uint64_t* empty)
{
    asm volatile(
        "{\n\t"
        ".reg .pred one, add;\n\t"
        ".reg .b64 da, db;\n\t"
        ".reg .b32 a, b;\n\t"
        ".reg .b16 both;\n\t"
        "mov.b16 both, 3;\n\t"
        "elect.sync _|one, 0xffffffff;\n\t"
        "setp.ne.b32 add, 0, 0;\n\t"
        "mov.b64 da, {%1, %2};\n\t"
        "mov.b64 db, {%4, %5};\n\t"
        "@one tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], da, db, %7, add;\n\t"
        "setp.eq.b32 add, 0, 0;\n\t"
        "add.u32 a, %1, %3;\n\t"
        "add.u32 b, %4, %6;\n\t"
        "mov.b64 da, {a, %2};\n\t"
        "mov.b64 db, {b, %5};\n\t"
        "@one tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], da, db, %7, add;\n\t"
        "add.u32 a, a, %3;\n\t"
        "add.u32 b, b, %6;\n\t"
        "mov.b64 da, {a, %2};\n\t"
        "mov.b64 db, {b, %5};\n\t"
        "@one tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], da, db, %7, add;\n\t"
        "add.u32 a, a, %3;\n\t"
        "add.u32 b, b, %6;\n\t"
        "mov.b64 da, {a, %2};\n\t"
        "mov.b64 db, {b, %5};\n\t"
        "@one tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], da, db, %7, add;\n\t"
        "@one tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%8], both;\n\t"
        "@one tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%9], both;\n\t"
        "}"
        ::"r"(tmem_d), "r"(a_lo), "r"(a_hi), "r"(a_step), "r"(b_lo), "r"(b_hi), "r"(b_step), "r"(idesc), "r"(smem_u32(done)), "r"(smem_u32(empty))
        : "memory");
}

// A pair's tile load with the announcement of its bytes, by one lane of a converged warp (as umma_f8_pair_block).
__device__ __forceinline__ void tma_expect_and_load_2d_pair(void* smem_dst, const void* tmap, uint32_t bar_cluster_addr, uint32_t bytes, uint32_t x, uint32_t y)
{
    asm volatile(
        "{\n\t"
        ".reg .pred one;\n\t"
        "elect.sync _|one, 0xffffffff;\n\t"
        "@one mbarrier.arrive.expect_tx.shared::cluster.b64 _, [%2], %5;\n\t"
        "@one cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];\n\t"
        "}"
        ::"r"(smem_u32(smem_dst)), "l"(tmap), "r"(bar_cluster_addr), "r"(x), "r"(y), "r"(bytes)
        : "memory");
}

__device__ __forceinline__ void tma_expect_and_load_3d_pair(void* smem_dst, const void* tmap, uint32_t bar_cluster_addr, uint32_t bytes, uint32_t x, uint32_t y,
                                                       uint32_t z)
{
    asm volatile(
        "{\n\t"
        ".reg .pred one;\n\t"
        "elect.sync _|one, 0xffffffff;\n\t"
        "@one mbarrier.arrive.expect_tx.shared::cluster.b64 _, [%2], %6;\n\t"
        "@one cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];\n\t"
        "}"
        ::"r"(smem_u32(smem_dst)), "l"(tmap), "r"(bar_cluster_addr), "r"(x), "r"(y), "r"(z), "r"(bytes)
        : "memory");
}

// By column: whether some product of a row's and a column's scale, of the whole warp's, may not stand for them.  Looks at the largest ones by
// their bits, and only when these say so at the finite ones alone.
__device__ __forceinline__ bool scales_apart(const float (&rows)[4][4], const float4 (&columns)[4])
{
    auto outside = [&](bool all) {
        uint32_t most[2] = {0u, 0u};  // of the rows' scales, of the columns'
        auto see = [&](uint32_t side, float s) {
            most[side] = max(most[side], all ? __float_as_uint(s) : (is_finite(s) ? __float_as_uint(s) & 0x7FFFFFFFu : 0u));
        };
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) {
            see(0, rows[i][0]), see(0, rows[i][1]), see(0, rows[i][2]), see(0, rows[i][3]);
            see(1, columns[i].x), see(1, columns[i].y), see(1, columns[i].z), see(1, columns[i].w);
        }
        const float top = __uint_as_float(__reduce_max_sync(0xFFFFFFFFu, most[0])) * kHeld * __uint_as_float(__reduce_max_sync(0xFFFFFFFFu, most[1]));
        return __float_as_uint(top) >= kFactorLimit;
    };
    return __builtin_expect(outside(true), 0) && outside(false);
}

constexpr uint32_t kBlockPairJoined = 32 * (kBlockPairPromoters + 1);  // threads of a named barrier
constexpr uint32_t kBlockPairFirst = 5;                                // the named barrier of the first factors

__device__ __forceinline__ void named_sync(uint32_t id)
{
    asm volatile("barrier.cta.sync %0, %1;" ::"r"(id), "n"(kBlockPairJoined) : "memory");
}

__device__ __forceinline__ void named_arrive(uint32_t id)
{
    asm volatile("barrier.cta.arrive %0, %1;" ::"r"(id), "n"(kBlockPairJoined) : "memory");
}

template <typename OutT, bool kByColumn>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kBlockPairThreads, 1)
block_gemm_pair_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_a32,
                       const __grid_constant__ CUtensorMap tmap_b, const __grid_constant__ CUtensorMap tmap_c,
                       const __grid_constant__ BlockGemmParams p)
{
    using S = BlockPairSmem<OutT>;
    constexpr uint32_t kStages = S::kStages, kCols = 64;  // columns of a promotion warp
    constexpr bool kLater = !kByColumn;

    grid_dep_launch();
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + S::kOffBar);
    uint64_t* empty = full + kStages;
    uint64_t* tmem_full = empty + kStages;
    uint64_t* tmem_empty = tmem_full + S::kTiles;
    uint64_t* tile_read = tmem_empty + S::kTiles;
    uint64_t* scale_full = tile_read + S::kTiles;
    uint64_t* scale_empty = scale_full + S::kScaleSlots;
    uint32_t* tmem_ptr_smem = reinterpret_cast<uint32_t*>(smem + S::kOffTmemPtr);
    volatile uint32_t* dead = reinterpret_cast<volatile uint32_t*>(smem + S::kOffDead);
    volatile uint32_t* leave = reinterpret_cast<volatile uint32_t*>(smem + S::kOffLeave);
    volatile uint32_t* apart_of = reinterpret_cast<volatile uint32_t*>(smem + S::kOffApart);
    uint32_t* tiles = reinterpret_cast<uint32_t*>(smem + S::kOffTiles);
    uint32_t* row_begin = tiles + p.experts + 1u;
    uint32_t* row_end = row_begin + p.experts;

    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
    const uint32_t cta = cluster_ctarank();  // 0 = leader
    const uint32_t pair = blockIdx.x >> 1, num_pairs = gridDim.x >> 1;
    const uint32_t n_tiles = (p.N + kBlockPairN - 1) / kBlockPairN;
    const uint32_t k_blocks = (p.K + 127u) / 128u;
    const uint64_t bar_ns = p.bar_timeout_ns;

    if (threadIdx.x == 32 * kBlockPairPromoters) {
        for (uint32_t s = 0; s < kStages; ++s) {
            mbar_init(&full[s], 4);  // both CTAs' producers (expect_tx)
            mbar_init(&empty[s], 1);
        }
        for (uint32_t b = 0; b < S::kTiles; ++b) {
            mbar_init(&tmem_full[b], 1);
            mbar_init(&tmem_empty[b], 1);  // warps 10 and 11 of the other CTA
            mbar_init(&tile_read[b], kBlockPairPromoters);
            leave[b] = 0u;
        }
        for (uint32_t i = 0; i < S::kScaleSlots; ++i) {
            mbar_init(&scale_full[i], kByColumn ? 2 : 1);  // the rows' factors (and the columns' bytes)
            mbar_init(&scale_empty[i], kBlockPairPromoters);
        }
        *dead = 0u;
        mbar_fence_init();
        tma_prefetch_desc(&tmap_a);
        tma_prefetch_desc(&tmap_a32);
        tma_prefetch_desc(&tmap_b);
        tma_prefetch_desc(&tmap_c);
    }
    if (warp == 10) {
        tmem_alloc_pair(tmem_ptr_smem, 512);
        tmem_relinquish_pair();
    }
    grid_dep_wait();
    if (warp == 0) {
        count_block_tiles(p, kBlockPairM, tiles, row_begin, row_end, lane);
    }
    tcgen05_fence_before();
    __syncthreads();
    cluster_sync_all();  // both CTAs' barriers exist before anybody arrives on the other's
    tcgen05_fence_after();
    const uint32_t tmem_base = *tmem_ptr_smem;
    const uint32_t num_units = tiles[p.experts] * n_tiles;
    const uint32_t my_units = num_units > pair ? (num_units - pair + num_pairs - 1u) / num_pairs : 0u;
    const uint32_t steps = my_units * k_blocks;  // blocks of K, over all units of this pair
    bool alive = true;  // false once a wait of this role has given up

    struct Unit {
        uint32_t e, m0, end, n0;  // expert; first row of the pair's tile, end of the expert's rows; first column
    };
    GroupedWalk own_walk;
    auto find = [&](GroupedWalk& walk, uint32_t unit) {
        const TileCoord tc = walk.seek(tiles, n_tiles, unit);
        return Unit{walk.e, row_begin[walk.e] + tc.m_tile * kBlockPairM, row_end[walk.e], tc.n_tile * kBlockPairN};
    };
    auto unit_at = [&](uint32_t unit) { return find(own_walk, unit); };

    if (warp == 8 || warp == 9) {
        // ------------------------------- TMA producers (both CTAs) ------------------------
        const bool rows = warp == 8;
        uint32_t it = 0;
        for (uint32_t unit = pair; alive && unit < num_units; unit += num_pairs) {
            const Unit u = unit_at(unit);
            const uint32_t m0 = u.m0 + cta * 128u;
            const uint32_t boxes = m0 < u.end ? (min(u.end - m0, 128u) + 31u) / 32u : 0u;  // of 32 rows
            const uint32_t n = u.n0 + cta * 64u;
            for (uint32_t kb = 0; alive && kb < k_blocks; ++kb, ++it) {
                const uint32_t s = it % kStages, k = kb * 128u;
                const uint32_t leader_bar = map_to_cta(smem_u32(&full[s]), 0);
                alive = mbar_wait_soon(&empty[s], ((it / kStages) & 1u) ^ 1u, p.status, 500, s, bar_ns);
                if (!alive) {
                    break;
                }
                if (!rows) {
                    tma_expect_and_load_3d_pair(smem + S::kOffB + s * S::kBBytes, &tmap_b, leader_bar, S::kBBytes, p.b_rows ? k : n, p.b_rows ? n : k, u.e);
                } else if (boxes == 4u || (p.a_cols && boxes)) {
                    tma_expect_and_load_2d_pair(smem + S::kOffA + s * S::kABytes, &tmap_a, leader_bar, S::kABytes, p.a_cols ? m0 : k, p.a_cols ? k : m0);
                } else {
                    if (elect_one()) {
                        mbar_arrive_expect_tx_cluster(leader_bar, boxes * (32u * 128u));
                        for (uint32_t i = 0; i < boxes; ++i) {
                            tma_load_2d_pair(smem + S::kOffA + s * S::kABytes + i * (32u * 128u), &tmap_a32, leader_bar, (int32_t)k, (int32_t)(m0 + i * 32u));
                        }
                    }
                    __syncwarp();
                }
            }
        }
    } else if (warp == 13) {
        // ------------------------------- factors (both CTAs, own 128 rows) ----------------
        uint32_t group = 0;
        for (uint32_t unit = pair; alive && unit < num_units; unit += num_pairs) {
            const Unit u = unit_at(unit);
            const uint32_t row = u.m0 + cta * 128u + lane;
            const float* b_scales = p.b_scales + u.e * p.b_scale_matrix + (u.n0 / 128u) * p.b_scale_col;
            for (uint32_t kb = 0; alive && kb < k_blocks; kb += 4u, ++group) {
                float a[4][4], b[4] = {1.0f, 1.0f, 1.0f, 1.0f};  // of four rows (and the columns) four blocks
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i) {
                    load_scales(p.a_scales + min(row + 32u * i, u.end - 1u) * p.a_scale_row, p.a_scale_block, kb, k_blocks, a[i]);
                }
                float4 columns[4];  // by column: of four of them
                if (!kByColumn) {
                    load_scales(b_scales, p.b_scale_block, kb, k_blocks, b);
                } else {
#pragma unroll
                    for (uint32_t j = 0; j < 4; ++j) {
                        const float* at = p.b_scales + (kb + j) * p.b_scale_block + u.n0 + 4u * lane;
                        columns[j] = kb + j < k_blocks && u.n0 + 4u * lane < p.N ? __ldcg(reinterpret_cast<const float4*>(at)) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    }
                }
                const uint32_t slot = group % S::kScaleSlots;
                alive = mbar_wait_soon(&scale_empty[slot], ((group / S::kScaleSlots) & 1u) ^ 1u, p.status, 505, slot, bar_ns);
                if (!alive) {
                    break;
                }
                if (kByColumn && elect_one()) {
                    const uint32_t bytes = min(p.N - u.n0, kBlockPairN) * 4u, blocks = min(k_blocks - kb, 4u);
                    mbar_arrive_expect_tx(&scale_full[slot], blocks * bytes);
                    for (uint32_t j = 0; j < blocks; ++j) {
                        bulk_load(smem + S::kOffScale + (slot * 4u + j) * (kBlockPairN * 4u), p.b_scales + (kb + j) * p.b_scale_block + u.n0, bytes,
                                  &scale_full[slot]);
                    }
                }
                __syncwarp();
                // whether some product may not stand for its two scales; by column: of the group's largest ones
                float f[4][4];
                bool apart;
                if (kByColumn) {
                    apart = scales_apart(a, columns);
#pragma unroll
                    for (uint32_t i = 0; i < 16; ++i) {
                        f[i / 4][i % 4] = a[i / 4][i % 4] * kHeld;
                    }
                } else {
                    uint32_t most = 0;
#pragma unroll
                    for (uint32_t j = 0; j < 4; ++j) {
                        const float held = b[j] * kHeld;
#pragma unroll
                        for (uint32_t i = 0; i < 4; ++i) {
                            f[i][j] = a[i][j] * held;
                            most = max(most, __float_as_uint(f[i][j]));
                        }
                    }
                    apart = __any_sync(0xFFFFFFFFu, most >= kFactorLimit);
                    if (__builtin_expect(apart, 0)) {
                        bool odd = false;
#pragma unroll
                        for (uint32_t i = 0; i < 16; ++i) {
                            odd = odd || needs_both_scales(a[i / 4][i % 4], b[i % 4], f[i / 4][i % 4]);
                        }
                        apart = __any_sync(0xFFFFFFFFu, odd);
                    }
                }
                if (__builtin_expect(apart, 0)) {
                    float4* power = reinterpret_cast<float4*>(smem + S::kOffScale) + slot * 128u + lane;
#pragma unroll
                    for (uint32_t i = 0; i < 4; ++i) {
                        float g[4];
#pragma unroll
                        for (uint32_t j = 0; j < 4; ++j) {
                            f[i][j] = kByColumn ? a[i][j] : wide_factor(a[i][j], b[j], g[j]);
                        }
                        if (!kByColumn) {
                            power[32u * i] = make_float4(g[0], g[1], g[2], g[3]);
                        }
                    }
                }
                float4* factor = reinterpret_cast<float4*>(smem + S::kOffFactor) + slot * 128u + lane;
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i) {
                    factor[32u * i] = make_float4(f[i][0], f[i][1], f[i][2], f[i][3]);
                }
                if (lane == 0) {
                    apart_of[slot] = apart ? 1u : 0u;
                }
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(&scale_full[slot]);
                }
            }
        }
    } else if (warp == 10 || warp == 11) {
        // ------------------------------- MMA issuers (leader CTA only) --------------------
        if (cta == 0) {
            const uint32_t idesc0 = make_idesc_f8(kBlockPairM, 0, p.a_fmt, p.b_fmt, p.a_cols != 0u, p.b_rows == 0u);
            const uint64_t desc_k = make_smem_desc(0, 16, 1024, 2);
            const uint64_t desc_a = p.a_cols ? make_smem_desc(0, 16384, 1024, 2) : desc_k, desc_b = p.b_rows ? desc_k : make_smem_desc(0, 16384, 512, 4);
            const uint32_t hi_a = (uint32_t)(desc_a >> 32), hi_b = (uint32_t)(desc_b >> 32);
            const uint32_t a_lo0 = (uint32_t)desc_a | (smem_u32(smem + S::kOffA) >> 4);
            const uint32_t b_lo0 = (uint32_t)desc_b | (smem_u32(smem + S::kOffB) >> 4);
            const uint32_t step_a = (p.a_cols ? 4096u : 32u) >> 4, step_b = (p.b_rows ? 32u : 2048u) >> 4;
            uint32_t unit = pair, i = warp - 10u;  // of step `it`: its unit, the how manieth there
            uint32_t idesc = 0, of_unit = 0xFFFFFFFFu;
            for (uint32_t it = warp - 10u; it < steps; it += 2u, i += 2u) {
                while (i >= k_blocks) {
                    i -= k_blocks;
                    unit += num_pairs;
                }
                if (unit != of_unit) {
                    // of a ragged last column of tiles as much is multiplied as the leader's columns need: the other CTA's are fewer
                    const uint32_t columns = (min(p.N - unit_at(unit).n0, 64u) + 15u) / 16u * 16u;
                    idesc = idesc0 | ((2u * columns >> 3) << 17);
                    of_unit = unit;
                }
                const uint32_t b = it & 3u, s = it % kStages;
                const uint32_t free_ph = ((it >> 2) & 1u) ^ 1u;
                alive = mbar_wait_both(&tile_read[b], free_ph, &tmem_empty[b], free_ph, p.status, 501, b, bar_ns) &&
                        mbar_wait_soon(&full[s], (it / kStages) & 1u, p.status, 503, s, bar_ns);
                if (!alive) {
                    break;  // nothing is issued, and no tile reported, after a wait has given up
                }
                tcgen05_fence_after();
                umma_f8_pair_block(tmem_base + b * kBlockPairN, a_lo0 + s * (S::kABytes >> 4), hi_a, step_a, b_lo0 + s * (S::kBBytes >> 4), hi_b, step_b,
                                   idesc, &tmem_full[b], &empty[s]);
            }
        } else {
            const uint32_t free_bar = map_to_cta(smem_u32(&tmem_empty[0]), 0);
            for (uint32_t it = warp - 10u; it < steps; it += 2u) {
                const uint32_t b = it & 3u;
                alive = mbar_wait_soon(&tile_read[b], (it >> 2) & 1u, p.status, 502, b, bar_ns);
                if (!alive) {
                    break;
                }
                if (lane == 0) {
                    mbar_arrive_cluster(free_bar + b * 8u);
                }
                __syncwarp();
            }
        }
    } else if (warp == 12) {
        // ------------------------------- tells of tiles and factors -----------------------
        // It is never two turns ahead on a named barrier: tile b is filled again after all have read it.  With the last block of a group it
        // waits for the next one's factors as well: when that is marked, or when a wait gives up, the promotion leaves its loop with
        // this step.
        uint32_t i = 0, group = 0;
        if (steps != 0u) {
            alive = mbar_wait_soon(&scale_full[0], 0u, p.status, 507, 0, bar_ns);
            if (!alive && lane == 0) {
                *dead = 0xFFFFFFFFu;
            }
            __syncwarp();
            named_arrive(kBlockPairFirst);
        }
        for (uint32_t it = 0; alive && it < steps; ++it) {
            const uint32_t b = it & 3u, next = (group + 1u) % S::kScaleSlots;
            const bool group_end = (i & 3u) == 3u || i + 1u == k_blocks;
            uint32_t apart = 0;
            if (group_end && it + 1u < steps) {
                alive = mbar_wait_both(&tmem_full[b], (it >> 2) & 1u, &scale_full[next], ((group + 1u) / S::kScaleSlots) & 1u, p.status, 506, b, bar_ns);
                apart = apart_of[next];
            } else {
                alive = mbar_wait_soon(&tmem_full[b], (it >> 2) & 1u, p.status, 506, b, bar_ns);
            }
            group += group_end ? 1u : 0u;
            i = i + 1u == k_blocks ? 0u : i + 1u;
            if ((!alive || apart != 0u) && lane == 0) {
                if (!alive) {
                    *dead = it + 1u;
                }
                leave[b] = it + 1u;
            }
            __syncwarp();
            tcgen05_fence_after();
            tcgen05_fence_before();
            named_arrive(1u + b);
        }
    } else {
        // ------------------------------- promotion and output (both CTAs, own 128 rows) ---
        const uint32_t q = warp & 3u, col = (warp >> 2) * kCols;
        const uint32_t tmem = tmem_base + ((q * 32u) << 16) + col;
        const uint32_t factors = smem_u32(smem + S::kOffFactor) + (q * 32u + lane) * 16u;
        const uint32_t scales = smem_u32(smem + S::kOffScale) + col * 4u;
        uint8_t* out = smem + S::kOffOut + warp * S::kOutBytes;
        uint32_t it = 0, group = 0;
        bool apart = false;  // the group that comes next is marked
        if (steps != 0u) {
            named_sync(kBlockPairFirst);
            alive = *dead != 0xFFFFFFFFu;
            apart = apart_of[0] != 0u;
        }
        for (uint32_t unit = pair; alive && unit < num_units; unit += num_pairs) {
            const Unit u = unit_at(unit);
            const uint32_t row0 = u.m0 + cta * 128u + q * 32u, col0 = u.n0 + col;
            const bool live = row0 < u.end && col0 < p.N;  // else there is nothing to fetch
            float acc[kCols] = {};
            // Sixteen columns are added while the next are on their way, a step's last while the next step's first are (by column, which
            // has no registers left for that, at once: 143 -> 132 us); a tile goes back when its last are in registers.
            float v[2][16], f = 0.0f;
            uint32_t scale = 0;
            uint32_t i = 0;
            bool left = false;
            for (; !apart && i < k_blocks; ++i, ++it) {
                const uint32_t b = it & 3u, j = i & 3u;
                named_sync(1u + b);
                tcgen05_fence_after();
                const uint32_t leave_step = leave[b];
                if (live) {
                    const uint32_t tile = tmem + b * kBlockPairN;
                    tmem_ld_16(tile, v[0]);
                    float f_next;
                    asm volatile("ld.shared.f32 %0, [%1];" : "=f"(f_next) : "r"(factors + (group % S::kScaleSlots * 128u) * 16u + j * 4u));
                    if (kLater && i != 0u) {
                        add_scaled<kByColumn>(&acc[48], v[1], f, scale + 192u);
                    }
                    f = f_next;
                    scale = scales + (group % S::kScaleSlots * 4u + j) * (kBlockPairN * 4u);
                    tmem_ld_fence(v[0]);
#pragma unroll
                    for (uint32_t c = 0; c < 3; ++c) {
                        tmem_ld_16(tile + 16u * c + 16u, v[(c + 1) & 1]);
                        add_scaled<kByColumn>(&acc[16 * c], v[c & 1], f, scale + 64u * c);
                        tmem_ld_fence(v[(c + 1) & 1]);
                    }
                }
                tcgen05_fence_before();
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(&tile_read[b]);
                    if (j == 0u && group != 0u) {
                        mbar_arrive(&scale_empty[(group - 1u) % S::kScaleSlots]);  // what it had has been added
                    }
                }
                if (!kLater && live) {
                    add_scaled<kByColumn>(&acc[48], v[1], f, scale + 192u);
                }
                if (leave_step == it + 1u) {
                    left = true;
                    break;
                }
                group += j == 3u || i + 1u == k_blocks ? 1u : 0u;
            }
            if (kLater && live && !apart) {
                add_scaled<kByColumn>(&acc[48], v[1], f, scale + 192u);
            }
            if (left) {
                alive = *dead != it + 1u;  // a tile that never filled is not written out
                apart = true;
                ++group, ++i, ++it;
            }
            float back = 1.0f / kHeld;
            if (apart) {
                scale_sums(acc, back);
                back = 1.0f;
            }
            for (uint32_t marked = 0; alive && i < k_blocks; ++i, ++it) {  // from a marked group to the end of the unit
                const uint32_t b = it & 3u, j = i & 3u, slot = group % S::kScaleSlots;
                named_sync(1u + b);
                tcgen05_fence_after();
                const uint32_t leave_step = leave[b];
                marked = j == 0u ? apart_of[slot] : marked;
                const uint32_t tile = tmem + b * kBlockPairN, of_row = (slot * 128u) * 16u + j * 4u;
                scale = scales + (slot * 4u + j) * (kBlockPairN * 4u);
                float g = 1.0f / kHeld;
                auto add = [&](uint32_t c) {
                    float(&x)[16] = v[c & 1];
                    if (kByColumn) {
                        add_scaled_apart(&acc[16 * c], x, f, scale + 64u * c);
                    } else {
                        scale_sums(x, g);
                        add_scaled<false>(&acc[16 * c], x, f, 0u);
                    }
                };
                if (live) {
                    tmem_ld_16(tile, v[0]);
                    f = ld_shared_f32(factors + of_row);
                    if (kByColumn) {
                        f = marked ? f : f * g;
                    } else if (marked) {
                        g = ld_shared_f32(factors + S::kOffScale - S::kOffFactor + of_row);
                    }
                    tmem_ld_fence(v[0]);
#pragma unroll
                    for (uint32_t c = 0; c < 3; ++c) {
                        tmem_ld_16(tile + 16u * c + 16u, v[(c + 1) & 1]);
                        add(c);
                        tmem_ld_fence(v[(c + 1) & 1]);
                    }
                }
                tcgen05_fence_before();
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(&tile_read[b]);
                    if (j == 0u && group != 0u) {
                        mbar_arrive(&scale_empty[(group - 1u) % S::kScaleSlots]);
                    }
                }
                if (live) {
                    add(3);
                }
                group += j == 3u || i + 1u == k_blocks ? 1u : 0u;
                apart = leave_step == it + 1u;
                if (apart && *dead == it + 1u) {
                    alive = false;
                    break;
                }
            }
            if (live && alive) {
                scale_sums(acc, back);
                if (row0 + 32u <= u.end || p.offsets == nullptr) {
                    // twice 32 rows of 32 columns, in the order that TMA reads with its swizzle; what lies outside the matrix is not written
                    if (lane == 0) {
                        bulk_store_wait_read();
                    }
                    __syncwarp();
                    stage_out<OutT>(out, lane, &acc[0]);
                    stage_out<OutT>(out + S::kOutBytes / 2u, lane, &acc[32]);
                    fence_proxy_async_shared();
                    __syncwarp();
                    if (lane == 0) {
                        tma_store_2d(&tmap_c, out, (int32_t)col0, (int32_t)row0);
                        if (col0 + 32u < p.N) {
                            tma_store_2d(&tmap_c, out + S::kOutBytes / 2u, (int32_t)(col0 + 32u), (int32_t)row0);
                        }
                        bulk_store_commit();
                    }
                } else if (row0 + lane < u.end) {
                    OutT* dst = static_cast<OutT*>(p.c) + (size_t)(row0 + lane) * p.N + col0;
#pragma unroll
                    for (uint32_t c = 0; c < kCols; c += 16) {
                        if (col0 + c < p.N) {
                            store_16(dst + c, &acc[c]);
                        }
                    }
                }
            }
        }
        if (lane == 0) {
            bulk_store_wait_all();
        }
    }

    tcgen05_fence_before();
    if (__syncthreads_or(alive ? 0 : 1)) {
        drain_after_abort(p.status);  // both CTAs stay while loads that report to the other's barriers may be in flight
    }
    cluster_sync_all();  // nobody leaves while the other CTA may still arrive on its barriers
    if (warp == 10) {
        tcgen05_fence_after();
        tmem_dealloc_pair(tmem_base, 512);
    }
}

}  // namespace catccos
