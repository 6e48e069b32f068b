// The products of block_gemm.cuh on CTA pairs (clusters of two SMs, tcgen05 cta_group::2), for calls that fill the GPU with 256 x 256
// tiles.
//
// CTA r of a pair loads rows [128 r, +128) of A and columns [128 r, +128) of B with plain TMA, 32 KB a block of K where a 128 x 256
// tile on one SM takes 48; the leader issues the products of both, and each CTA has the results for its own 128 rows and all 256
// columns in its own tensor memory.
//
// A block's way from the tensor core through the promotion and back takes longer than its products: about 1000 cycles until a
// finished product is seen, 300 for the promotion, 200 back, against 512.  Two tiles of 256 columns (all that tensor memory
// holds) would leave the tensor core waiting half of the time, so the columns are two halves, each with two tiles of its own,
// multiplied one after the other: half h has columns 64 h to 64 h + 63 of each CTA's B.
//
//   full[s], tmem_empty[h][b]   live in the leader; both CTAs' TMA bytes, and a warp of each CTA's promotion, go there
//   empty[s], tmem_full[h][b]   live in each CTA; the leader's tcgen05.commit arrives on both copies
//   scale_full[i], scale_empty[i]  live in each CTA: the factors of its rows (and, by column, of the columns) for one block of K
//
// 640 threads: warps 0-15 promotion and output (warp w: half w / 8, lane quarter w % 4, the half's columns of CTA (w / 4) % 2's B),
// warp 16 TMA, 17 and 18 the products of a half each, 19 the factors: a row's scale times that of each CTA's columns.  The
// promotion warps take registers from the other four.  A look at a barrier in shared memory takes some 150 cycles, so no warp of
// the promotion makes two in a row: of a half's eight warps one waits for the tile, one for the factors of the next block, which all
// fetch ahead, one gives the tile back and one the factors, and named barriers join them.
#pragma once

#include "block_gemm.cuh"
#include "mx_gemm_pair.cuh"

namespace catccos {

constexpr uint32_t kBlockPairThreads = 640;
constexpr uint32_t kBlockPairPromoters = 16;                           // warps
constexpr uint32_t kBlockPairRegs = 96;                                // of a thread at launch
constexpr uint32_t kBlockPairPromoteRegs = 104, kBlockPairOtherRegs = 64;
static_assert(32 * kBlockPairPromoters * kBlockPairPromoteRegs + (kBlockPairThreads - 32 * kBlockPairPromoters) * kBlockPairOtherRegs <=
                  kBlockPairThreads * kBlockPairRegs, "the warpgroups' shares are what the block was launched with");

struct BlockPairSmem {
    static constexpr uint32_t kStages = 6;
    static constexpr uint32_t kABytes = 128 * 128;  // this CTA's rows
    static constexpr uint32_t kBBytes = 128 * 128;  // this CTA's columns
    static constexpr uint32_t kOffA = 0;
    static constexpr uint32_t kOffB = kOffA + kStages * kABytes;
    static constexpr uint32_t kScaleSlots = 8;
    static constexpr uint32_t kOffScale = kOffB + kStages * kBBytes;               // by column: 256 scales a slot
    static constexpr uint32_t kOffFactor = kOffScale + kScaleSlots * kPairBlockN * 4;  // [CTA whose columns][128 rows] a slot
    static constexpr uint32_t kOffBar = kOffFactor + kScaleSlots * 256 * 4;
    static constexpr uint32_t kNumBars = 2 * kStages + 8 + 2 * kScaleSlots;
    static constexpr uint32_t kOffTmemPtr = kOffBar + kNumBars * 8;
    static constexpr uint32_t kOffTiles = kOffTmemPtr + 16;
    static constexpr uint32_t dynamic_bytes(uint32_t experts) { return kOffTiles + (3u * experts + 1u) * 4u + 1024u; }
};
static_assert(BlockPairSmem::dynamic_bytes(kGroupedMaxExperts) <= 232448, "one CTA's shared memory");

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

__device__ __forceinline__ void tma_load_3d_pair(void* smem_dst, const void* tmap, uint32_t bar_cluster_addr, int32_t x, int32_t y, int32_t z)
{
    asm volatile(
        "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
        ::"r"(smem_u32(smem_dst)), "l"(tmap), "r"(bar_cluster_addr), "r"(x), "r"(y), "r"(z)
        : "memory");
}

// Of the eight warps of a CTA that promote a half: true on all if all say so.
__device__ __forceinline__ bool promoters_agree(uint32_t barrier, bool ok)
{
    uint32_t bad;
    asm volatile(
        "{\n\t"
        ".reg .pred p, q;\n\t"
        "setp.ne.u32 p, %1, 0;\n\t"
        "barrier.cta.red.or.pred q, %2, %3, p;\n\t"
        "selp.u32 %0, 1, 0, q;\n\t"
        "}"
        : "=r"(bad)
        : "r"(ok ? 0u : 1u), "r"(barrier), "n"(16 * kBlockPairPromoters)
        : "memory");
    return bad == 0u;
}

template <typename OutT, bool kByColumn>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kBlockPairThreads, 1)
block_gemm_pair_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_a32,
                       const __grid_constant__ CUtensorMap tmap_b, const __grid_constant__ BlockGemmParams p)
{
    using S = BlockPairSmem;
    constexpr uint32_t kStages = S::kStages, kCols = 64;  // columns of a promotion warp

    grid_dep_launch();
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + S::kOffBar);
    uint64_t* empty = full + kStages;
    uint64_t* tmem_full = empty + kStages;
    uint64_t* tmem_empty = tmem_full + 4;  // [half][tile]
    uint64_t* scale_full = tmem_empty + 4;
    uint64_t* scale_empty = scale_full + S::kScaleSlots;
    uint32_t* tmem_ptr_smem = reinterpret_cast<uint32_t*>(smem + S::kOffTmemPtr);
    uint32_t* tiles = reinterpret_cast<uint32_t*>(smem + S::kOffTiles);
    uint32_t* row_begin = tiles + p.experts + 1u;
    uint32_t* row_end = row_begin + p.experts;

    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
    const uint32_t cta = cluster_ctarank();  // 0 = leader
    const uint32_t pair = blockIdx.x >> 1, num_pairs = gridDim.x >> 1;
    const uint32_t n_tiles = (p.N + kPairBlockN - 1) / kPairBlockN;
    const uint32_t k_blocks = (p.K + 127u) / 128u;
    const uint64_t bar_ns = p.bar_timeout_ns;

    if (threadIdx.x == 32 * kBlockPairPromoters) {
        for (uint32_t s = 0; s < kStages; ++s) {
            mbar_init(&full[s], 2);  // both CTAs' producers (expect_tx)
            mbar_init(&empty[s], 2);  // the products of both halves
        }
        for (uint32_t b = 0; b < 4; ++b) {
            mbar_init(&tmem_full[b], 1);
            mbar_init(&tmem_empty[b], 2);  // a warp of each CTA, for all that promote the half
        }
        for (uint32_t i = 0; i < S::kScaleSlots; ++i) {
            mbar_init(&scale_full[i], kByColumn ? 2 : 1);  // the rows' factors (and the columns' bytes)
            mbar_init(&scale_empty[i], 2);  // a warp of each half
        }
        mbar_fence_init();
        tma_prefetch_desc(&tmap_a);
        tma_prefetch_desc(&tmap_a32);
        tma_prefetch_desc(&tmap_b);
    }
    if (warp == 17) {
        tmem_alloc_pair(tmem_ptr_smem, 512);
        tmem_relinquish_pair();
    }
    grid_dep_wait();
    if (warp == 0) {
        count_block_tiles(p, kPairBlockM, tiles, row_begin, row_end, lane);
    }
    tcgen05_fence_before();
    __syncthreads();
    cluster_sync_all();  // both CTAs' barriers exist before anybody arrives on the other's
    tcgen05_fence_after();
    const uint32_t tmem_base = *tmem_ptr_smem;
    const uint32_t num_units = tiles[p.experts] * n_tiles;
    bool alive = true;  // false once a wait of this role has given up

    struct Unit {
        uint32_t e, m0, end, n0;  // expert; first row of the pair's tile, end of the expert's rows; first column
    };
    GroupedWalk walk;
    auto unit_at = [&](uint32_t unit) {
        const TileCoord tc = walk.seek(tiles, n_tiles, unit);
        return Unit{walk.e, row_begin[walk.e] + tc.m_tile * kPairBlockM, row_end[walk.e], tc.n_tile * kPairBlockN};
    };

    // The changes of registers belong into the branches: code behind one is built for as many as the branch then has, and code
    // that all run again has what the block was launched with.
    if (warp >= kBlockPairPromoters) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kBlockPairOtherRegs));
        if (warp == 16) {
            // ------------------------------- TMA producer (both CTAs) -------------------------
            uint32_t it = 0;
            for (uint32_t unit = pair; alive && unit < num_units; unit += num_pairs) {
                const Unit u = unit_at(unit);
                const uint32_t m0 = u.m0 + cta * 128u;
                const uint32_t boxes = m0 < u.end ? (min(u.end - m0, 128u) + 31u) / 32u : 0u;  // of 32 rows
                const uint32_t tx_bytes = (p.a_cols && boxes ? S::kABytes : boxes * (32u * 128u)) + S::kBBytes;
                const int32_t n = (int32_t)(u.n0 + cta * 128u);
                for (uint32_t kb = 0; alive && kb < k_blocks; ++kb, ++it) {
                    const uint32_t s = it % kStages;
                    const uint32_t leader_bar = map_to_cta(smem_u32(&full[s]), 0);
                    alive = mbar_wait_soon(&empty[s], ((it / kStages) & 1u) ^ 1u, p.status, 500, s, bar_ns);
                    if (!alive) {
                        break;
                    }
                    if (elect_one()) {
                        mbar_arrive_expect_tx_cluster(leader_bar, tx_bytes);
                        const int32_t k = (int32_t)(kb * 128u);
                        tma_load_3d_pair(smem + S::kOffB + s * S::kBBytes, &tmap_b, leader_bar, p.b_rows ? k : n, p.b_rows ? n : k, (int32_t)u.e);
                        uint8_t* a = smem + S::kOffA + s * S::kABytes;
                        if (p.a_cols) {
                            if (boxes) {
                                tma_load_2d_pair(a, &tmap_a, leader_bar, (int32_t)m0, k);
                            }
                        } else if (boxes == 4u) {
                            tma_load_2d_pair(a, &tmap_a, leader_bar, k, (int32_t)m0);
                        } else {
                            for (uint32_t i = 0; i < boxes; ++i) {
                                tma_load_2d_pair(a + i * (32u * 128u), &tmap_a32, leader_bar, k, (int32_t)(m0 + i * 32u));
                            }
                        }
                    }
                    __syncwarp();
                }
            }
        } else if (warp < 19) {
            // ------------------------------- MMA issuers (leader CTA only) --------------------
            if (cta == 0) {
                const uint32_t half = warp - 17u;
                const uint32_t idesc0 = make_idesc_f8(kPairBlockM, 0, p.a_fmt, p.b_fmt, p.a_cols != 0u, p.b_rows == 0u);
                const uint64_t desc_k = make_smem_desc(0, 16, 1024, 2), desc_mn = make_smem_desc(0, 16384, 1024, 2);
                const uint64_t desc_a = p.a_cols ? desc_mn : desc_k, desc_b = p.b_rows ? desc_k : desc_mn;
                const uint32_t hi_a = (uint32_t)(desc_a >> 32), hi_b = (uint32_t)(desc_b >> 32);
                const uint32_t a_lo0 = (uint32_t)desc_a | (smem_u32(smem + S::kOffA) >> 4);
                const uint32_t b_lo0 = ((uint32_t)desc_b | (smem_u32(smem + S::kOffB) >> 4)) + half * ((p.b_rows ? 64u * 128u : 64u) >> 4);
                const uint32_t step_a = (p.a_cols ? 4096u : 32u) >> 4, step_b = (p.b_rows ? 32u : 4096u) >> 4;
                uint64_t* const tile_full = tmem_full + 2u * half;
                uint64_t* const tile_empty = tmem_empty + 2u * half;
                uint32_t s = 0, ph = 0, it = 0;
                for (uint32_t unit = pair; alive && unit < num_units; unit += num_pairs) {
                    // of a ragged last column of tiles as much is multiplied as the leader's columns need (the other CTA's are
                    // fewer), at least the smallest product
                    const uint32_t left = p.N - unit_at(unit).n0;
                    const uint32_t columns = min(max(left, 64u * half + 16u) - 64u * half, 64u);
                    const uint32_t idesc = idesc0 | (((columns + 15u) / 16u * 32u >> 3) << 17);
                    for (uint32_t i = 0; alive && i < k_blocks; ++i, ++it) {
                        const uint32_t buf = it & 1u;
                        // the operands are there before the tile is free, as a rule: what is waited for last is what counts
                        alive = mbar_wait_soon(&full[s], ph, p.status, 503, s, bar_ns) &&
                                mbar_wait_soon(&tile_empty[buf], ((it >> 1) & 1u) ^ 1u, p.status, 501 + half, buf, bar_ns);
                        if (!alive) {
                            break;  // nothing is issued, and no tile reported, after a wait has given up
                        }
                        tcgen05_fence_after();
                        umma_f8_pair_block(tmem_base + half * 256u + buf * 128u, a_lo0 + s * (S::kABytes >> 4), hi_a, step_a,
                                           b_lo0 + s * (S::kBBytes >> 4), hi_b, step_b, idesc, &tile_full[buf], &empty[s]);
                        s = (s + 1 == kStages) ? 0u : s + 1;
                        ph ^= s == 0u ? 1u : 0u;
                    }
                }
            }
        } else {
            // ------------------------------- factors (both CTAs, own 128 rows) ----------------
            uint32_t it = 0;
            for (uint32_t unit = pair; alive && unit < num_units; unit += num_pairs) {
                const Unit u = unit_at(unit);
                const uint32_t row = u.m0 + cta * 128u + lane;
                const uint32_t scale_bytes = min(p.N - u.n0, kPairBlockN) * 4u;
                const float* b_scales = p.b_scales + u.e * p.b_scale_matrix + (u.n0 / 128u) * p.b_scale_col;
                const size_t b_next = u.n0 + 128u < p.N ? p.b_scale_col : 0u;
                for (uint32_t kb0 = 0; alive && kb0 < k_blocks; kb0 += 4u) {
                    float a[4][4], b[2][4];  // of four blocks
#pragma unroll
                    for (uint32_t i = 0; i < 4; ++i) {
                        load_scales(p.a_scales + min(row + 32u * i, u.end - 1u) * p.a_scale_row, p.a_scale_block, kb0, k_blocks, a[i]);
                    }
                    if (!kByColumn) {
                        load_scales(b_scales, p.b_scale_block, kb0, k_blocks, b[0]);
                        load_scales(b_scales + b_next, p.b_scale_block, kb0, k_blocks, b[1]);
                    }
#pragma unroll
                    for (uint32_t j = 0; j < 4; ++j) {
                        if (kb0 + j >= k_blocks || !alive) {
                            break;
                        }
                        const uint32_t slot = it % S::kScaleSlots;
                        alive = mbar_wait_soon(&scale_empty[slot], ((it / S::kScaleSlots) & 1u) ^ 1u, p.status, 505, slot, bar_ns);
                        if (!alive) {
                            break;
                        }
                        if (kByColumn && elect_one()) {
                            mbar_arrive_expect_tx(&scale_full[slot], scale_bytes);
                            bulk_load(smem + S::kOffScale + slot * (kPairBlockN * 4u), p.b_scales + (kb0 + j) * p.b_scale_block + u.n0, scale_bytes,
                                      &scale_full[slot]);
                        }
                        __syncwarp();
                        float* factor = reinterpret_cast<float*>(smem + S::kOffFactor) + slot * 256u + lane;
#pragma unroll
                        for (uint32_t i = 0; i < 4; ++i) {
                            factor[32u * i] = kByColumn ? a[i][j] : a[i][j] * b[0][j];
                            factor[128u + 32u * i] = kByColumn ? a[i][j] : a[i][j] * b[1][j];
                        }
                        __syncwarp();
                        if (lane == 0) {
                            mbar_arrive(&scale_full[slot]);
                        }
                        ++it;
                    }
                }
            }
        }
        __syncwarp();
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kBlockPairRegs));
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kBlockPairPromoteRegs));
        // ------------------------------- promotion and output (both CTAs, own 128 rows) ---
        const uint32_t q = warp & 3u, half = warp >> 3, from = (warp >> 2) & 1u, col = from * 128u + half * kCols;
        const uint32_t tmem = tmem_base + ((q * 32u) << 16) + half * 256u + from * kCols, w8 = warp & 7u;
        const float* factors = reinterpret_cast<const float*>(smem + S::kOffFactor) + from * 128u + q * 32u + lane;
        const uint32_t free_bar0 = map_to_cta(smem_u32(&tmem_empty[2u * half]), 0), free_bar1 = map_to_cta(smem_u32(&tmem_empty[2u * half + 1u]), 0);
        uint32_t it = 0;
        float next = 0.0f;  // the next block's factor
        if (pair < num_units) {
            if (w8 == 1u) {
                alive = mbar_wait_soon(&scale_full[0], 0, p.status, 508, 0, bar_ns);
            }
            alive = promoters_agree(1u + half, alive);
            next = factors[0];
        }
        for (uint32_t unit = pair; alive && unit < num_units; unit += num_pairs) {
            const Unit u = unit_at(unit);
            const uint32_t row0 = u.m0 + cta * 128u + q * 32u, row = row0 + lane, col0 = u.n0 + col;
            const bool live = row0 < u.end && col0 < p.N;  // else there is nothing to fetch
            float acc[kCols] = {};
            for (uint32_t i = 0; i < k_blocks; ++i, ++it) {
                const uint32_t buf = it & 1u, slot = it % S::kScaleSlots;
                if (w8 == 0u) {
                    alive = mbar_wait_soon(&tmem_full[2u * half + buf], (it >> 1) & 1u, p.status, 506, buf, bar_ns);
                } else if (w8 == 1u && (i + 1u < k_blocks || unit + num_pairs < num_units)) {
                    const uint32_t nt = it + 1u;
                    alive = mbar_wait_soon(&scale_full[nt % S::kScaleSlots], (nt / S::kScaleSlots) & 1u, p.status, 507, nt % S::kScaleSlots, bar_ns);
                }
                alive = promoters_agree(1u + half, alive);
                if (!alive) {
                    break;  // a tile that never filled is not written out
                }
                tcgen05_fence_after();
                const float f = next;
                next = factors[(it + 1u) % S::kScaleSlots * 256u];  // behind the last block: whatever is there
                if (live) {
                    promote<kCols, kByColumn>(acc, tmem + buf * 128u, f, reinterpret_cast<const float*>(smem + S::kOffScale) + slot * kPairBlockN + col);
                }
                tcgen05_fence_before();
                if (w8 == 2u || w8 == 3u) {
                    asm volatile("barrier.cta.sync %0, %1;" ::"r"(3u + half), "n"(16 * kBlockPairPromoters) : "memory");
                    if (lane == 0) {
                        if (w8 == 2u) {
                            mbar_arrive_cluster(buf ? free_bar1 : free_bar0);
                        } else {
                            mbar_arrive(&scale_empty[slot]);
                        }
                    }
                    __syncwarp();
                } else {
                    asm volatile("barrier.cta.arrive %0, %1;" ::"r"(3u + half), "n"(16 * kBlockPairPromoters) : "memory");
                }
            }
            if (alive && row < u.end) {
                OutT* dst = static_cast<OutT*>(p.c) + (size_t)row * p.N + col0;
#pragma unroll
                for (uint32_t c = 0; c < kCols; c += 16) {
                    if (col0 + c < p.N) {
                        store_16(dst + c, &acc[c]);
                    }
                }
            }
        }
        __syncwarp();
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kBlockPairRegs));
    }

    tcgen05_fence_before();
    if (__syncthreads_or(alive ? 0 : 1)) {
        drain_after_abort(p.status);  // both CTAs stay while loads that report to the other's barriers may be in flight
    }
    cluster_sync_all();  // nobody leaves while the other CTA may still arrive on its barriers
    if (warp == 17) {
        tcgen05_fence_after();
        tmem_dealloc_pair(tmem_base, 512);
    }
}

}  // namespace catccos
