// The products of block_gemm.cuh on CTA pairs (clusters of two SMs, tcgen05 cta_group::2), for calls that fill the GPU with 256 x 256
// tiles.
//
// CTA r of a pair loads rows [128 r, +128) of A and columns [128 r, +128) of B (of a ragged last column of tiles, its half) with
// plain TMA, 32 KB a block of K where a 128 x 256 tile on one SM takes 48; the leader issues the products of both, and each CTA
// has the tile of its own 128 rows and all 256 columns in its own tensor memory.  Two such tiles fill tensor memory: one is
// multiplied while the sixteen promotion warps (row = lane, 64 columns each) scale the other and add it to their sums.
//
//   full[s], tmem_empty[b]     live in the leader; both CTAs' TMA bytes, and promotion warps, go there
//   empty[s], tmem_full[b]     live in each CTA; the leader's tcgen05.commit arrives on both copies
//   scale_full[i], scale_empty[i]  live in each CTA: the factors of its rows (and, by column, of the columns) for one block of K
//
// 640 threads: warps 0-15 promotion and output (warp w: lane quarter w % 4, columns 64 (w / 4)), warp 16 TMA, 17 MMA, 18 and 19
// the factors: a row's scale times that of each half of the columns.  The promotion warps take registers from the other four.
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
    static constexpr uint32_t kScaleSlots = 4;
    static constexpr uint32_t kOffScale = kOffB + kStages * kBBytes;               // by column: 256 scales a slot
    static constexpr uint32_t kOffFactor = kOffScale + kScaleSlots * kPairBlockN * 4;  // [half][128 rows] a slot
    static constexpr uint32_t kOffBar = kOffFactor + kScaleSlots * 256 * 4;
    static constexpr uint32_t kNumBars = 2 * kStages + 4 + 2 * kScaleSlots;
    static constexpr uint32_t kOffTmemPtr = kOffBar + kNumBars * 8;
    static constexpr uint32_t kOffTiles = kOffTmemPtr + 16;
    static constexpr uint32_t dynamic_bytes(uint32_t experts) { return kOffTiles + (3u * experts + 1u) * 4u + 1024u; }
};
static_assert(BlockPairSmem::dynamic_bytes(kGroupedMaxExperts) <= 232448, "one CTA's shared memory");

__device__ __forceinline__ void umma_f8_pair(uint32_t tmem_d, uint32_t a_lo, uint32_t a_hi, uint32_t b_lo, uint32_t b_hi, uint32_t idesc,
                                             uint32_t accumulate)
{
    asm volatile(
        "{\n\t"
        ".reg .pred p;\n\t"
        ".reg .b64 da, db;\n\t"
        "mov.b64 da, {%1, %2};\n\t"
        "mov.b64 db, {%3, %4};\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], da, db, %5, p;\n\t"
        "}"
        ::"r"(tmem_d), "r"(a_lo), "r"(a_hi), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"(accumulate)
        : "memory");
}

__device__ __forceinline__ void tma_load_3d_pair(void* smem_dst, const void* tmap, uint32_t bar_cluster_addr, int32_t x, int32_t y, int32_t z)
{
    asm volatile(
        "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
        ::"r"(smem_u32(smem_dst)), "l"(tmap), "r"(bar_cluster_addr), "r"(x), "r"(y), "r"(z)
        : "memory");
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
    uint64_t* tmem_empty = tmem_full + 2;
    uint64_t* scale_full = tmem_empty + 2;
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
            mbar_init(&empty[s], 1);
        }
        for (uint32_t b = 0; b < 2; ++b) {
            mbar_init(&tmem_full[b], 1);
            mbar_init(&tmem_empty[b], 2 * kBlockPairPromoters);  // of both CTAs
        }
        for (uint32_t i = 0; i < S::kScaleSlots; ++i) {
            mbar_init(&scale_full[i], kByColumn ? 3 : 2);  // warps 18 and 19 (and the columns' bytes)
            mbar_init(&scale_empty[i], kBlockPairPromoters);
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
        uint32_t e, m0, end, n0, width;  // expert; first row of the pair's tile, end of the expert's rows; first column, columns multiplied
    };
    GroupedWalk walk;
    auto unit_at = [&](uint32_t unit) {
        const TileCoord tc = walk.seek(tiles, n_tiles, unit);
        const uint32_t left = p.N - tc.n_tile * kPairBlockN;
        return Unit{walk.e, row_begin[walk.e] + tc.m_tile * kPairBlockM, row_end[walk.e], tc.n_tile * kPairBlockN,
                    left < kPairBlockN ? (left + 31u) / 32u * 32u : kPairBlockN};
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
                const int32_t n = (int32_t)(u.n0 + cta * (u.width / 2u));
                for (uint32_t kb = 0; alive && kb < k_blocks; ++kb, ++it) {
                    const uint32_t s = it % kStages;
                    const uint32_t leader_bar = map_to_cta(smem_u32(&full[s]), 0);
                    alive = mbar_wait_warp(&empty[s], ((it / kStages) & 1u) ^ 1u, p.status, 500, s, bar_ns);
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
        } else if (warp == 17) {
            // ------------------------------- MMA issuer (leader CTA only) ---------------------
            if (cta == 0) {
                const uint32_t idesc0 = make_idesc_f8(kPairBlockM, 0, p.a_fmt, p.b_fmt, p.a_cols != 0u, p.b_rows == 0u);
                const uint64_t desc_k = make_smem_desc(0, 16, 1024, 2), desc_mn = make_smem_desc(0, 16384, 1024, 2);
                const uint64_t desc_a = p.a_cols ? desc_mn : desc_k, desc_b = p.b_rows ? desc_k : desc_mn;
                const uint32_t hi_a = (uint32_t)(desc_a >> 32), hi_b = (uint32_t)(desc_b >> 32);
                const uint32_t a_lo0 = (uint32_t)desc_a | (smem_u32(smem + S::kOffA) >> 4);
                const uint32_t b_lo0 = (uint32_t)desc_b | (smem_u32(smem + S::kOffB) >> 4);
                const uint32_t step_a = (p.a_cols ? 4096u : 32u) >> 4, step_b = (p.b_rows ? 32u : 4096u) >> 4;
                uint32_t s = 0, ph = 0, it = 0;
                for (uint32_t unit = pair; alive && unit < num_units; unit += num_pairs) {
                    const uint32_t idesc = idesc0 | ((unit_at(unit).width >> 3) << 17);
                    for (uint32_t i = 0; alive && i < k_blocks; ++i, ++it) {
                        const uint32_t buf = it & 1u;
                        alive = mbar_wait_warp(&tmem_empty[buf], ((it >> 1) & 1u) ^ 1u, p.status, 501, buf, bar_ns) &&
                                mbar_wait_warp(&full[s], ph, p.status, 503, s, bar_ns);
                        if (!alive) {
                            break;  // nothing is issued, and no tile reported, after a wait has given up
                        }
                        tcgen05_fence_after();
                        if (elect_one()) {
                            const uint32_t a_lo = a_lo0 + s * (S::kABytes >> 4), b_lo = b_lo0 + s * (S::kBBytes >> 4);
#pragma unroll
                            for (uint32_t j = 0; j < 4; ++j) {
                                umma_f8_pair(tmem_base + buf * kPairBlockN, a_lo + j * step_a, hi_a, b_lo + j * step_b, hi_b, idesc, j);
                            }
                            tcgen05_commit_pair(&empty[s], 3);
                            tcgen05_commit_pair(&tmem_full[buf], 3);
                        }
                        __syncwarp();
                        s = (s + 1 == kStages) ? 0u : s + 1;
                        ph ^= s == 0u ? 1u : 0u;
                    }
                }
            }
        } else if (warp >= 18) {
            // ------------------------------- factors (both CTAs, own 128 rows) ----------------
            const uint32_t r0 = (warp - 18u) * 64u + lane;  // this lane's rows: r0 and r0 + 32
            uint32_t it = 0;
            for (uint32_t unit = pair; alive && unit < num_units; unit += num_pairs) {
                const Unit u = unit_at(unit);
                const uint32_t row = u.m0 + cta * 128u + r0;
                const uint32_t scale_bytes = min(p.N - u.n0, kPairBlockN) * 4u;
                const float* b_scales = p.b_scales + u.e * p.b_scale_matrix + (u.n0 / 128u) * p.b_scale_col;
                ScaleReader sa[2], sb[2];
#pragma unroll
                for (uint32_t i = 0; i < 2; ++i) {
                    sa[i].start(p.a_scales + min(row + 32u * i, u.end - 1u) * p.a_scale_row, p.a_scale_block, 0, k_blocks);
                    sb[i].start(b_scales + (u.n0 + 128u * i < p.N ? i : 0u) * p.b_scale_col, p.b_scale_block, 0, kByColumn ? 0u : k_blocks);
                }
                for (uint32_t kb = 0; alive && kb < k_blocks; ++kb, ++it) {
                    const uint32_t slot = it % S::kScaleSlots;
                    float a[2], b[2];
#pragma unroll
                    for (uint32_t i = 0; i < 2; ++i) {
                        a[i] = sa[i].get(kb);
                        b[i] = kByColumn ? 1.0f : sb[i].get(kb);
                    }
                    alive = mbar_wait_warp(&scale_empty[slot], ((it / S::kScaleSlots) & 1u) ^ 1u, p.status, 505, slot, bar_ns);
                    if (!alive) {
                        break;
                    }
                    if (kByColumn && warp == 18 && elect_one()) {
                        mbar_arrive_expect_tx(&scale_full[slot], scale_bytes);
                        bulk_load(smem + S::kOffScale + slot * (kPairBlockN * 4u), p.b_scales + kb * p.b_scale_block + u.n0, scale_bytes,
                                  &scale_full[slot]);
                    }
                    __syncwarp();
                    float* factor = reinterpret_cast<float*>(smem + S::kOffFactor) + slot * 256u + r0;
                    factor[0] = a[0] * b[0];
                    factor[32] = a[1] * b[0];
                    factor[128] = a[0] * b[1];
                    factor[160] = a[1] * b[1];
                    __syncwarp();
                    if (lane == 0) {
                        mbar_arrive(&scale_full[slot]);
                    }
                }
            }
        }
        __syncwarp();
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kBlockPairRegs));
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kBlockPairPromoteRegs));
        // ------------------------------- promotion and output (both CTAs, own 128 rows) ---
        const uint32_t q = warp & 3u, col = (warp >> 2) * kCols;
        const uint32_t tmem = tmem_base + ((q * 32u) << 16) + col;
        const uint32_t free_bar0 = map_to_cta(smem_u32(&tmem_empty[0]), 0), free_bar1 = map_to_cta(smem_u32(&tmem_empty[1]), 0);
        uint32_t it = 0;
        for (uint32_t unit = pair; alive && unit < num_units; unit += num_pairs) {
            const Unit u = unit_at(unit);
            const uint32_t row0 = u.m0 + cta * 128u + q * 32u, row = row0 + lane, col0 = u.n0 + col;
            const bool live = row0 < u.end && col0 < p.N;  // else there is nothing to fetch
            float acc[kCols] = {};
            for (uint32_t i = 0; i < k_blocks; ++i, ++it) {
                const uint32_t buf = it & 1u, slot = it % S::kScaleSlots;
                alive = mbar_wait_warp(&scale_full[slot], (it / S::kScaleSlots) & 1u, p.status, 507, slot, bar_ns) &&
                        mbar_wait_warp(&tmem_full[buf], (it >> 1) & 1u, p.status, 506, buf, bar_ns);
                if (!alive) {
                    break;  // a tile that never filled is not written out
                }
                tcgen05_fence_after();
                if (live) {
                    const float f = reinterpret_cast<const float*>(smem + S::kOffFactor)[slot * 256u + (col & 128u) + q * 32u + lane];
                    promote<kCols, kByColumn>(acc, tmem + buf * kPairBlockN, f, reinterpret_cast<const float*>(smem + S::kOffScale) + slot * kPairBlockN + col);
                }
                tcgen05_fence_before();
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive_cluster(buf ? free_bar1 : free_bar0);
                    mbar_arrive(&scale_empty[slot]);
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
