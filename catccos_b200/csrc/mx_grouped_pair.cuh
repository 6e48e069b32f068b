// Grouped MXFP8 GEMM on CTA pairs: the experts' products of mx_grouped_gemm.cuh on the 256 x 256 tiles of mx_gemm_pair.cuh, for
// calls with many rows an expert.
//
// A 128 x 256 tile on one SM moves 48 KB into and 48 KB out of shared memory a K tile, 750 cycles at 128 bytes, for 512 cycles of
// products; a pair's SM moves 32 and 32.  Against that, an expert's rows are padded to 256 instead of 128.
//
// Tile, rings, tensor-memory layout and roles are those of mx_gemm_pair_kernel without its gates, split tiles and staged
// output (a box of output rows would run into the next expert's); the list of work is that of mx_grouped_gemm_kernel.
#pragma once

#include "mx_gemm_pair.cuh"
#include "mx_grouped_gemm.cuh"

namespace catccos {

struct GroupedPairSmem {
    using S = PairSmem;
    static constexpr uint32_t kOffTiles = S::kOffOut;  // the list of work lies where the other kernel stages its output
    static_assert((3u * kGroupedMaxExperts + 1u) * 4u <= 4 * kOutStageBytes, "the list of work fits");
};

template <typename OutT>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kGemmThreads, 1)
mx_grouped_pair_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_a32,
                       const __grid_constant__ CUtensorMap tmap_b, const __grid_constant__ GroupedParams p)
{
    using S = PairSmem;
    constexpr uint32_t kStages = S::kStages;

    grid_dep_launch();
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + S::kOffBar);
    uint64_t* full = bars;
    uint64_t* empty = full + kStages;
    uint64_t* tmem_full = empty + kStages;
    uint64_t* tmem_empty = tmem_full + 2;
    uint64_t* overlap_free = tmem_empty + 2;
    uint64_t* sf_full = overlap_free + 2;
    uint64_t* sf_empty = sf_full + 2;
    uint64_t* atoms = sf_empty + 2;
    uint32_t* tmem_ptr_smem = reinterpret_cast<uint32_t*>(smem + S::kOffTmemPtr);
    uint32_t* tiles = reinterpret_cast<uint32_t*>(smem + GroupedPairSmem::kOffTiles);
    uint32_t* row_begin = tiles + p.experts + 1u;
    uint32_t* row_end = row_begin + p.experts;

    const uint32_t warp = threadIdx.x >> 5;
    const uint32_t lane = threadIdx.x & 31;
    const uint32_t cta = cluster_ctarank();  // 0 = leader
    const uint32_t pair = blockIdx.x >> 1, num_pairs = gridDim.x >> 1;
    const uint32_t n_tiles = (p.N + kPairBlockN - 1) / kPairBlockN;
    const uint32_t k_tiles = p.K / kGemmBlockK;
    const uint64_t bar_ns = p.bar_timeout_ns;

    if (threadIdx.x == 128) {
        for (uint32_t s = 0; s < kStages; ++s) {
            mbar_init(&full[s], 2);  // both CTAs' producers (expect_tx)
            mbar_init(&empty[s], 1);
        }
        for (uint32_t a = 0; a < 2; ++a) {
            mbar_init(&tmem_full[a], 1);
            mbar_init(&tmem_empty[a], 8);  // four epilogue warps in each CTA
            mbar_init(&overlap_free[a], 8);
            mbar_init(&sf_full[a], kSfGroup);  // one commit behind each K tile's copies
            mbar_init(&sf_empty[a], 1);
            mbar_init(&atoms[a], 8);  // four scale-loader warps in each CTA
        }
        mbar_fence_init();
        tma_prefetch_desc(&tmap_a);
        tma_prefetch_desc(&tmap_a32);
        tma_prefetch_desc(&tmap_b);
    }
    if (warp == 5) {
        tmem_alloc_pair(tmem_ptr_smem, kTmemCols);
        tmem_relinquish_pair();
    }
    grid_dep_wait();  // the offsets, the rows and their scales come from the kernels before this one
    if (warp == 0) {
        count_grouped_tiles(p, kPairBlockM, tiles, row_begin, row_end, lane);
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

    if (warp == 4) {
        // ------------------------------- TMA producer (both CTAs) -------------------------
        uint32_t it = 0;
        for (uint32_t unit = pair; alive && unit < num_units; unit += num_pairs) {
            const Unit u = unit_at(unit);
            const uint32_t m0 = u.m0 + cta * 128u;
            const uint32_t boxes = m0 < u.end ? (min(u.end - m0, 128u) + 31u) / 32u : 0u;  // of 32 rows
            const uint32_t tx_bytes = boxes * (32u * kGemmBlockK) + S::kBBytes;
            const int32_t n = (int32_t)(u.n0 + cta * (u.width / 2u));
            const uint32_t b_row0 = u.e * p.K;
            for (uint32_t kt = 0; alive && kt < k_tiles; ++kt, ++it) {
                const uint32_t s = it % kStages;
                const uint32_t leader_bar = map_to_cta(smem_u32(&full[s]), 0);
                alive = mbar_wait_warp(&empty[s], ((it / kStages) & 1u) ^ 1u, p.status, 200, s, bar_ns);
                if (!alive) {
                    break;
                }
                if (elect_one()) {
                    mbar_arrive_expect_tx_cluster(leader_bar, tx_bytes);
                    const int32_t k = (int32_t)(kt * kGemmBlockK);
                    tma_load_2d_pair(smem + S::kOffB + s * S::kBBytes, &tmap_b, leader_bar, n, (int32_t)b_row0 + k);
                    uint8_t* a = smem + S::kOffA + s * S::kABytes;
                    if (boxes == 4u) {
                        tma_load_2d_pair(a, &tmap_a, leader_bar, k, (int32_t)m0);
                    } else {
                        for (uint32_t i = 0; i < boxes; ++i) {
                            tma_load_2d_pair(a + i * (32u * kGemmBlockK), &tmap_a32, leader_bar, k, (int32_t)(m0 + i * 32u));
                        }
                    }
                }
                __syncwarp();
            }
        }
    } else if (warp == 5) {
        // ------------------------------- MMA issuer (leader CTA only) ---------------------
        if (cta == 0) {
            const uint32_t idesc0 = make_idesc_mxf8(kPairBlockM, 0, true) | ((p.a_fmt & 7u) << 7) | ((p.b_fmt & 7u) << 10);
            const uint32_t hi_a = (uint32_t)(make_smem_desc(0, 16, 1024, 2) >> 32);
            const uint64_t desc_b = make_smem_desc(0, 16384, 1024, 2);
            const uint32_t hi_b = (uint32_t)(desc_b >> 32);
            const uint32_t a_lo0 = (uint32_t)make_smem_desc(0, 16, 1024, 2) | (smem_u32(smem + S::kOffA) >> 4);
            const uint32_t b_lo0 = (uint32_t)desc_b | (smem_u32(smem + S::kOffB) >> 4);
            uint32_t s = 0, ph = 0;  // operand stage and its phase
            uint32_t group = 0;      // scale groups consumed
            uint32_t ui = 0;
            for (uint32_t unit = pair; alive && unit < num_units; unit += num_pairs, ++ui) {
                const uint32_t acc = ui & 1u;
                const uint32_t d_col = tmem_base + (acc ? S::kAccCol1 : 0u);
                alive = mbar_wait_warp(&tmem_empty[acc], ((ui >> 1) & 1u) ^ 1u, p.status, 201, acc, bar_ns);
                if (ui > 0 && alive) {
                    alive = mbar_wait_warp(&overlap_free[acc ^ 1u], ((ui - 1) >> 1) & 1u, p.status, 202, acc, bar_ns);
                }
                const uint32_t idesc = idesc0 | ((unit_at(unit).width >> 3) << 17);
                for (uint32_t i = 0; alive && i < k_tiles; ++i) {
                    const uint32_t buf = group & 1u;
                    if (i % kSfGroup == 0u) {
                        alive = mbar_wait_warp(&sf_full[buf], (group >> 1) & 1u, p.status, 207, buf, bar_ns);
                    }
                    alive = alive && mbar_wait_warp(&full[s], ph, p.status, 203, s, bar_ns);
                    if (!alive) {
                        break;  // nothing is issued, and the accumulator never reported, after a wait has given up
                    }
                    tcgen05_fence_after();
                    const uint32_t a_lo = a_lo0 + s * (S::kABytes >> 4);
                    const uint32_t b_lo = b_lo0 + s * (S::kBBytes >> 4);
                    const uint32_t sf = tmem_base + S::kSfCol + buf * S::kSfGroupCols + (i % kSfGroup) * S::kSfSetCols;
                    const bool group_end = i % kSfGroup == kSfGroup - 1u || i + 1u == k_tiles;
                    if (elect_one()) {
#pragma unroll
                        for (uint32_t kb = 0; kb < 4; ++kb) {
                            umma_mxf8_pair_lohi(d_col, a_lo + kb * (32u >> 4), hi_a, b_lo + kb * (4096u >> 4), hi_b,
                                                idesc_with_sf_id(idesc, kb), sf, sf + 4, (kb != 0u || i != 0u) ? 1u : 0u);
                        }
                        tcgen05_commit_pair(&empty[s], 3);
                        if (group_end) {
                            tcgen05_commit_pair(&sf_empty[buf], 3);
                        }
                        if (i + 1u == k_tiles) {
                            tcgen05_commit_pair(&tmem_full[acc], 3);
                        }
                    }
                    __syncwarp();
                    group += group_end ? 1u : 0u;
                    s = (s + 1 == kStages) ? 0u : s + 1;
                    ph ^= s == 0u ? 1u : 0u;
                }
            }
        }
    } else if (warp >= 6) {
        // ------------------------------- scale loaders (both CTAs) ------------------------
        // Warp j loads the A scales of this CTA's rows [32 j, +32) for all four K tiles of a group (16 bytes per row) and
        // the B scales of all columns of the pair's tile for K tile j.
        constexpr uint32_t kNB = kPairBlockN / 32;
        const uint32_t j = warp - 6;
        const bool a_wide = p.K % 512u == 0u && ((uintptr_t)p.a_scales & 15u) == 0u && p.a_scale_stride % 16u == 0u;
        uint32_t cur_lo[kNB], cur_hi[kNB], nxt_lo[kNB], nxt_hi[kNB];
        uint4 cur_a, nxt_a;

        struct Cursor {
            uint32_t unit, kt;
            Unit u;
        };
        auto next = [&](Cursor& c) {
            c.kt += kSfGroup;
            if (c.kt >= k_tiles) {
                c.kt = 0;
                c.unit += num_pairs;
                if (c.unit < num_units) {
                    c.u = unit_at(c.unit);
                }
            }
        };
        auto load = [&](const Cursor& c, uint32_t (&rlo)[kNB], uint32_t (&rhi)[kNB], uint4& ra) {
            const uint32_t kt = c.kt + j;
            const uint8_t* b_scales = p.b_scales + ((size_t)c.u.e * (p.K / 64u) + 2u * kt) * p.N * 2u;
#pragma unroll
            for (uint32_t i = 0; i < kNB; ++i) {
                const uint32_t n = c.u.n0 + i * 32 + lane;
                rlo[i] = 0x7F7Fu;
                rhi[i] = 0x7F7Fu;
                if (n < p.N && kt < k_tiles) {
                    rlo[i] = *reinterpret_cast<const uint16_t*>(b_scales + (size_t)n * 2u);
                    rhi[i] = *reinterpret_cast<const uint16_t*>(b_scales + ((size_t)p.N + n) * 2u);
                }
            }
            const uint32_t last = min(c.kt + kSfGroup, k_tiles);  // K tiles [c.kt, last) of the group exist
            const uint32_t row = c.u.m0 + cta * 128u + j * 32 + lane;
            ra = make_uint4(0x7F7F7F7Fu, 0x7F7F7F7Fu, 0x7F7F7F7Fu, 0x7F7F7F7Fu);
            if (row < c.u.end) {
                const uint32_t* src = reinterpret_cast<const uint32_t*>(p.a_scales + (size_t)row * p.a_scale_stride) + c.kt;
                if (a_wide) {
                    ra = __ldcg(reinterpret_cast<const uint4*>(src));  // K % 512 == 0: the four K tiles are in the row
                } else {
                    ra.x = __ldcg(src);
                    ra.y = c.kt + 1u < last ? __ldcg(src + 1) : ra.y;
                    ra.z = c.kt + 2u < last ? __ldcg(src + 2) : ra.z;
                    ra.w = c.kt + 3u < last ? __ldcg(src + 3) : ra.w;
                }
            }
        };

        Cursor c = {pair, 0, {}};
        if (c.unit < num_units) {
            c.u = unit_at(c.unit);
            load(c, cur_lo, cur_hi, cur_a);
        }
        uint32_t group = 0;
        while (alive && c.unit < num_units) {
            const bool real = c.kt + j < k_tiles;  // the last group of a unit may be short
            next(c);
            if (c.unit < num_units) {
                load(c, nxt_lo, nxt_hi, nxt_a);
            }
            const uint32_t buf = group & 1u, ph = (group >> 1) & 1u;
            alive = mbar_wait_warp(&sf_empty[buf], ph ^ 1u, p.status, 205, buf, bar_ns);
            uint8_t* sfa = smem + S::kOffSf + buf * S::kSfBufBytes;
            uint8_t* sfb = sfa + kSfGroup * S::kSfaBytes + j * S::kSfbBytes;
            {
                // an atom row holds the words of tile rows lane, lane + 32, lane + 64, lane + 96: this warp's is word j
                uint32_t* dst = reinterpret_cast<uint32_t*>(sfa + lane * 16u) + j;
                dst[0] = cur_a.x;
                dst[S::kSfaBytes / 4] = cur_a.y;
                dst[2 * S::kSfaBytes / 4] = cur_a.z;
                dst[3 * S::kSfaBytes / 4] = cur_a.w;
            }
#pragma unroll
            for (uint32_t h = 0; h < kNB / 4; ++h) {
                uint4 v;
                v.x = cur_lo[h * 4 + 0] | (cur_hi[h * 4 + 0] << 16);
                v.y = cur_lo[h * 4 + 1] | (cur_hi[h * 4 + 1] << 16);
                v.z = cur_lo[h * 4 + 2] | (cur_hi[h * 4 + 2] << 16);
                v.w = cur_lo[h * 4 + 3] | (cur_hi[h * 4 + 3] << 16);
                *reinterpret_cast<uint4*>(sfb + h * 512u + lane * 16u) = v;
            }
            fence_proxy_async_shared();
            __syncwarp();
            // All loader warps of both CTAs report their atoms to the leader; the leader's warp j then copies K tile j's atoms of
            // both CTAs into both CTAs' tensor memory (one cta_group::2 copy does the same offsets in the two).
            if (lane == 0) {
                mbar_arrive_cluster(map_to_cta(smem_u32(&atoms[buf]), 0));
            }
            if (cta == 0) {
                alive = mbar_wait_warp(&atoms[buf], ph, p.status, 208, buf, bar_ns) && alive;
                tcgen05_fence_after();
                if (elect_one()) {
                    if (real) {
                        const uint32_t hi_sf = (uint32_t)(make_smem_desc(0, 0, 128, 0) >> 32);
                        const uint32_t sf_t = tmem_base + S::kSfCol + buf * S::kSfGroupCols + j * S::kSfSetCols;
                        tcgen05_cp_sf_pair_lohi(sf_t, smem_u32(sfa + j * S::kSfaBytes) >> 4, hi_sf);
#pragma unroll
                        for (uint32_t h = 0; h < kPairBlockN / 128; ++h) {
                            tcgen05_cp_sf_pair_lohi(sf_t + 4 + 4 * h, (smem_u32(sfb) >> 4) + h * (512u >> 4), hi_sf);
                        }
                    }
                    tcgen05_commit_pair(&sf_full[buf], 1);
                }
                __syncwarp();
            }
            ++group;
            cur_a = nxt_a;
#pragma unroll
            for (uint32_t i = 0; i < kNB; ++i) {
                cur_lo[i] = nxt_lo[i];
                cur_hi[i] = nxt_hi[i];
            }
        }
    } else {
        // ------------------------------- epilogue (both CTAs, own 128 rows) ---------------
        const uint32_t q = warp;
        const uint32_t lane_base = tmem_base + ((q * 32u) << 16);
        uint32_t ui = 0;
        for (uint32_t unit = pair; alive && unit < num_units; unit += num_pairs, ++ui) {
            const Unit u = unit_at(unit);
            const uint32_t row0 = u.m0 + cta * 128u + q * 32u;  // this warp's first row
            const uint32_t row = row0 + lane;
            const uint32_t acc = ui & 1u;
            const uint32_t d_col = acc ? S::kAccCol1 : 0u;
            alive = mbar_wait_warp(&tmem_full[acc], (ui >> 1) & 1u, p.status, 206, acc, bar_ns);
            if (!alive) {
                break;  // an accumulator that never filled is not written out
            }
            tcgen05_fence_after();
            OutT* dst = static_cast<OutT*>(p.c) + (size_t)row * p.N + u.n0;
            // The half that holds the columns shared with the other accumulator goes first, columns 128..255 of accumulator 0,
            // 0..127 of accumulator 1, and is given back before anything is converted or stored.
            for (uint32_t hi = 0; hi < 2; ++hi) {
                const uint32_t col0 = (acc == 0u ? 1u - hi : hi) * 128u;
                uint32_t r[4][32];
                if (row0 < u.end) {  // a warp whose rows all lie behind the expert's last has nothing to fetch
#pragma unroll
                    for (uint32_t i = 0; i < 4; ++i) {
                        tmem_ld_32x32(lane_base + d_col + col0 + i * 32u, r[i]);
                    }
                    tmem_ld_wait();
                }
                tcgen05_fence_before();
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive_cluster(map_to_cta(smem_u32(hi == 0u ? &overlap_free[acc] : &tmem_empty[acc]), 0));
                }
                if (row < u.end) {
#pragma unroll
                    for (uint32_t i = 0; i < 8; ++i) {
                        if (u.n0 + col0 + i * 16u < p.N) {
                            uint32_t o[8];
#pragma unroll
                            for (uint32_t x = 0; x < 8; ++x) {
                                o[x] = pack2<OutT>(__uint_as_float(r[i / 2][(i & 1) * 16 + 2 * x]), __uint_as_float(r[i / 2][(i & 1) * 16 + 2 * x + 1]));
                            }
                            st_global_v8(dst + col0 + i * 16u, o);
                        }
                    }
                }
            }
        }
    }

    tcgen05_fence_before();
    if (__syncthreads_or(alive ? 0 : 1)) {
        drain_after_abort(p.status);  // both CTAs stay while loads that report to the other's barriers may be in flight
    }
    cluster_sync_all();  // nobody leaves while the other CTA may still arrive on its barriers
    if (warp == 5) {
        tcgen05_fence_after();
        tmem_dealloc_pair(tmem_base, kTmemCols);
    }
}

}  // namespace catccos
