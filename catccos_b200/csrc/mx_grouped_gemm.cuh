// Grouped MXFP8 GEMM for sm_100a, the experts' products of a mixture-of-experts layer: with offsets [experts + 1] on the device,
//   C[offsets[e] .. offsets[e + 1])[N] = dequant(A rows) x dequant(B[e])[K, N]        for every expert e.
//
//   A      8-bit codes, rows K bytes apart or more (the packed rows of mx_quant_scatter_packed_kernel are read in place)
//   SFA    E8M0 bytes, K/32 a row, rows any multiple of four bytes apart
//   B      8-bit codes [experts, K, N];  SFB E8M0 [experts, K/64, N, 2]
//   C      bf16 or fp16 [rows, N]; rows outside the offsets are left as they are
//
// (mx_grouped_pair.cuh has the form for many rows an expert.)  The tile, the shared-memory ring, the tensor-memory layout and the warps' roles are those of mx_gemm_kernel.  What differs
// is the list of work: every CTA reads the offsets, counts each expert's 128-row tiles and walks the (expert, row tile, column
// tile) units blockIdx.x, blockIdx.x + gridDim.x, ... with the column tile running fastest, so that the CTAs that run at one
// time share a few experts' weights and rows in L2.  The host knows an upper bound of the units only.
//
// Decode (a few rows an expert) is bound by the weights' bytes; a row tile then loads its rows in boxes of 32, not 128 (A would
// be as much shared-memory traffic as B at 128 columns).  Rows of a box behind the expert's last belong to the next expert or
// to nobody: their products are not stored, and rows of the tensor core's tile do not meet.
#pragma once

#include "mx_gemm.cuh"

namespace catccos {

constexpr uint32_t kGroupedMaxExperts = 1024;

struct GroupedParams {
    const uint8_t* a_scales;
    size_t a_scale_stride;    // bytes between the scales of two rows
    const uint8_t* b_scales;
    const int32_t* offsets;
    void* c;
    uint32_t rows, experts, N, K;
    uint32_t a_fmt, b_fmt;    // 0 = E4M3, 1 = E5M2
    uint64_t bar_timeout_ns;
    StatusBlock* status;
};

// An expert's rows [begin, end).  Offsets that do not ascend or leave the matrix are cut to what lies inside.
__host__ __device__ __forceinline__ void grouped_rows(int32_t lo, int32_t hi, uint32_t rows, uint32_t& begin, uint32_t& end)
{
    begin = lo < 0 ? 0u : ((uint32_t)lo < rows ? (uint32_t)lo : rows);
    end = hi < 0 ? 0u : ((uint32_t)hi < rows ? (uint32_t)hi : rows);
    end = end < begin ? begin : end;
}

template <uint32_t BLOCK_N>
struct GroupedSmem {
    using S = GemmSmem<BLOCK_N>;
    // behind the GEMM's own: first tile of each expert [experts + 1], first row and end of each expert's rows
    static constexpr uint32_t kOffTiles = (S::kBytes + 15u) / 16u * 16u;
    static constexpr uint32_t dynamic_bytes(uint32_t experts) { return kOffTiles + (3u * experts + 1u) * 4u + 1024u; }
};

// The units of a CTA in ascending order; the expert only moves forward.
struct GroupedWalk {
    uint32_t e = 0;

    // row tile and column tile of `unit` (below the number of units); e is its expert
    __device__ __forceinline__ TileCoord seek(const uint32_t* tiles, uint32_t n_tiles, uint32_t unit)
    {
        const uint32_t tile = unit / n_tiles;
        while (tile >= tiles[e + 1u]) {
            ++e;
        }
        return {tile - tiles[e], unit - tile * n_tiles};
    }
};

// One warp: the experts' rows, and how many tiles of tile_rows rows lie before each expert's (tiles[experts]: all of them).
__device__ __forceinline__ void count_grouped_tiles(const GroupedParams& p, uint32_t tile_rows, uint32_t* tiles, uint32_t* row_begin,
                                                    uint32_t* row_end, uint32_t lane)
{
    uint32_t before = 0;
    for (uint32_t e0 = 0; e0 < p.experts; e0 += 32u) {
        const uint32_t e = e0 + lane;
        uint32_t begin = 0, end = 0;
        if (e < p.experts) {
            grouped_rows(__ldcg(p.offsets + e), __ldcg(p.offsets + e + 1u), p.rows, begin, end);
            row_begin[e] = begin;
            row_end[e] = end;
        }
        const uint32_t own = (end - begin + tile_rows - 1u) / tile_rows;
        uint32_t incl = own;
#pragma unroll
        for (uint32_t d = 1; d < 32; d <<= 1) {
            const uint32_t o = __shfl_up_sync(0xFFFFFFFFu, incl, d);
            incl += lane >= d ? o : 0u;
        }
        if (e < p.experts) {
            tiles[e] = before + incl - own;
        }
        before += __shfl_sync(0xFFFFFFFFu, incl, 31);
    }
    if (lane == 0) {
        tiles[p.experts] = before;
    }
}

template <uint32_t BLOCK_N, typename OutT>
__global__ void __launch_bounds__(kGemmThreads, 1)
mx_grouped_gemm_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_a32,
                       const __grid_constant__ CUtensorMap tmap_b, const __grid_constant__ GroupedParams p)
{
    using S = GemmSmem<BLOCK_N>;
    constexpr uint32_t kStages = S::kStages;

    grid_dep_launch();
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + S::kOffBar);
    uint64_t* full = bars;
    uint64_t* empty = bars + kStages;
    uint64_t* tmem_full = bars + 2 * kStages;
    uint64_t* tmem_empty = tmem_full + 2;
    uint64_t* overlap_free = tmem_empty + 2;
    uint32_t* tmem_ptr_smem = reinterpret_cast<uint32_t*>(smem + S::kOffTmemPtr);
    uint32_t* tiles = reinterpret_cast<uint32_t*>(smem + GroupedSmem<BLOCK_N>::kOffTiles);
    uint32_t* row_begin = tiles + p.experts + 1u;
    uint32_t* row_end = row_begin + p.experts;

    const uint32_t warp = threadIdx.x >> 5;
    const uint32_t lane = threadIdx.x & 31;
    const uint32_t n_tiles = (p.N + BLOCK_N - 1) / BLOCK_N;
    const uint32_t k_tiles = p.K / kGemmBlockK;
    const uint64_t bar_ns = p.bar_timeout_ns;

    if (threadIdx.x == 128) {
        for (uint32_t s = 0; s < kStages; ++s) {
            mbar_init(&full[s], 2);  // the producer's expect_tx arrival and one scale-loader warp
            mbar_init(&empty[s], 1);
        }
        for (uint32_t a = 0; a < 2; ++a) {
            mbar_init(&tmem_full[a], 1);
            mbar_init(&tmem_empty[a], 4);
            mbar_init(&overlap_free[a], 4);
        }
        mbar_fence_init();
        tma_prefetch_desc(&tmap_a);
        tma_prefetch_desc(&tmap_a32);
        tma_prefetch_desc(&tmap_b);
    }
    if (warp == 5) {
        tmem_alloc(tmem_ptr_smem, kTmemCols);
        tmem_relinquish();
    }
    grid_dep_wait();  // the offsets, the rows and their scales come from the kernels before this one
    if (warp == 0) {
        count_grouped_tiles(p, kGemmBlockM, tiles, row_begin, row_end, lane);
    }
    tcgen05_fence_before();
    __syncthreads();
    tcgen05_fence_after();
    const uint32_t tmem_base = *tmem_ptr_smem;
    const uint32_t num_units = tiles[p.experts] * n_tiles;
    bool alive = true;  // false once a wait of this role has given up
    GroupedWalk walk;

    if (warp == 4) {
        // ------------------------------- TMA producer -------------------------------------
        uint32_t it = 0;
        for (uint32_t unit = blockIdx.x; alive && unit < num_units; unit += gridDim.x) {
            const TileCoord tc = walk.seek(tiles, n_tiles, unit);
            const uint32_t m0 = row_begin[walk.e] + tc.m_tile * kGemmBlockM;
            const uint32_t boxes = (min(row_end[walk.e] - m0, kGemmBlockM) + 31u) / 32u;
            const uint32_t n0 = tc.n_tile * BLOCK_N;
            const uint32_t tx_bytes = boxes * (32u * kGemmBlockK) + S::kBBytes;
            const uint32_t b_row0 = walk.e * p.K;
            for (uint32_t kt = 0; alive && kt < k_tiles; ++kt, ++it) {
                const uint32_t s = it % kStages;
                alive = mbar_wait_warp(&empty[s], ((it / kStages) & 1u) ^ 1u, p.status, 100, s, bar_ns);
                if (!alive) {
                    break;
                }
                if (elect_one()) {
                    mbar_arrive_expect_tx(&full[s], tx_bytes);
                    for (uint32_t h = 0; h < BLOCK_N / S::kBRow; ++h) {
                        tma_load_2d(smem + S::kOffB + s * S::kBBytes + h * 16384u, &tmap_b, &full[s], (int32_t)(n0 + h * 128u),
                                    (int32_t)(b_row0 + kt * kGemmBlockK));
                    }
                    uint8_t* a = smem + S::kOffA + s * S::kABytes;
                    if (boxes == 4u) {
                        tma_load_2d(a, &tmap_a, &full[s], (int32_t)(kt * kGemmBlockK), (int32_t)m0);
                    } else {
                        for (uint32_t i = 0; i < boxes; ++i) {
                            tma_load_2d(a + i * (32u * kGemmBlockK), &tmap_a32, &full[s], (int32_t)(kt * kGemmBlockK),
                                        (int32_t)(m0 + i * 32u));
                        }
                    }
                }
                __syncwarp();
            }
        }
    } else if (warp == 5) {
        // ------------------------------- MMA issuer ---------------------------------------
        const uint32_t idesc0 = make_idesc_mxf8(kGemmBlockM, 0, true) | ((p.a_fmt & 7u) << 7) | ((p.b_fmt & 7u) << 10);
        const uint32_t hi_a = (uint32_t)(make_smem_desc(0, 16, 1024, 2) >> 32);
        const uint64_t desc_b = make_smem_desc(0, 16384, 8 * S::kBRow, S::kBRow == 64 ? 4 : 2);
        const uint32_t hi_b = (uint32_t)(desc_b >> 32);
        const uint32_t a_lo0 = (uint32_t)make_smem_desc(0, 16, 1024, 2) | (smem_u32(smem + S::kOffA) >> 4);
        const uint32_t b_lo0 = (uint32_t)desc_b | (smem_u32(smem + S::kOffB) >> 4);
        constexpr uint32_t kKbStepA = 32u >> 4, kKbStepB = (32u * S::kBRow) >> 4;
        uint32_t s = 0, ph = 0, ti = 0;
        for (uint32_t unit = blockIdx.x; alive && unit < num_units; unit += gridDim.x, ++ti) {
            const uint32_t acc = ti & 1u;
            const uint32_t d_col = tmem_base + (acc ? S::kAccCol1 : 0u);
            alive = mbar_wait_warp(&tmem_empty[acc], ((ti >> 1) & 1u) ^ 1u, p.status, 101, acc, bar_ns);
            if (S::kOverlap && ti > 0 && alive) {
                alive = mbar_wait_warp(&overlap_free[acc ^ 1u], ((ti - 1) >> 1) & 1u, p.status, 102, acc, bar_ns);
            }
            // a ragged last column of tiles is multiplied as wide as it is (a multiple of 16)
            const uint32_t left = p.N - unit % n_tiles * BLOCK_N;
            const uint32_t idesc = idesc0 | ((min(left, BLOCK_N) >> 3) << 17);
            for (uint32_t kt = 0; alive && kt < k_tiles; ++kt) {
                alive = mbar_wait_warp(&full[s], ph, p.status, 103, s, bar_ns);
                if (!alive) {
                    break;  // nothing is issued, and the accumulator never reported, after a wait has given up
                }
                tcgen05_fence_after();
                const uint32_t a_lo = a_lo0 + s * (S::kABytes >> 4);
                const uint32_t b_lo = b_lo0 + s * (S::kBBytes >> 4);
                const uint32_t sf = tmem_base + S::kSfCol + s * S::kSfSetCols;
                if (elect_one()) {
#pragma unroll
                    for (uint32_t kb = 0; kb < 4; ++kb) {
                        umma_mxf8_lohi(d_col, a_lo + kb * kKbStepA, hi_a, b_lo + kb * kKbStepB, hi_b, idesc_with_sf_id(idesc, kb),
                                       sf, sf + 4, (kb != 0u || kt != 0u) ? 1u : 0u);
                    }
                    tcgen05_commit(&empty[s]);
                    if (kt + 1u == k_tiles) {
                        tcgen05_commit(&tmem_full[acc]);
                    }
                }
                __syncwarp();
                s = (s + 1 == kStages) ? 0u : s + 1;
                ph ^= s == 0u ? 1u : 0u;
            }
        }
    } else if (warp >= 6) {
        // ------------------------------- scale loaders ------------------------------------
        // Warp j takes the K tiles whose running index is j modulo 4 (mx_gemm_kernel has the layout of the atoms).
        constexpr uint32_t kNB = S::kSfbAtoms * 4;  // B words per lane
        const uint32_t j = warp - 6;
        const uint32_t my_units = num_units > blockIdx.x ? (num_units - blockIdx.x + gridDim.x - 1) / gridDim.x : 0u;
        const uint32_t total_it = my_units * k_tiles;
        uint32_t cur_a[4], cur_lo[kNB], cur_hi[kNB];
        uint32_t nxt_a[4], nxt_lo[kNB], nxt_hi[kNB];
        uint32_t seq = 0, seq_it = 0;  // the unit of the K tile looked at last, and its first K tile's index

        auto issue_loads = [&](uint32_t it, uint32_t (&ra)[4], uint32_t (&rlo)[kNB], uint32_t (&rhi)[kNB]) {
            while (it - seq_it >= k_tiles) {
                ++seq;
                seq_it += k_tiles;
            }
            const uint32_t kt = it - seq_it;
            const TileCoord tc = walk.seek(tiles, n_tiles, blockIdx.x + seq * gridDim.x);
            const uint32_t m0 = row_begin[walk.e] + tc.m_tile * kGemmBlockM;
            const uint32_t end = row_end[walk.e];
            const uint32_t n0 = tc.n_tile * BLOCK_N;
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) {
                const uint32_t row = m0 + i * 32 + lane;
                ra[i] = 0x7F7F7F7Fu;
                if (row < end) {
                    ra[i] = __ldcg(reinterpret_cast<const uint32_t*>(p.a_scales + (size_t)row * p.a_scale_stride + kt * 4u));
                }
            }
            const uint8_t* b_scales = p.b_scales + ((size_t)walk.e * (p.K / 64u) + 2u * kt) * p.N * 2u;
#pragma unroll
            for (uint32_t i = 0; i < kNB; ++i) {
                const uint32_t n = n0 + i * 32 + lane;
                rlo[i] = 0x7F7Fu;
                rhi[i] = 0x7F7Fu;
                if (i * 32u < BLOCK_N && n < p.N) {
                    rlo[i] = *reinterpret_cast<const uint16_t*>(b_scales + (size_t)n * 2u);
                    rhi[i] = *reinterpret_cast<const uint16_t*>(b_scales + ((size_t)p.N + n) * 2u);
                }
            }
        };

        uint32_t it = j;
        if (it < total_it) {
            issue_loads(it, cur_a, cur_lo, cur_hi);
        }
        for (; alive && it < total_it; it += kSfWarps) {
            const bool has_next = it + kSfWarps < total_it;
            if (has_next) {
                issue_loads(it + kSfWarps, nxt_a, nxt_lo, nxt_hi);
            }
            const uint32_t s = it % kStages;
            alive = mbar_wait_warp(&empty[s], ((it / kStages) & 1u) ^ 1u, p.status, 105, s, bar_ns);
            if (!alive) {
                break;
            }
            uint8_t* sfa = smem + S::kOffSfa + s * S::kSfaBytes;
            uint8_t* sfb = smem + S::kOffSfb + s * S::kSfbBytes;
            *reinterpret_cast<uint4*>(sfa + lane * 16u) = make_uint4(cur_a[0], cur_a[1], cur_a[2], cur_a[3]);
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
            tcgen05_fence_after();
            if (elect_one()) {
                const uint32_t hi_sf = (uint32_t)(make_smem_desc(0, 0, 128, 0) >> 32);  // 32 rows x 16 bytes, no swizzle
                const uint32_t sf_t = tmem_base + S::kSfCol + s * S::kSfSetCols;
                tcgen05_cp_sf_lohi(sf_t, smem_u32(sfa) >> 4, hi_sf);
#pragma unroll
                for (uint32_t h = 0; h < S::kSfbAtoms; ++h) {
                    tcgen05_cp_sf_lohi(sf_t + 4 + 4 * h, (smem_u32(sfb) >> 4) + h * (512u >> 4), hi_sf);
                }
                tcgen05_commit(&full[s]);
            }
            __syncwarp();
            if (has_next) {
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i) cur_a[i] = nxt_a[i];
#pragma unroll
                for (uint32_t i = 0; i < kNB; ++i) {
                    cur_lo[i] = nxt_lo[i];
                    cur_hi[i] = nxt_hi[i];
                }
            }
        }
    } else {
        // ------------------------------- epilogue -----------------------------------------
        const uint32_t q = warp;  // TMEM lane quarter == warp index modulo 4
        constexpr uint32_t kChunks = BLOCK_N / 32;
        uint32_t ti = 0;
        for (uint32_t unit = blockIdx.x; alive && unit < num_units; unit += gridDim.x, ++ti) {
            const TileCoord tc = walk.seek(tiles, n_tiles, unit);
            const uint32_t first = row_begin[walk.e] + tc.m_tile * kGemmBlockM + q * 32u;
            const uint32_t end = row_end[walk.e];
            const uint32_t n0 = tc.n_tile * BLOCK_N;
            const uint32_t acc = ti & 1u;
            const uint32_t d_col = acc ? S::kAccCol1 : 0u;
            alive = mbar_wait_warp(&tmem_full[acc], (ti >> 1) & 1u, p.status, 106, acc, bar_ns);
            if (!alive) {
                break;  // an accumulator that never filled is not written out
            }
            tcgen05_fence_after();
            const uint32_t row = first + lane;
            OutT* dst = static_cast<OutT*>(p.c) + (size_t)row * p.N + n0;
            // the chunks that hold the columns shared with the other accumulator go first
            for (uint32_t ci = 0; ci < kChunks; ++ci) {
                uint32_t chunk = ci;
                if (S::kOverlap && acc == 0) {
                    chunk = ci < S::kOverlapChunks ? kChunks - S::kOverlapChunks + ci : ci - S::kOverlapChunks;
                }
                uint32_t r[32];
                if (first < end) {  // a warp whose rows all lie behind the expert's last has nothing to fetch
                    tmem_ld_32x32(tmem_base + ((q * 32u) << 16) + d_col + chunk * 32u, r);
                    tmem_ld_wait();
                }
                if (S::kOverlap && ci == S::kOverlapChunks - 1) {
                    tcgen05_fence_before();
                    __syncwarp();
                    if (lane == 0) {
                        mbar_arrive(&overlap_free[acc]);
                    }
                }
                if (row < end) {
#pragma unroll
                    for (uint32_t v = 0; v < 2; ++v) {
                        if (n0 + chunk * 32u + v * 16u < p.N) {
                            uint32_t o[8];
#pragma unroll
                            for (uint32_t x = 0; x < 8; ++x) {
                                o[x] = pack2<OutT>(__uint_as_float(r[v * 16 + 2 * x]), __uint_as_float(r[v * 16 + 2 * x + 1]));
                            }
                            st_global_v8(dst + chunk * 32u + v * 16u, o);
                        }
                    }
                }
            }
            tcgen05_fence_before();
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(&tmem_empty[acc]);
            }
        }
    }

    tcgen05_fence_before();
    if (__syncthreads_or(alive ? 0 : 1)) {
        drain_after_abort(p.status);
    }
    if (warp == 5) {
        tcgen05_fence_after();
        tmem_dealloc(tmem_base, kTmemCols);
    }
}

}  // namespace catccos
