// Which form a product of blocks of 128 takes: CTA pairs (block_gemm_pair.cuh), or tiles of few rows with K in parts (block_gemm.cuh).
// Host code without CUDA, so that it is tested by itself.
#pragma once

#include <algorithm>
#include <cmath>
#include <cstdint>

namespace catccos {

constexpr uint32_t kBlockFewColumns = 128;  // of the weight, to a tile of few rows
constexpr uint32_t kBlockFewMaxParts = 8;
constexpr uint32_t kBlockPairM = 256, kBlockPairN = 128;
static_assert(kBlockPairN == kBlockFewColumns, "the plan counts columns of tiles alike");

struct BlockCall {
    uint32_t rows, experts, n, k;
    bool grouped;     // rows of experts: how many each has is on the device
    bool pairs_only;  // scales by column, or a stored by column: the form for few rows has neither
};

// The options: 0 is automatic
struct BlockChoice {
    int block_rows;  // 16, 32, 64: tiles of so many rows
    int split_k;     // at most so many parts of K
    int cta_pair;    // 1: pairs, 2: no pairs
};

// rows 0: pairs
struct BlockPlan {
    uint32_t rows, parts;
};

// Units of a launch of single CTAs (grouped: as many as there may be, one row tile that is not full for every expert with rows).
inline uint64_t block_units(const BlockCall& c, uint32_t tile_rows, uint32_t tile_columns)
{
    const uint64_t tiles = c.grouped ? c.rows / tile_rows + std::min(c.rows, c.experts) : ((uint64_t)c.rows + tile_rows - 1) / tile_rows;
    return tiles * ((c.n + tile_columns - 1) / tile_columns);
}

// The form that takes least by a fit to 600 measured calls (dense with 1 to 1024 rows, experts with 1 to 512 rows each; 14 to 22 % off): a
// launch, then for each round of units a block of K, which takes longer the more SMs are busy, and the output; the meeting of the parts.
// So chosen, a call takes 2.4 % more than in the best form in the mean of 176; by the rows alone (16, 32, 64, pairs above 128 rows an expert)
// it would be 13 %.  21 of them take more than 10 % more, at most 1.37 times as long (256 x 2304 x 7168 30.8 us, in pairs 22.5): clusters of
// four and eight CTAs, which have to lie in one GPC, are counted as if as many fitted as single CTAs.  An expert's rows are reckoned with
// as in plan_grouped.
inline BlockPlan plan_block_gemm(const BlockCall& call, const BlockChoice& choice, uint32_t num_sms)
{
    struct Cost {
        uint32_t rows;
        double launch, block, busy_block, round, meeting;
    };
    constexpr Cost costs[] = {{0, 4.28, 0.299, 0.053, 0.50, 0}, {16, 3.71, 0.219, 0.205, 0.28, 1.29}, {32, 3.82, 0.241, 0.235, 0.56, 1.96}, {64, 5.06, 0.286, 0.360, 0.72, 2.37}};
    if (call.pairs_only || choice.cta_pair == 1) {
        return {0, 1};
    }
    const uint32_t k_blocks = (call.k + 127u) / 128u;
    const double active = std::min(call.rows, call.experts) < 2 ? 1.0 : 0.9 * std::min(call.rows, call.experts);
    BlockPlan best = {0, 0};
    double least = 0;
    for (const Cost& c : costs) {
        if ((choice.block_rows != 0 && (uint32_t)choice.block_rows != c.rows) || (choice.block_rows == 0 && choice.cta_pair == 2 && c.rows == 0)) {
            continue;  // a test names the form
        }
        const uint32_t tile_rows = c.rows ? c.rows : kBlockPairM;
        uint32_t parts = 1;
        const uint64_t most = block_units(call, tile_rows, kBlockFewColumns);
        while (c.rows != 0 && parts < kBlockFewMaxParts && most * parts * 2 <= 2 * (uint64_t)num_sms && parts * 2 <= k_blocks &&
               (choice.split_k == 0 || parts * 2 <= (uint32_t)choice.split_k)) {
            parts *= 2;
        }
        const double tiles = call.grouped ? std::max(active, call.rows / (double)tile_rows + 0.7 * active) : std::ceil(call.rows / (double)tile_rows);
        const double units = tiles * ((call.n + kBlockFewColumns - 1) / kBlockFewColumns) * parts, slots = c.rows ? 2 * num_sms : num_sms / 2;
        const double time = c.launch + (parts > 1 ? c.meeting : 0) +
                            std::ceil(units / slots) * ((k_blocks + parts - 1) / parts * (c.block + c.busy_block * std::min(1.0, units / slots)) + c.round);
        if (best.parts == 0 || time < least) {
            best = {c.rows, parts};
            least = time;
        }
    }
    return best;
}

}  // namespace catccos
